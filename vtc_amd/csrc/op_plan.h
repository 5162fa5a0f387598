// Launch shapes of the operators as plain host functions of their sizes: tiles and K splits of the feed-forward's products, tokens of a
// rotary block.  They need no GPU, so host code can ask what a call will run (tests/op_plan_table.cpp).
#pragma once
#include <algorithm>
#include <cmath>
#include <cstdint>

namespace vtc {

// A launch holds fewer than 2^32 threads; the difference is room for a few blocks on top
constexpr long long kLaunchThreads = (1ll << 32) - (1 << 17);
constexpr long long kMaxBlocks = kLaunchThreads / 256;   // of 256 threads

inline int div_up(long long a, int b) { return (int)((a + b - 1) / b); }

// How a product runs: tile size and K splits, by a model of its time (us) fitted to kernel times measured at 768 x 2048.  A round is
// as many tiles as the chip holds at once (256 of 256 rows, one per CU; 512 of 128 x 64, two per CU); `fill` is its share in use,
// since K-tiles slow down as more CUs fetch.  Per K-tile: 1.35 + 0.75 fill for 256 x 256 (x 3/4 for 192 columns), 0.42 + 0.38 fill
// for 128 x 64; per tile the epilogue's share.  Partials cross memory twice at 4 TB/s and cost a launch.  Measured, 256-wide / small:
//   gate and up      512 rows 22 / 10   2048 26 / 24   4096 30 / 43   16384 109 / 183
//   ..., slopes kept 512 rows 29 / 13   2048 33 / 31   4096 38 / 54   16384 147 / 236
//   down             512 rows 36 / 12   2048 37 / 18   8192 43 / 39   16384  59 / 81
//   dx               512 rows 72 / 16   2048 74 / 30   8192 86 / 82   16384 109 / 173
//   dg and du        512 rows 36 / 13   2048 37 / 20   8192 88 / 73   16384 149 / 162
//   weights          512 rows 31 / 22   2048 46 / 44   8192 91 / 137  16384 165 / 290
// Whole training steps at other widths, by this rule / all small / all 256-wide (bf16, us): 256 x 512, 8192 rows 66 / 65 / 121, 31936 rows 199 /
// 198 / 207; 1024 x 4096, 2048 rows 229 / 264 / 349, 8192 rows 740 / 1018 / 742; 2048 x 8192, 512 rows 333 / 355 / 634, 2048 rows 772 / 1007 /
// 906, 8192 rows 2445 / 3979 / 2461; 389 x 1031, 1024 rows 60 / 60 / 166, 8192 rows 198 / 189 / 228.
struct OgPlan { bool small; int splits, kps; };
struct OgCost { long long tiles_big, tiles_small; double width, end_big, end_small; };   // tiles; epilogue of a tile
inline OgPlan og_plan(const OgCost& o, int nk, int splits_big, int splits_small, double out_elems) {
  OgPlan best{false, 1, (nk + 1) & ~1};
  double cost = 1e300;
  for (int small = 0; small < 2; ++small)
    for (int sp = 1; sp <= (small ? splits_small : splits_big); ++sp) {
      if (small && o.tiles_small * sp > kMaxBlocks) break;   // (256-wide tiles run on 256 blocks at most)
      int k = (nk + sp - 1) / sp;
      if (!small) k = (k + 1) & ~1;
      if (sp > 1 && k < 4) break;
      if ((nk + k - 1) / k != sp) continue;
      const double cap = small ? 512.0 : 256.0, units = (double)(small ? o.tiles_small : o.tiles_big) * sp;
      auto round = [&](double fill) { return small ? k * (0.42 + 0.38 * fill) + o.end_small : k * o.width * (1.35 + 0.75 * fill) + o.end_big; };
      const double full = std::floor(units / cap), rest = units / cap - full;
      double c = full * round(1.0) + (rest > 0.0 ? round(rest) : 0.0);
      if (sp > 1) c += 4.0 + sp * out_elems * 8.0 / 4.0e6;
      if (c < cost) { cost = c; best = OgPlan{small != 0, sp, k}; }
    }
  return best;
}
// Tiles of the products: gate and up, C = A B^T of many rows (down, dx; nk K-tiles), dg and du, the three weights' gradients.  F8: inner
// width with its padding columns.
inline OgPlan plan_gate(int64_t M, int K, int F8, bool save) {
  return og_plan({(long long)div_up(M, 256) * div_up(F8, 128), (long long)div_up(M, 128) * div_up(F8, 32), 1.0, save ? 12.0 : 5.0, save ? 6.0 : 4.0},
                 div_up(K, 64), 1, 1, 0);
}
inline OgPlan plan_rows(int64_t M, int N, int nk) {
  return og_plan({(long long)div_up(M, 256) * div_up(N, 192), (long long)div_up(M, 128) * div_up(N, 64), 0.75, 4.0, 2.0}, nk, 1, 32, (double)M * N);
}
inline OgPlan plan_dgate(int64_t M, int N, int F8) {
  return og_plan({(long long)div_up(M, 256) * div_up(F8, 192), (long long)div_up(M, 128) * div_up(F8, 64), 0.75, 20.0, 7.0}, div_up(N, 64), 1, 1, 0);
}
inline OgPlan plan_weights(int64_t M, int K, int F, int N) {
  const int K8 = (K + 7) & ~7, F8 = (F + 7) & ~7;
  const int rows[3] = {F, F, N}, pitch[3] = {K8, K8, F8};
  long long big = 0, small = 0, elems = 0;
  for (int i = 0; i < 3; ++i) {
    big += (long long)div_up(rows[i], 256) * div_up(pitch[i], 256);
    small += (long long)div_up(rows[i], 128) * div_up(pitch[i], 64);
    elems += (long long)rows[i] * pitch[i];
  }
  return og_plan({big, small, 1.0, 6.0, 3.0}, div_up(M, 64), 32, 32, (double)elems);
}

// Tokens of a rotary block: ~4 items per thread, at least ~1000 blocks where there are rows for it, no more blocks than a launch holds, and
// the angle table within its LDS (table: tokens it holds)
inline int rotary_tokens_per_block(long long tokens, long long per_token, long long table) {
  long long n = std::max(1ll, 1024 / per_token);
  n = std::min(n, std::max(1ll, tokens / 1024));
  n = std::max(n, (tokens + kMaxBlocks - 1) / kMaxBlocks);
  return (int)std::min(n, table);
}

}  // namespace vtc
