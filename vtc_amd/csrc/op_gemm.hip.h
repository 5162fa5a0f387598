// Matrix products of the gated feed-forward block, any sizes: 256 x BN x 64 tiles, 8 waves, persistent, the schedule of
// gemm256.hip.h (two K-tile buffers in LDS, four half-tiles, one half-tile prefetched per phase, counted vmcnt, staggered wave
// rows) with three differences:
//   * operands are fetched through buffer descriptors rebuilt per half-tile (scalar work): rows, columns and K beyond the matrix
//     read as zero, so no size has to divide anything but 8 (16-byte pieces), and the 32-bit offsets are relative to the tile
//     (matrices beyond 4 GiB work);
//   * an operand may be stored with the contraction index along its ROWS ("KS": dy^T h, dg^T x, dy W_down).  Its half-tile is 64
//     k-rows x 128 columns (256 B each); ds_read_b64_tr_b16 hands every lane 4 k of one column, so two of them make the fragment
//     that one ds_read_b128 reads from the other layout and nothing is transposed in memory.  32-byte pieces of a k-row are
//     XOR-swizzled by (k & 3) | (k >> 3 & 1) << 2: the 8 k-rows a half-wave reads fall into 8 different pieces;
//   * the contraction may run over two operand pairs (dx = dg W_gate + du W_up) or be split over K into fp32 partials.
//
// Accumulators hold C^T: lane (fr, fq) has row i * 16 + fr and, of each 32-column group, columns 8 fq .. + 8.
#pragma once
#include "common.hip.h"
#include "gemm256.hip.h"
#include "op_act.hip.h"

namespace vtc {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

struct OpMat {
  const h16* p;
  long long ld;   // elements between rows of the stored matrix (a multiple of 8)
};
// One product C[M, N] (+)= A B^T.  Stored shapes: A is [M][K] (or [K][M] when KS), B is [N][K] (or [K][N]).
struct OpProb {
  OpMat a[2], b[2];
  void* c;
  long long ldc;
  int M, N, Nb;    // N: columns of C that are written; Nb: rows (KS: columns) of B that exist (C's padding columns come out as zero)
  int tiles_m, tiles_n, group_n, tile0;   // tile0: index of the problem's first tile in the launch
  int cvec;        // columns of a row of c start 16-byte aligned: whole-vector stores
};
enum : int { OG_PLAIN = 0,   // 16-bit C (+ bias)
             OG_PART = 1,    // fp32 partial of a K split
             OG_GATE = 2,    // b[0] = W_gate, b[1] = W_up: h = act(g) u, g and u stored when asked for
             OG_DGATE = 3 }; // C = dh: dg = dh u act'(g), du = dh act(g), and their column sums
struct OpGemmParams {
  OpProb prob[3];
  int nprob, ntiles;          // ntiles: tiles of all problems
  int K[2], nk0, nk;          // contraction lengths of the two segments; K-tiles of the first, of both (even)
  int splits, kps;            // K splits, K-tiles of a split (even); split s covers [s kps, min(nk, (s + 1) kps))
  long long split_stride;     // elements between partials
  const void *bias, *bias2;   // OG_PLAIN: bias; OG_GATE: b_gate, b_up (type: bias_f32 ? fp32 : the operands')
  int bias_f32, act;
  h16 *g, *u;                 // OG_GATE: stored pre-activations (may be null); OG_DGATE: read
  h16 *dg, *du;               // OG_DGATE
  long long ldg;              // of g, u, dg, du (and h)
  float* colsum;              // OG_DGATE: [2][2 tiles_m][N] sums of dg, du over the 128 rows of a wave row, or null
};

__device__ __forceinline__ float op_bias(const void* b, int i, int f32, bool f16) {
  if (!b) return 0.f;
  if (f32) return ((const float*)b)[i];
  const h16 v = ((const h16*)b)[i];
  return f16 ? from_h16<true>(v) : from_h16<false>(v);
}

template <bool F16, bool AKS, bool BKS, int EPI, int BN>
__global__ __launch_bounds__(512, 2) void op_gemm_kernel(const OpGemmParams p) {
  using TC = Tile256<BN>;
  constexpr int NJ1 = TC::NJ1;
  static_assert(!BKS || BN == 256, "a KS operand B is staged in halves of 128 columns");
  static_assert(EPI != OG_GATE || BN == 256, "gate and up columns sit in the two halves of a tile");
  __shared__ __attribute__((aligned(16))) char smem[TC::SMEM];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 2, wn = wave & 3;
  const int fr = lane & 15, fq = lane >> 4;
  constexpr unsigned OOB = 0x80000000u;

  // ---- staging: lane offsets (bytes from the half-tile's origin) and the scalar description of the tile being staged
  const int lr = lane >> 3, lc = lane & 7;
  unsigned va[2], vb[2], vb1[NJ1];   // offsets of the two instructions of a half-tile (B1: NJ1)
  int kca[2], kcb[2], kcb1[NJ1];     // KC operands: first k of the lane's piece inside the K-tile
  struct Src { const char *a, *b0, *b1; int am, bn0, bn1; long long lda, ldb, ldb1; int K; };   // am / bn: rows or columns left in the half
  constexpr int NSEG = (EPI == OG_PLAIN && BKS) ? 2 : 1;   // dx sums over two operand pairs
  constexpr bool MULTI = AKS;                              // several problems in one launch: the weights' gradients
  Src src[NSEG];
  int kt_base = 0, nk_cur = 0;       // first K-tile of the tile being staged

  auto unit = [&](unsigned t, int& pi, int& tm, int& tn, int& k0, int& k1) {   // work unit -> problem, tile, K-tiles
    const unsigned ti = t / (unsigned)p.splits;
    const int s = (int)(t - ti * (unsigned)p.splits);
    pi = 0;
    if constexpr (MULTI) {
      if (p.nprob > 1 && (int)ti >= p.prob[1].tile0) pi = 1;
      if (p.nprob > 2 && (int)ti >= p.prob[2].tile0) pi = 2;
    }
    const OpProb& q = p.prob[pi];
    const unsigned r0 = ti - (unsigned)q.tile0, per = (unsigned)(q.tiles_m * q.group_n);
    const unsigned g = r0 / per, r = r0 - g * per;
    tm = (int)(r / (unsigned)q.group_n);
    tn = (int)(g * (unsigned)q.group_n + r % (unsigned)q.group_n);
    k0 = s * p.kps;
    k1 = min(p.nk, k0 + p.kps);
  };

  auto set_sources = [&](int pi, int tm, int tn) {
    const OpProb& q = p.prob[pi];
    const int m0 = tm * 256;
    const int n0 = EPI == OG_GATE ? tn * 128 : tn * BN;
    const int n1 = EPI == OG_GATE ? n0 : n0 + 128;
#pragma unroll
    for (int s = 0; s < NSEG; ++s) {
      Src& d = src[s];
      const OpMat A = q.a[s], B = EPI == OG_GATE ? q.b[0] : q.b[s], B1 = EPI == OG_GATE ? q.b[1] : q.b[s];
      d.K = p.K[s];
      d.lda = A.ld; d.ldb = B.ld; d.ldb1 = B1.ld;
      d.am = q.M - m0; d.bn0 = q.Nb - n0; d.bn1 = q.Nb - n1;
      d.a = (const char*)A.p + (AKS ? (long long)m0 * 2 : (long long)m0 * A.ld * 2);
      d.b0 = (const char*)B.p + (BKS ? (long long)n0 * 2 : (long long)n0 * B.ld * 2);
      d.b1 = (const char*)B1.p + (BKS ? (long long)n1 * 2 : (long long)n1 * B1.ld * 2);
    }
  };
  // lane offsets do not depend on the tile (both segments of a product have the same pitch per side)
  {
    const OpProb& q = p.prob[0];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = (wave * 2 + i) * 8 + lr;                 // KC: row of the half-tile, piece lc holds chunk lc ^ swz(r)
      const int ch = lc ^ lds_swz(r);
      const int kr = (wave * 2 + i) * 4 + (lane >> 4);       // KS: k-row of the half-tile
      const int sw = (kr & 3) | ((kr >> 3 & 1) << 2);
      const int cc = ((((lane & 15) >> 1) ^ sw) << 1) | (lane & 1);   // 16-byte column piece
      kca[i] = AKS ? cc * 8 : ch * 8;
      va[i] = AKS ? (unsigned)(kr * (int)q.a[0].ld * 2 + cc * 16) : (unsigned)(r * (int)q.a[0].ld * 2 + ch * 16);
      const int wr = (r & ~31) + perm32(r & 31);
      kcb[i] = BKS ? cc * 8 : ch * 8;
      vb[i] = BKS ? (unsigned)(kr * (int)q.b[0].ld * 2 + cc * 16) : (unsigned)(wr * (int)q.b[0].ld * 2 + ch * 16);
    }
#pragma unroll
    for (int i = 0; i < NJ1; ++i) {
      const int r = (wave * NJ1 + i) * 8 + lr;
      const int ch = lc ^ lds_swz(r);
      const int wr = NJ1 == 2 ? (r & ~31) + perm32(r & 31) : r;
      kcb1[i] = BKS ? kcb[i] : ch * 8;
      vb1[i] = BKS ? vb[i] : (unsigned)(wr * (int)q.b[0].ld * 2 + ch * 16);
    }
  }
  // (several problems of one launch may have different pitches: recomputed at a switch, see `repitch`)
  auto repitch = [&](int pi) {
    const OpProb& q = p.prob[pi];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int kr = (wave * 2 + i) * 4 + (lane >> 4);
      if constexpr (AKS) va[i] = (unsigned)(kr * (int)q.a[0].ld * 2 + kca[i] * 2);
      if constexpr (BKS) { vb[i] = (unsigned)(kr * (int)q.b[0].ld * 2 + kcb[i] * 2); vb1[i] = vb[i]; }
    }
  };

  // one 16-byte-per-lane copy to LDS.  KC: rows beyond the matrix lie behind num_records, k beyond K is masked per lane.
  // KS: k-rows beyond K lie behind num_records, columns beyond the matrix are masked per lane.
  auto fetch = [&](bool ks, const char* base, long long ld, int left, int K, int kt, unsigned vo, int piece, char* lds) {
    int rows, cols, lim;
    const char* b;
    if (ks) {
      rows = min(64, K - kt * 64);
      cols = min(left, 128);
      b = base + (long long)kt * 64 * ld * 2;
      lim = left;
    } else {
      rows = min(left, 128);
      cols = K - kt * 64;          // > 0 wherever the piece is not masked
      b = base + (long long)kt * 128;
      lim = K - kt * 64;
    }
    const int n = (rows > 0 && cols > 0) ? (int)(((long long)(rows - 1) * ld + ((cols + 7) & ~7)) * 2) : 0;   // rows are padded to 16 bytes
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)b, 0, n, 0x00020000);
    const unsigned off = piece < lim ? vo : OOB;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, LPTR(lds), 16, (int)off, 0, 0, 0);
  };
  auto seg = [&](int& kt) -> const Src& {   // K-tile of the tile -> segment and K-tile inside it
    if constexpr (NSEG == 2) {
      if (kt >= p.nk0) { kt -= p.nk0; return src[1]; }
    }
    return src[0];
  };
  auto issue_a = [&](int h, int buf, int kt_) {
    int kt = kt_ + kt_base;
    const Src& s = seg(kt);
    char* d = smem + buf * TC::BUF + (h ? TC::OFF_A1 : TC::OFF_A0) + wave * 2048;
    const char* base = s.a + (h ? (AKS ? 256ll : 128 * s.lda * 2) : 0ll);
#pragma unroll
    for (int i = 0; i < 2; ++i) fetch(AKS, base, s.lda, s.am - h * 128, s.K, kt, va[i], kca[i], d + i * 1024);
  };
  auto issue_b0 = [&](int buf, int kt_) {
    int kt = kt_ + kt_base;
    const Src& s = seg(kt);
    char* d = smem + buf * TC::BUF + TC::OFF_B0 + wave * 2048;
#pragma unroll
    for (int i = 0; i < 2; ++i) fetch(BKS, s.b0, s.ldb, s.bn0, s.K, kt, vb[i], kcb[i], d + i * 1024);
  };
  auto issue_b1 = [&](int buf, int kt_) {
    int kt = kt_ + kt_base;
    const Src& s = seg(kt);
    char* d = smem + buf * TC::BUF + TC::OFF_B1 + wave * (NJ1 * 1024);
#pragma unroll
    for (int i = 0; i < NJ1; ++i) fetch(BKS, s.b1, s.ldb1, s.bn1, s.K, kt, vb1[i], kcb1[i], d + i * 1024);
  };

  // ---- fragments
  const int tq = (lane & 15) >> 2, tp = lane & 3;                // KS: k inside a block of 4, piece of 4 columns
  const int ksw = tq | ((fq & 1) << 2);
  int a_off[4], b0_off[2], b1_off[NJ1], a_sw[4], b0_sw[2], b1_sw[NJ1];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = wm * 64 + i * 16 + fr;
    if constexpr (AKS) { a_off[i] = (fq * 8 + tq) * 256 + (((wm * 4 + i) ^ ksw) << 5) + 8 * tp; a_sw[i] = 0; }
    else { a_off[i] = r * 128; a_sw[i] = lds_swz(r); }
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int r = wn * 32 + j * 16 + fr;
    if constexpr (BKS) { b0_off[j] = (fq * 8 + tq) * 256 + (((wn * 2 + (tp >> 1)) ^ ksw) << 5) + (tp & 1) * 16 + 8 * j; b0_sw[j] = 0; }
    else { b0_off[j] = r * 128; b0_sw[j] = lds_swz(r); }
  }
#pragma unroll
  for (int j = 0; j < NJ1; ++j) {
    const int r = wn * (16 * NJ1) + j * 16 + fr;
    if constexpr (BKS) { b1_off[j] = b0_off[j]; b1_sw[j] = 0; }
    else { b1_off[j] = r * 128; b1_sw[j] = lds_swz(r); }
  }
  auto frag_kc = [&](const char* base, int off, int sw, int ks) { return *(const u16x8*)(base + off + (((ks * 4 + fq) ^ sw) << 4)); };
  auto frag_ks = [&](const char* base, int off, int ks) {
    const char* a = base + off + ks * 8192;
    const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(a));
    const s16x4 v2 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(a + 1024));
    return __builtin_bit_cast(u16x8, __builtin_shufflevector(v1, v2, 0, 1, 2, 3, 4, 5, 6, 7));
  };

  f32x4 acc0[2][4][2], acc1[2][4][NJ1];
  u16x8 fa[2][4], fb0[2][2], fb1[2][NJ1];
  auto read_a = [&](int buf, int off) {
    const char* base = smem + buf * TC::BUF + off;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int i = 0; i < 4; ++i) { if constexpr (AKS) fa[ks][i] = frag_ks(base, a_off[i], ks); else fa[ks][i] = frag_kc(base, a_off[i], a_sw[i], ks); }
  };
  auto read_b0 = [&](int buf) {
    const char* base = smem + buf * TC::BUF + TC::OFF_B0;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int j = 0; j < 2; ++j) { if constexpr (BKS) fb0[ks][j] = frag_ks(base, b0_off[j], ks); else fb0[ks][j] = frag_kc(base, b0_off[j], b0_sw[j], ks); }
  };
  auto read_b1 = [&](int buf) {
    const char* base = smem + buf * TC::BUF + TC::OFF_B1;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int j = 0; j < NJ1; ++j) { if constexpr (BKS) fb1[ks][j] = frag_ks(base, b1_off[j], ks); else fb1[ks][j] = frag_kc(base, b1_off[j], b1_sw[j], ks); }
  };
  auto mma0 = [&](int mq) {
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc0[mq][i][j] = mfma16<F16>(fb0[ks][j], fa[ks][i], acc0[mq][i][j]);
    __builtin_amdgcn_s_setprio(0);
  };
  auto mma1 = [&](int mq) {
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < NJ1; ++j) acc1[mq][i][j] = mfma16<F16>(fb1[ks][j], fa[ks][i], acc1[mq][i][j]);
    __builtin_amdgcn_s_setprio(0);
  };
  auto sync_reads = [&]() {
    __builtin_amdgcn_s_barrier();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  auto end_phase = [&]() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
  };

  // K-tile T: quadrants (0,B0) (0,B1) (1,B1) (1,B0).  Staging order B1(T+1), A1(T+1), A0(T+2), B0(T+2), across tiles: in the last
  // two K-tiles "T+1" / "T+2" are K-tiles 0 and 1 of the block's next tile (HOOK switches the sources between phases 2 and 3).
  // Every slot is restaged at least two phases after its last read; at the K-tile boundary A0 and B0 (4 copies) stay in flight.
#define VTC_OG_KTILE(BUF, C1, K1, C2, K2, HOOK)                                     \
  {                                                                                 \
    read_b0(BUF);                                                                   \
    __builtin_amdgcn_sched_barrier(0);                                              \
    read_a(BUF, TC::OFF_A0);                                                        \
    if (C1) issue_b1((BUF) ^ 1, (K1));                                              \
    sync_reads();                                                                   \
    mma0(0);                                                                        \
    end_phase();                                                                    \
    read_b1(BUF);                                                                   \
    if (C1) issue_a(1, (BUF) ^ 1, (K1));                                            \
    sync_reads();                                                                   \
    mma1(0);                                                                        \
    end_phase();                                                                    \
    HOOK;                                                                           \
    read_a(BUF, TC::OFF_A1);                                                        \
    if (C2) issue_a(0, BUF, (K2));                                                  \
    sync_reads();                                                                   \
    mma1(1);                                                                        \
    end_phase();                                                                    \
    if (C2) {                                                                       \
      issue_b0(BUF, (K2));                                                          \
      asm volatile("s_waitcnt vmcnt(4)" ::: "memory");                              \
    } else {                                                                        \
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                              \
    }                                                                               \
    __builtin_amdgcn_s_barrier();                                                   \
    __builtin_amdgcn_sched_barrier(0);                                              \
    mma0(1);                                                                        \
    end_phase();                                                                    \
  }

  const unsigned G = gridDim.x, nunits = (unsigned)p.ntiles * (unsigned)p.splits;
  unsigned tl = blockIdx.x;
  {
    int pi, tm, tn, k0, k1;
    unit(xcd_remap(tl, nunits), pi, tm, tn, k0, k1);
    set_sources(pi, tm, tn);
    if constexpr (MULTI) repitch(pi);
    kt_base = k0;
    issue_a(0, 0, 0); issue_b0(0, 0); issue_b1(0, 0); issue_a(1, 0, 0);
    issue_a(0, 1, 1); issue_b0(1, 1);
  }
  bool first_tile = true;
  while (tl < nunits) {
    int pi, tile_m, tile_n, k0, k1;
    const unsigned ucur = xcd_remap(tl, nunits);
    unit(ucur, pi, tile_m, tile_n, k0, k1);
    nk_cur = k1 - k0;
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int j = 0; j < 2; ++j) acc0[a][i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < NJ1; ++j) acc1[a][i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
    if (first_tile) {
      asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      first_tile = false;
    }
    const unsigned tl_next = tl + G;
    const bool has_next = tl_next < nunits;
    if (wm == 1) __builtin_amdgcn_s_barrier();   // wave row 1 runs one barrier behind: one row computes while the other reads
    for (int t = 0; t + 2 < nk_cur; t += 2) {
      VTC_OG_KTILE(0, true, t + 1, true, t + 2, )
      VTC_OG_KTILE(1, true, t + 2, true, t + 3, )
    }
    VTC_OG_KTILE(0, true, nk_cur - 1, has_next, 0, if (has_next) {
      int pn; int tmn; int tnn; int kn; int kn1;
      unit(xcd_remap(tl_next, nunits), pn, tmn, tnn, kn, kn1);
      set_sources(pn, tmn, tnn);
      if constexpr (MULTI) repitch(pn);
      kt_base = kn;
    })
    VTC_OG_KTILE(1, has_next, 0, has_next, 1, )
    if (wm == 0) __builtin_amdgcn_s_barrier();
    tl = tl_next;

    // ---- epilogue.  Global accesses through descriptors of the tile: rows outside are dropped by the hardware, columns per lane.
    const OpProb& q = p.prob[pi];
    const int rows = min(256, q.M - tile_m * 256);
    const int n0 = EPI == OG_GATE ? tile_n * 128 : tile_n * BN;
    const int cols = q.N - n0, bcols = q.Nb - n0;                // columns left from the tile's first; those that have a bias
    constexpr int W1 = 4 * NJ1;
    const int c0 = wn * 32 + 8 * fq;                             // columns of the tile: B0 group, B1 group
    const int c1 = EPI == OG_GATE ? c0 : 128 + wn * (16 * NJ1) + W1 * fq;
    auto tile_rsrc = [&](const void* base, long long ld, int es) {
      const char* b = (const char*)base + ((long long)tile_m * 256 * ld + n0) * es;
      return __builtin_amdgcn_make_buffer_rsrc((void*)b, 0, (int)(((long long)(rows - 1) * ld + cols) * es), 0x00020000);
    };
    auto row_of = [&](int g) { return (g >> 2) * 128 + wm * 64 + (g & 3) * 16 + fr; };
    // N consecutive values of row r from column c: one store where rows start aligned, else one by one
    auto store16 = [&](__amdgpu_buffer_rsrc_t rs, long long ld, int vec, int r, int c, const float* v, auto count) {
      constexpr int N = decltype(count)::value;
      const unsigned off = (unsigned)((r * (int)ld + c) * 2);
      if (vec) {
        const unsigned o = (r < rows && c < cols) ? off : OOB;
        if constexpr (N == 8)
          __builtin_amdgcn_raw_buffer_store_b128(u32x4{pack2<F16>(v[0], v[1]), pack2<F16>(v[2], v[3]), pack2<F16>(v[4], v[5]), pack2<F16>(v[6], v[7])}, rs, o, 0, 0);
        else {
          typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
          __builtin_amdgcn_raw_buffer_store_b64(u32x2{pack2<F16>(v[0], v[1]), pack2<F16>(v[2], v[3])}, rs, o, 0, 0);
        }
      } else {
#pragma unroll
        for (int k = 0; k < N; ++k)
          __builtin_amdgcn_raw_buffer_store_b16(to_h16<F16>(v[k]), rs, (r < rows && c + k < cols) ? off + 2 * k : OOB, 0, 0);
      }
    };
    using I8 = std::integral_constant<int, 8>;
    using IW1 = std::integral_constant<int, W1>;
    float v0[8], v1[W1];
    auto take = [&](int g) {
      const int mq = g >> 2, i = g & 3;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) v0[4 * j + r] = acc0[mq][i][j][r];
#pragma unroll
      for (int j = 0; j < NJ1; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) v1[4 * j + r] = acc1[mq][i][j][r];
    };
    if constexpr (EPI == OG_PLAIN) {
      float b0[8], b1[W1];
#pragma unroll
      for (int k = 0; k < 8; ++k) b0[k] = c0 + k < bcols ? op_bias(p.bias, n0 + c0 + k, p.bias_f32, F16) : 0.f;
#pragma unroll
      for (int k = 0; k < W1; ++k) b1[k] = c1 + k < bcols ? op_bias(p.bias, n0 + c1 + k, p.bias_f32, F16) : 0.f;
      const __amdgpu_buffer_rsrc_t rc = tile_rsrc(q.c, q.ldc, 2);
#pragma unroll
      for (int g = 0; g < 8; ++g) {
        take(g);
#pragma unroll
        for (int k = 0; k < 8; ++k) v0[k] += b0[k];
#pragma unroll
        for (int k = 0; k < W1; ++k) v1[k] += b1[k];
        store16(rc, q.ldc, q.cvec, row_of(g), c0, v0, I8{});
        store16(rc, q.ldc, q.cvec, row_of(g), c1, v1, IW1{});
      }
    } else if constexpr (EPI == OG_PART) {
      // partial s of the problem: [M][N] fp32 with the pitch ldc (a multiple of 8)
      const int s = (int)(ucur % (unsigned)p.splits);
      const __amdgpu_buffer_rsrc_t rc = tile_rsrc((const float*)q.c + s * p.split_stride, q.ldc, 4);
#pragma unroll
      for (int g = 0; g < 8; ++g) {
        take(g);
        const int r = row_of(g);
#pragma unroll
        for (int h = 0; h < 2; ++h)
          __builtin_amdgcn_raw_buffer_store_b128(u32x4{__float_as_uint(v0[4 * h]), __float_as_uint(v0[4 * h + 1]), __float_as_uint(v0[4 * h + 2]), __float_as_uint(v0[4 * h + 3])},
                                                 rc, (r < rows && c0 + 4 * h < cols) ? (unsigned)((r * (int)q.ldc + c0 + 4 * h) * 4) : OOB, 0, 0);
#pragma unroll
        for (int h = 0; h < NJ1; ++h)
          __builtin_amdgcn_raw_buffer_store_b128(u32x4{__float_as_uint(v1[4 * h]), __float_as_uint(v1[4 * h + 1]), __float_as_uint(v1[4 * h + 2]), __float_as_uint(v1[4 * h + 3])},
                                                 rc, (r < rows && c1 + 4 * h < cols) ? (unsigned)((r * (int)q.ldc + c1 + 4 * h) * 4) : OOB, 0, 0);
      }
    } else if constexpr (EPI == OG_GATE) {
      if constexpr (NJ1 == 2) {
        float bg[8], bu[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          bg[k] = c0 + k < bcols ? op_bias(p.bias, n0 + c0 + k, p.bias_f32, F16) : 0.f;
          bu[k] = c0 + k < bcols ? op_bias(p.bias2, n0 + c0 + k, p.bias_f32, F16) : 0.f;
        }
        const __amdgpu_buffer_rsrc_t rh = tile_rsrc(q.c, p.ldg, 2);
        auto run = [&](auto act) {
          constexpr int ACT = decltype(act)::value;
#pragma unroll
          for (int g = 0; g < 8; ++g) {
            take(g);
            float h[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              v0[k] += bg[k];
              v1[k] += bu[k];
              h[k] = op_act<ACT, false>(v0[k]) * v1[k];
            }
            if (p.g) {
              store16(tile_rsrc(p.g, p.ldg, 2), p.ldg, 1, row_of(g), c0, v0, I8{});
              store16(tile_rsrc(p.u, p.ldg, 2), p.ldg, 1, row_of(g), c0, v1, I8{});
            }
            store16(rh, p.ldg, 1, row_of(g), c0, h, I8{});
          }
        };
        if (p.act == ACT_GELU) run(std::integral_constant<int, ACT_GELU>{});
        else if (p.act == ACT_SILU) run(std::integral_constant<int, ACT_SILU>{});
        else if (p.act == ACT_SIGMOID) run(std::integral_constant<int, ACT_SIGMOID>{});
        else run(std::integral_constant<int, ACT_NONE>{});
      }
    } else {   // OG_DGATE
      if constexpr (NJ1 == 2) {
        const __amdgpu_buffer_rsrc_t rg = tile_rsrc(p.g, p.ldg, 2), ru = tile_rsrc(p.u, p.ldg, 2), rdg = tile_rsrc(p.dg, p.ldg, 2),
                                     rdu = tile_rsrc(p.du, p.ldg, 2);
        auto run = [&](auto act) {
          constexpr int ACT = decltype(act)::value;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int c = half ? c1 : c0;
            float sg[8], su[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) sg[k] = su[k] = 0.f;
#pragma unroll
            for (int g0 = 0; g0 < 8; g0 += 4) {
              __builtin_amdgcn_sched_barrier(0);   // the loads of four row groups at a time: all sixteen would not fit the registers
              u32x4 xg[4], xu[4];
#pragma unroll
              for (int gg = 0; gg < 4; ++gg) {
                const int r = row_of(g0 + gg);
                const unsigned off = (r < rows && c < cols) ? (unsigned)((r * (int)p.ldg + c) * 2) : OOB;
                xg[gg] = __builtin_amdgcn_raw_buffer_load_b128(rg, off, 0, 0);
                xu[gg] = __builtin_amdgcn_raw_buffer_load_b128(ru, off, 0, 0);
              }
#pragma unroll
              for (int gg = 0; gg < 4; ++gg) {
                const int mq = g0 >> 2, i = gg, r = row_of(g0 + gg);
                float dg[8], du[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                  const float dh = half ? acc1[mq][i][k >> 2][k & 3] : acc0[mq][i][k >> 2][k & 3];
                  const float gv = from_h16<F16>((h16)(k & 1 ? xg[gg][k >> 1] >> 16 : xg[gg][k >> 1] & 0xffffu));
                  const float uv = from_h16<F16>((h16)(k & 1 ? xu[gg][k >> 1] >> 16 : xu[gg][k >> 1] & 0xffffu));
                  float a, d;
                  op_act_grad<ACT, false>(gv, a, d);
                  dg[k] = dh * uv * d;
                  du[k] = dh * a;
                  sg[k] += dg[k];
                  su[k] += du[k];
                }
                store16(rdg, p.ldg, 1, r, c, dg, I8{});
                store16(rdu, p.ldg, 1, r, c, du, I8{});
              }
            }
            if (p.colsum) {   // rows outside contributed 0: dh is 0 there
#pragma unroll
              for (int k = 0; k < 8; ++k) {
#pragma unroll
                for (int o = 1; o < 16; o <<= 1) { sg[k] += __shfl_xor(sg[k], o); su[k] += __shfl_xor(su[k], o); }
              }
              if (fr == 0 && c < cols) {
                float* dst = p.colsum + (long long)(tile_m * 2 + wm) * p.ldg + n0 + c;
                const long long second = (long long)q.tiles_m * 2 * p.ldg;
#pragma unroll
                for (int k = 0; k < 8; ++k) { dst[k] = sg[k]; dst[second + k] = su[k]; }
              }
            }
          }
        };
        if (p.act == ACT_GELU) run(std::integral_constant<int, ACT_GELU>{});
        else if (p.act == ACT_SILU) run(std::integral_constant<int, ACT_SILU>{});
        else if (p.act == ACT_SIGMOID) run(std::integral_constant<int, ACT_SIGMOID>{});
        else run(std::integral_constant<int, ACT_NONE>{});
      }
    }
  }
#undef VTC_OG_KTILE
}

}  // namespace vtc
