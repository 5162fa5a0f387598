// Walks the operand windows of vtc_amd/csrc/op_extent.h through products as op_gemm_kernel and op_small_tile do, and compares each
// with the operand's extent in 64 bits.  One product per line of standard input:
//   K ld columns col0 most tiles segments      (tiles: K-tiles over all segments, starting at k = 0)
// Ends with status 1 at the first window that leaves the operand or misses a part of it that a tile needs.
#include <algorithm>
#include <cstdio>

#include "op_extent.h"

int main() {
  long long K, ld, columns, col0, most, tiles, segments, lines = 0;
  while (scanf("%lld %lld %lld %lld %lld %lld %lld", &K, &ld, &columns, &col0, &most, &tiles, &segments) == 7) {
    ++lines;
    const long long cols = columns - col0, c8 = (std::min(std::max(cols, 0ll), most) + 7) / 8 * 8;
    const int end = vtc::ks_end((int)cols, (int)most, (int)ld), start = vtc::ks_left((int)cols, (int)K, 0);
    int left = start, segment = 0;
    long long k = 0;   // the window's first k-row
    for (long long t = 0; t < tiles; ++t) {
      if (segments == 2 && left <= 0 && segment == 0) { left = start; segment = 1; k = 0; }
      const long long got = vtc::ks_bytes(left, (int)(2 * ld), end);
      const long long rows = cols > 0 ? std::max(K - k, 0ll) : 0;
      const long long exist = rows > 0 ? (rows - 1) * 2 * ld + 2 * c8 : 0;          // what there is from the window's start on
      const long long need = rows > 0 ? (std::min(rows, 64ll) - 1) * 2 * ld + 2 * c8 : 0;
      if (got < need || got > exist) {
        printf("K %lld, pitch %lld, columns %lld from %lld: K-tile %lld has a window of %lld bytes, needed %lld, existing %lld\n", K, ld, columns, col0, t, got, need, exist);
        return 1;
      }
      left -= 64;
      k += 64;
    }
  }
  printf("%lld products walked\n", lines);
  return 0;
}
