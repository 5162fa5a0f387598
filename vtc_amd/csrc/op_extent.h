// Sizes of the operand windows that op_gemm.hip.h fetches through, as plain functions of whole numbers: host code can walk a product
// of any size with them (tests/op_extent_walk.cpp).
//
// An operand stored with the contraction index along its rows ("KS") is fetched in half-tiles of at most 128 columns, 64 k-rows at a
// time.  Its descriptor starts at the next k-row and ends with the operand's last one, so k-rows and columns that do not exist read
// as zero: `left` k-rows (at most kRowsAhead of them) at the pitch, the last one cut behind the half-tile's columns.  `left` falls by
// 64 with every K-tile and passes zero: where a tile's second half lies behind the matrix it starts there, and K-tiles follow that
// only the other operand or the other segment needs.  All of those windows are empty.
#pragma once

#if defined(__HIPCC__)
#define VTC_HD __host__ __device__ __forceinline__
#else
#define VTC_HD inline
#endif

namespace vtc {

// k-rows a descriptor of a K-strided half-tile spans: 64, and the most that 128 columns can run over at the least pitch of 8
constexpr int kRowsAhead = 192;

// bytes of the last k-row less a pitch (cols: columns left from the half-tile's first one; most: columns of a half-tile)
VTC_HD int ks_end(int cols, int most, int ld) {
  const int c = cols < most ? cols : most;
  return (((c > 0 ? c : 0) + 7) & ~7) * 2 - ld * 2;
}
VTC_HD int ks_left(int cols, int K, int k0) { return cols > 0 ? K - k0 : 0; }
// bytes of the window; with left held in 0..kRowsAhead the product stays below 2^29 (pitches of at most 2^20 elements)
VTC_HD int ks_bytes(int left, int ld2, int end) {
  const int rows = left < 0 ? 0 : left < kRowsAhead ? left : kRowsAhead;
  const int n = rows * ld2 + end;
  return n > 0 ? n : 0;
}

}  // namespace vtc
