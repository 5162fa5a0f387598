// Sizes of the operand windows that op_gemm.hip.h fetches through, as plain functions of whole numbers: host code can walk a product
// of any size with them (tests/op_extent_walk.cpp).
//
// An operand stored with the contraction index along its rows ("KS") is fetched in half-tiles of at most 128 columns, 64 k-rows at a
// time.  Its descriptor starts at the next k-row and ends with the operand's last one, so k-rows and columns that do not exist read
// as zero: `left` k-rows (at most kRowsAhead of them) at the pitch, the last one cut behind the half-tile's columns.  `left` falls by
// 64 with every K-tile; of an operand that is there it ends within two K-tiles behind zero.  A half-tile that lies wholly behind the matrix is
// fetched all the same, for as many K-tiles as the product has, and each of its windows has to be empty: it starts with as many rows as
// an int holds, which no product uses up, and ends in front of the first.  (Left counting down from 0, rows x pitch would wrap to
// a window of 2 GiB; holding it at 0 in the K loop takes 7 us more of a 575 us training step, 15968 rows x 768 x 2048.)
#pragma once

#if defined(__HIPCC__)
#define VTC_HD __host__ __device__ __forceinline__
#else
#define VTC_HD inline
#endif

namespace vtc {

// k-rows a descriptor of a K-strided half-tile spans: 64, and the most that 128 columns can run over at the least pitch of 8
constexpr int kRowsAhead = 192;

constexpr int kMaxPitch = 1 << 20;   // elements between rows of a matrix (of more than one row)

// bytes of the last k-row less a pitch (cols: columns left from the half-tile's first one; most: columns of a half-tile)
VTC_HD int ks_end(int cols, int most, int ld) {
  const int c = ((cols < most ? cols : most) + 7) & ~7;
  return cols > 0 ? c * 2 - ld * 2 : -kRowsAhead * 2 * kMaxPitch;
}
VTC_HD int ks_left(int cols, int K, int k0) { return cols > 0 ? K - k0 : 0x7fffffff; }
// bytes of the window, below 2^29
VTC_HD int ks_bytes(int left, int ld2, int end) {
  const int n = (left < kRowsAhead ? left : kRowsAhead) * ld2 + end;
  return n > 0 ? n : 0;
}

}  // namespace vtc
