// Gated feed-forward block: g = x Wg^T + bg, u = x Wu^T + bu, h = act(g) u, y = h Wd^T + bd, and its gradients
//   dh = dy Wd, dg = dh u act'(g), du = dh act(g), dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x, dWd = dy^T h.
//
// Both projections, the activation and the product are one kernel: a tile holds the same columns of W_gate (first half) and W_up
// (second half), so a lane's two accumulators are g and u of the same elements and only h leaves the chip (g and u as well when a
// backward pass will want them).  Backward: dh never exists in memory (its tile turns into dg and du in the epilogue).
// Rounding: h, dg and du are stored in the operands' 16-bit type, since they are operands of the next matrix product; what the
// forward pass keeps for the backward one (s = u act'(g) and a = act(g), so that no activation is computed twice) has 24 bits;
// every sum is fp32 (column sums are joined in fp64).
//
// Few rows (at most 32: single frames, live streams) are bound by reading the weights once, and by latency: skinny_kernel
// below.  Everything else runs on op_gemm_kernel or, where that would leave CUs idle, op_small_kernel.
#pragma once
#include "common.hip.h"
#include "op_act.hip.h"
#include "op_gemm.hip.h"

namespace vtc {

// rows x cols of src, zero-filled to dcols columns (a multiple of 8): operands whose rows are not made of aligned 16-byte pieces.
// One launch for all of a call's (blockIdx.y): a copy each took 3 us, nine of them 26 of the 85 us of a step at 1237 x 389 x 1031.
struct PadJob { const h16* src; h16* dst; long long pitch, rows; int cols, dcols; };
struct PadParams { PadJob j[5]; };
__global__ __launch_bounds__(256) void pad_copy_kernel(PadParams p) {
  const PadJob& j = p.j[blockIdx.y];
  const int pieces = j.dcols / 8;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < j.rows * pieces; i += (long long)gridDim.x * 256) {
    const long long r = i / pieces;
    const int c = (int)(i - r * pieces) * 8;
    u16x8 v;
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = c + k < j.cols ? j.src[r * j.pitch + c + k] : (h16)0;
    *(u16x8*)(j.dst + r * j.dcols + c) = v;
  }
}

// column sums of kColRows rows (dy -> partial sums of d b_down); part [blocks of rows][pitch].  red: 4 x 512 floats
constexpr int kColRows = 64;
struct ColSumParams { const h16* x; long long ld, rows; float* part; int pitch, cols, row_blocks, blocks; };   // blocks: row_blocks x 512 columns each
template <bool F16>
__device__ __forceinline__ void colsum_tile(const ColSumParams& p, unsigned block, float (*red)[512]) {
  const int rb = (int)(block % (unsigned)p.row_blocks), cb = (int)(block / (unsigned)p.row_blocks);
  const int v = cb * 64 + (threadIdx.x & 63), w = threadIdx.x >> 6;
  const long long r0 = (long long)rb * kColRows, r1 = min(p.rows, r0 + kColRows);
  float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (v * 8 < p.cols)
#pragma unroll 8
    for (long long r = r0 + w; r < r1; r += 4) {
      const u16x8 f = *(const u16x8*)(p.x + r * p.ld + v * 8);
#pragma unroll
      for (int k = 0; k < 8; ++k) s[k] += from_h16<F16>(f[k]);
    }
#pragma unroll
  for (int k = 0; k < 8; ++k) red[w][(threadIdx.x & 63) * 8 + k] = s[k];
  __syncthreads();
  if (w == 0 && v * 8 < p.pitch)
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int i = threadIdx.x * 8 + k;
      p.part[(long long)rb * p.pitch + v * 8 + k] = (red[0][i] + red[1][i]) + (red[2][i] + red[3][i]);
    }
}
template <bool F16>
__global__ __launch_bounds__(256) void colsum_kernel(const ColSumParams p) {
  __shared__ float red[4][512];
  colsum_tile<F16>(p, blockIdx.x, red);
}

// The rest of a small backward pass behind dg and du in one launch: the weights' gradients (the longest first), dx, dy's column sums.
// They do not depend on each other; each alone leaves CUs idle and costs a launch.  Backward with biases, launched apart / together:
// 512 rows, 768 x 2048, 59 / 44 us; 2048 rows 100 / 77; 1237 x 389 x 1031 with its forward 72 / 63.
struct SmallGradsParams { OpGemmParams w, dx; ColSumParams c; unsigned w_blocks, dx_blocks; };
template <bool F16, int DX_EPI>
__global__ __launch_bounds__(256, 2) void small_grads_kernel(const SmallGradsParams p) {
  __shared__ __attribute__((aligned(16))) char smem[3 * kOsStage];
  if (blockIdx.x < p.w_blocks) op_small_tile<F16, true, true, OG_PART>(p.w, blockIdx.x, p.w_blocks, smem);
  else if (blockIdx.x - p.w_blocks < p.dx_blocks) op_small_tile<F16, false, true, DX_EPI>(p.dx, blockIdx.x - p.w_blocks, p.dx_blocks, smem);
  else colsum_tile<F16>(p.c, blockIdx.x - p.w_blocks - p.dx_blocks, (float (*)[512])smem);
}

// What is left of a pass once its products are there, in one launch (blockIdx.y): K-split partials (+ bias) -> 16-bit results, and
// partial column sums -> bias gradients, out[c] = sum over n partial rows, in order, fp64 (16 slices of rows by 16 columns a block).
struct ColReduce { const float* part; void* out; long long n; int pitch, cols; };
struct SplitReduce { const float* part; h16* out; long long ldo, pitch, rows, stride; int splits, cols, vec; const void* bias; };
struct ReduceParams { SplitReduce r[4]; ColReduce c[3]; int nr, nc, bias_f32; };   // bias_f32: biases and their gradients are fp32
template <bool F16> __device__ __forceinline__ void col_reduce(const ColReduce& q, int out_f32) {
  __shared__ double red[16][16];
  const int c = blockIdx.x * 16 + (threadIdx.x & 15), w = threadIdx.x >> 4;
  if ((int)blockIdx.x * 16 >= q.cols) return;
  double s = 0.0;
  if (c < q.cols)
#pragma unroll 8
    for (long long i = w; i < q.n; i += 16) s += (double)q.part[i * q.pitch + c];
  red[w][threadIdx.x & 15] = s;
  __syncthreads();
  if (w || c >= q.cols) return;
  for (int i = 1; i < 16; ++i) s += red[i][threadIdx.x];
  const float v = (float)s;
  if (out_f32) ((float*)q.out)[c] = v;
  else ((h16*)q.out)[c] = to_h16<F16>(v);
}
template <bool F16>
__global__ __launch_bounds__(256) void reduce_kernel(const ReduceParams p) {
  if ((int)blockIdx.y >= p.nr) { col_reduce<F16>(p.c[blockIdx.y - p.nr], p.bias_f32); return; }
  const SplitReduce& q = p.r[blockIdx.y];
  const long long pieces = q.pitch / 4;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < q.rows * pieces; i += (long long)gridDim.x * 256) {
    const long long r = i / pieces;
    const int c = (int)(i - r * pieces) * 4;
    if (c >= q.cols) continue;
    const float* src = q.part + r * q.pitch + c;
    float4 s = *(const float4*)src;
    for (int k = 1; k < q.splits; ++k) {
      const float4 t = *(const float4*)(src + k * q.stride);
      s.x += t.x; s.y += t.y; s.z += t.z; s.w += t.w;
    }
    if (q.bias) {
      s.x += op_bias(q.bias, c, p.bias_f32, F16);
      if (c + 1 < q.cols) s.y += op_bias(q.bias, c + 1, p.bias_f32, F16);
      if (c + 2 < q.cols) s.z += op_bias(q.bias, c + 2, p.bias_f32, F16);
      if (c + 3 < q.cols) s.w += op_bias(q.bias, c + 3, p.bias_f32, F16);
    }
    h16* o = q.out + r * q.ldo + c;
    if (q.vec) {
      typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
      *(u32x2*)o = u32x2{pack2<F16>(s.x, s.y), pack2<F16>(s.z, s.w)};
    } else {
      const float v[4] = {s.x, s.y, s.z, s.w};
      for (int k = 0; k < 4 && c + k < q.cols; ++k) o[k] = to_h16<F16>(v[k]);
    }
  }
}

// ---- few rows: C[M <= 16 MT][N] = A W^T.  A block owns 16 columns, its 8 waves take every 8th K step of 32 straight from global
// memory (the weights are read once, by nobody else), their partial tiles meet in LDS.  MFMA computes C^T: lane (fr, fq) holds
// row fr of A and columns 4 fq .. + 4.  Bound: latency; one row, 768 x 2048: 4.8 us for gate and up (6.3 MB), 4.8 us for down.
struct SkinnyParams {
  const h16 *x, *w0, *w1;     // w1: W_up (GATE)
  long long ldx, ldw;
  int M, K, N, Nb;            // N: columns written (padding included), Nb: rows of w
  const void *b0, *b1;
  int bias_f32, act;
  h16* out;
  Saved24 s, a;               // GATE: kept for the backward pass (s.hi null: nothing is)
  long long ldo;
};
template <bool F16, int MT, bool GATE>
__global__ __launch_bounds__(512) void skinny_kernel(const SkinnyParams p) {
  constexpr int NW = GATE ? 2 : 1;
  __shared__ float part[8][NW * MT * 256];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int fr = lane & 15, fq = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const int rows_w = min(16, p.Nb - n0);
  constexpr unsigned OOB = 0x80000000u;
  auto rsrc = [&](const h16* b, long long ld, int rows) {
    return __builtin_amdgcn_make_buffer_rsrc((void*)b, 0, rows > 0 ? (int)(((rows - 1) * ld + ((p.K + 7) & ~7)) * 2) : 0, 0x00020000);
  };
  const __amdgpu_buffer_rsrc_t r0 = rsrc(p.w0 + n0 * p.ldw, p.ldw, rows_w), r1 = GATE ? rsrc(p.w1 + n0 * p.ldw, p.ldw, rows_w) : r0;
  const __amdgpu_buffer_rsrc_t rx = rsrc(p.x, p.ldx, p.M);
  const unsigned vw = (unsigned)(fr * (int)p.ldw * 2), vx = (unsigned)(fr * (int)p.ldx * 2), stepx = (unsigned)(16 * (int)p.ldx * 2);
  f32x4 acc[NW][MT];
#pragma unroll
  for (int w = 0; w < NW; ++w)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[w][m] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int steps = (p.K + 31) / 32;
  constexpr int D = 4;                          // K steps in flight; steps behind the end read as zero
  for (int s0 = wave; s0 < steps; s0 += 8 * D) {
    u16x8 a[D][NW], b[D][MT];
#pragma unroll
    for (int j = 0; j < D; ++j) {
      const int k = (s0 + 8 * j) * 32 + fq * 8;
      const unsigned ko = k < p.K ? (unsigned)k * 2u : OOB;   // OOB + any row offset stays out of range (below 2^30 each)
      a[j][0] = __builtin_bit_cast(u16x8, __builtin_amdgcn_raw_buffer_load_b128(r0, vw + ko, 0, 0));
      if constexpr (GATE) a[j][1] = __builtin_bit_cast(u16x8, __builtin_amdgcn_raw_buffer_load_b128(r1, vw + ko, 0, 0));
#pragma unroll
      for (int m = 0; m < MT; ++m) b[j][m] = __builtin_bit_cast(u16x8, __builtin_amdgcn_raw_buffer_load_b128(rx, vx + m * stepx + ko, 0, 0));
    }
#pragma unroll
    for (int j = 0; j < D; ++j)
#pragma unroll
      for (int w = 0; w < NW; ++w)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[w][m] = mfma16<F16>(a[j][w], b[j][m], acc[w][m]);
  }
#pragma unroll
  for (int w = 0; w < NW; ++w)
#pragma unroll
    for (int m = 0; m < MT; ++m) *(f32x4*)&part[wave][(w * MT + m) * 256 + fr * 16 + fq * 4] = acc[w][m];   // [row][column]
  __syncthreads();
  for (int i = threadIdx.x; i < MT * 256; i += 512) {
    const int r = i >> 4, c = i & 15, col = n0 + c;
    float v0 = 0.f, v1 = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      v0 += part[w][i];
      if constexpr (GATE) v1 += part[w][MT * 256 + i];
    }
    if (r >= p.M || col >= p.N) continue;
    if (col < p.Nb) v0 += op_bias(p.b0, col, p.bias_f32, F16);
    if constexpr (GATE) {
      if (col < p.Nb) v1 += op_bias(p.b1, col, p.bias_f32, F16);
      float a = v0, d = 1.f;
      if (p.s.hi) {
        if (p.act == ACT_GELU) op_act_grad<ACT_GELU, false>(v0, a, d);
        else if (p.act == ACT_SILU) op_act_grad<ACT_SILU, false>(v0, a, d);
        else if (p.act == ACT_SIGMOID) op_act_grad<ACT_SIGMOID, false>(v0, a, d);
        const unsigned bs = __float_as_uint(v1 * d) + 0x80u, ba = __float_as_uint(a) + 0x80u;   // see OpTile::store24
        const long long at = r * p.ldo + col;
        p.s.hi[at] = (unsigned short)(bs >> 16); p.s.lo[at] = (unsigned char)(bs >> 8);
        p.a.hi[at] = (unsigned short)(ba >> 16); p.a.lo[at] = (unsigned char)(ba >> 8);
      } else {
        if (p.act == ACT_GELU) a = op_act<ACT_GELU, false>(v0);
        else if (p.act == ACT_SILU) a = op_act<ACT_SILU, false>(v0);
        else if (p.act == ACT_SIGMOID) a = op_act<ACT_SIGMOID, false>(v0);
      }
      v0 = a * v1;
    }
    p.out[r * p.ldo + col] = to_h16<F16>(v0);
  }
}

}  // namespace vtc
