// Group norm with an activation on channel-last rows (N, L, C), forward and backward.
//
// Mathematics, per sample n and group g of C / G neighbouring channels, over the real rows l < length[n] (all L without lengths):
//   mean, rstd = 1 / sqrt(var + eps);  z = (x - mean) rstd w_c + b_c;  y = act(z).
//   backward: dz = dy act'(z);  db_c = sum dz;  dw_c = sum dz xhat (over n and l);
//   dx = rstd (w_c dz - (A + xhat B) / M),  A = sum w_c dz,  B = sum w_c dz xhat over the group, M = its element count.
// Rows at and behind length[n] are not read; y and dx are zero there.  A sample of length 0 has mean = rstd = 0.
//
// Two forms.  Samples that fit a block's registers are read once (gn_slab_kernel, gn_bwd_slab_kernel); everything else - long or odd
// samples, wide groups, strides that are no whole vectors - streams: statistics per row block, merge, elementwise pass, in which x (and
// dy) are read a second time, last rows first, since those are still in the last-level cache.  Bound: memory and the activation's
// vector instructions (about 25 issue slots of an element for GELU, 83 us of 131 M elements).  64 x 3999 x 512 f16 with GELU (524 MB,
// 105 us at a copy's rate) streams in 64 (statistics) + 5 + 104 us, 186 with its launches.  Figures of both forms: kGnSlabVectors in vtc_ops.hip.
// 5 x 1531 x 201 fp32 (streaming, 4-byte accesses): statistics 5, elementwise 11, backward sums 7, merges 4 + 3, dx 7 us.
//
// Statistics: every partial is (mean, M2 = sum of squared distances from it) and partials merge about their common mean, so a mean
// that is large against the spread does not cancel; inside a thread the sums are of x - x_first (the row block's first row, per
// channel), in fp32 over at most a few hundred rows; merges across row blocks are fp64.  All orders are fixed, no atomics:
// results are bit-reproducible.
#pragma once
#include "common.hip.h"
#include "op_act.hip.h"
#include "rotary.hip.h"   // OpVec: 1..16-byte vector access with conversion

namespace vtc {

constexpr int kGnMaxChannels = 8192;

struct GnParams {
  const void *x, *dy;
  void* out;                    // y (forward) or dx (backward)
  long long xn, xl, dn, dl, on, ol;   // element strides of sample and row (channels are contiguous)
  const void *w, *b;            // affine per channel, may be null
  const int* length;            // [N] or null
  float *mean, *rstd;           // [N][G]
  float* part;                  // statistics: [N][chunks][G][2] (mean, M2); backward sums: [N][chunks][C][2]
  double* sums;                 // backward: [N][C][2] sums over rows
  double* gsums;                // backward, streaming: [N][G][2] (A / M, B / M)
  void *dw, *db;                // gradients of the affine, may be null
  long long N, L;
  int C, G, cpg, cv, rows, chunks;   // cv = C / VEC; rows per row block (chunk) of the sums, row blocks per sample
  int arows, achunks;           // the same of the elementwise pass, which may follow the number of samples
  int merge_here;               // forward: the elementwise pass merges the row blocks' partials itself (few of them)
  int cvb;                      // whole-sample kernels: 16-byte channel vectors of a block
  int affine_f32;               // w, b, dw, db are fp32 (else the tensors' type)
  float eps;
};

template <int DT> __device__ __forceinline__ float gn_param(const void* p, int i, int f32, float none) {
  if (!p) return none;
  return f32 ? ((const float*)p)[i] : op_load<DT>(((const typename OpType<DT>::T*)p)[i]);
}
__device__ __forceinline__ long long gn_length(const GnParams& p, long long n) {
  if (!p.length) return p.L;
  const long long l = p.length[n];
  return l < 0 ? 0 : (l < p.L ? l : p.L);
}

// ---- (mean, M2) of every group over one block of rows.  Threads walk channel vectors (fastest) and rows.
template <int DT, int VEC>
__global__ __launch_bounds__(256) void gn_stats_kernel(const GnParams p) {
  typedef typename OpType<DT>::T T;
  extern __shared__ float sh[];   // per channel: mean and M2 of the row block; in front, the row-parallel partial sums
  const long long n = blockIdx.x / (unsigned)p.chunks;
  const int chunk = (int)(blockIdx.x % (unsigned)p.chunks);
  const long long len = gn_length(p, n), r0 = (long long)chunk * p.rows;
  const int rows = (int)max(0ll, min((long long)p.rows, len - r0));
  float2* out = (float2*)p.part + (n * p.chunks + chunk) * p.G;
  if (rows == 0) return;   // finalize never reads the partial of an empty row block
  const T* x = (const T*)p.x + n * p.xn + r0 * p.xl;
  float* ch_mean = sh;
  float* ch_m2 = sh + p.C;
  float* red = sh + 2 * p.C;   // [256][2 * VEC]
  const int lanes = min(p.cv, 256);           // channel vectors side by side
  const int rp = 256 / lanes;                 // rows side by side
  const int tc = threadIdx.x % lanes, tr = threadIdx.x / lanes;
  for (int v0 = 0; v0 < p.cv; v0 += 256) {
    const int v = v0 + tc;
    const bool on = tr < rp && v < p.cv;
    float first[VEC], s[VEC], q[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) s[k] = q[k] = first[k] = 0.f;
    if (on) {
      const T* src = x + (long long)v * VEC;
      OpVec<DT, VEC>::load(src, first);
#pragma unroll 8
      for (int r = tr; r < rows; r += rp) {
        float f[VEC];
        OpVec<DT, VEC>::load(src + r * p.xl, f);
#pragma unroll
        for (int k = 0; k < VEC; ++k) { const float d = f[k] - first[k]; s[k] += d; q[k] = fmaf(d, d, q[k]); }
      }
    }
    if (rp > 1) {   // add the row-parallel threads of a channel vector (they share `first`)
#pragma unroll
      for (int k = 0; k < VEC; ++k) { red[threadIdx.x * 2 * VEC + k] = s[k]; red[threadIdx.x * 2 * VEC + VEC + k] = q[k]; }
      __syncthreads();
      if (on && tr == 0)
        for (int o = 1; o < rp; ++o)
#pragma unroll
          for (int k = 0; k < VEC; ++k) {
            s[k] += red[(o * lanes + tc) * 2 * VEC + k];
            q[k] += red[(o * lanes + tc) * 2 * VEC + VEC + k];
          }
    }
    if (on && tr == 0) {
      const float inv = 1.f / (float)rows;
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        const float m = s[k] * inv;
        ch_mean[v * VEC + k] = first[k] + m;
        ch_m2[v * VEC + k] = fmaxf(fmaf(-s[k], m, q[k]), 0.f);
      }
    }
    __syncthreads();
  }
  // channels -> groups: `w` neighbouring lanes per group
  int w = 1;
  while (w < 64 && w < p.cpg) w <<= 1;
  const int sub = threadIdx.x & (w - 1);
  for (int g0 = 0; g0 < p.G; g0 += 256 / w) {   // uniform trip count: every lane takes part in the shuffles
    const int g = g0 + threadIdx.x / w;
    float m = 0.f, m2 = 0.f;
    if (g < p.G) for (int c = sub; c < p.cpg; c += w) m += ch_mean[g * p.cpg + c];
    for (int o = w >> 1; o > 0; o >>= 1) m += __shfl_xor(m, o);
    m /= (float)p.cpg;
    if (g < p.G)
      for (int c = sub; c < p.cpg; c += w) {
        const float d = ch_mean[g * p.cpg + c] - m;
        m2 += fmaf(d * (float)rows, d, ch_m2[g * p.cpg + c]);
      }
    for (int o = w >> 1; o > 0; o >>= 1) m2 += __shfl_xor(m2, o);
    if (g < p.G && sub == 0) out[g] = make_float2(m, m2);
  }
}

// ---- merge the row blocks of a sample: 16 groups x 16 threads, thread i takes row blocks i, i + 16, ..  First the mean, then the squared
// distances from it, in fp64: one division per group (Chan's formula pairwise takes two per partial: 21 us instead of 5 for 64 x 3999 rows in
// 32 groups).
__device__ __forceinline__ double gn_slices(double v, double (*sh)[16], int slice, int in) {   // sum over the 16 threads of a group, in a tree
  __syncthreads();
  sh[slice][in] = v;
  __syncthreads();
  for (int h = 8; h > 0; h >>= 1) {
    if (slice < h) sh[slice][in] += sh[slice + h][in];
    __syncthreads();
  }
  return sh[0][in];
}
// mean and rstd of 16 groups from g0 on, by a block of 256; stat: [16] results for the block
__device__ __forceinline__ void gn_finalize(const GnParams& p, long long n, int g0, double (*sh)[16], float2* stat) {
  const int in = threadIdx.x & 15, g = g0 + in, slice = threadIdx.x >> 4;
  const long long len = gn_length(p, n);
  const float2* part = (const float2*)p.part + n * p.chunks * p.G + g;
  const int live = g < p.G ? (int)min((long long)p.chunks, (len + p.rows - 1) / p.rows) : 0;
  auto rows = [&](int k) { return (double)min((long long)p.rows, len - (long long)k * p.rows); };
  double s = 0.0;
#pragma unroll 4
  for (int k = slice; k < live; k += 16) s += rows(k) * part[(long long)k * p.G].x;
  const double mean = len > 0 ? gn_slices(s, sh, slice, in) / (double)len : 0.0;
  s = 0.0;
#pragma unroll 4
  for (int k = slice; k < live; k += 16) {
    const float2 t = part[(long long)k * p.G];
    const double d = t.x - mean;
    s += t.y + rows(k) * p.cpg * d * d;
  }
  s = gn_slices(s, sh, slice, in);
  if (slice == 0 && g < p.G) stat[in] = make_float2((float)mean, len > 0 ? (float)(1.0 / sqrt(s / ((double)len * p.cpg) + (double)p.eps)) : 0.f);
  __syncthreads();
}
__global__ __launch_bounds__(256) void gn_finalize_kernel(const GnParams p) {
  __shared__ double sh[16][16];
  __shared__ float2 stat[16];
  const unsigned per = (unsigned)(p.G + 15) / 16;
  const long long n = blockIdx.x / per;
  const int g0 = (int)(blockIdx.x % per) * 16, g = g0 + threadIdx.x;
  gn_finalize(p, n, g0, sh, stat);
  if (threadIdx.x >= 16 || g >= p.G) return;
  p.mean[n * p.G + g] = stat[threadIdx.x].x;
  p.rstd[n * p.G + g] = stat[threadIdx.x].y;
}
constexpr int kGnMergeHere = 32;   // most groups whose partials the elementwise pass merges in every block

// ---- y = act((x - mean) rstd w + b), row blocks again; rows behind the length become zero
template <int DT, int VEC, int ACT>
__global__ __launch_bounds__(256) void gn_apply_kernel(const GnParams p) {
  typedef typename OpType<DT>::T T;
  const unsigned blk = gridDim.x - 1 - blockIdx.x;   // last rows first: they are what the statistics pass left in the last-level cache
  const long long n = blk / (unsigned)p.achunks;
  const long long len = gn_length(p, n), r0 = (long long)(blk % (unsigned)p.achunks) * p.arows;
  const int rows = (int)min((long long)p.arows, p.L - r0);
  __shared__ double sh[16][16];
  __shared__ float2 stat[kGnMergeHere];
  if (p.merge_here) {
    for (int g0 = 0; g0 < p.G; g0 += 16) gn_finalize(p, n, g0, sh, stat + g0);
    if (blk % (unsigned)p.achunks == 0 && (int)threadIdx.x < p.G) {
      p.mean[n * p.G + threadIdx.x] = stat[threadIdx.x].x;
      p.rstd[n * p.G + threadIdx.x] = stat[threadIdx.x].y;
    }
  }
  const int real = (int)max(0ll, min((long long)rows, len - r0));
  const T* x = (const T*)p.x + n * p.xn + r0 * p.xl;
  T* y = (T*)p.out + n * p.on + r0 * p.ol;
  const int lanes = min(p.cv, 256), rp = 256 / lanes;
  const int tc = threadIdx.x % lanes, tr = threadIdx.x / lanes;
  if (tr >= rp) return;
  for (int v = tc; v < p.cv; v += 256) {
    float mu[VEC], a[VEC], b[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      const int c = v * VEC + k, g = c / p.cpg;
      const float2 st = p.merge_here ? stat[g] : make_float2(p.mean[n * p.G + g], p.rstd[n * p.G + g]);
      mu[k] = st.x;
      a[k] = st.y * gn_param<DT>(p.w, c, p.affine_f32, 1.f);
      b[k] = gn_param<DT>(p.b, c, p.affine_f32, 0.f);
      // 16-bit inputs: the mean folded into the offset costs |mean| rstd |w| 2^-24, their own rounding is 2^11 times that
      if constexpr (DT != 0) b[k] = fmaf(-mu[k], a[k], b[k]);
    }
    const T* xs = x + (long long)v * VEC;
    T* ys = y + (long long)v * VEC;
    int r = tr;
#pragma unroll 4
    for (; r < real; r += rp) {
      float f[VEC];
      OpVec<DT, VEC>::load(xs + r * p.xl, f);
#pragma unroll
      for (int k = 0; k < VEC; ++k) f[k] = op_act<ACT, DT == 0>(DT == 0 ? fmaf(f[k] - mu[k], a[k], b[k]) : fmaf(f[k], a[k], b[k]));
      OpVec<DT, VEC>::store(ys + r * p.ol, f);
    }
    for (; r < rows; r += rp) {
      float f[VEC];
#pragma unroll
      for (int k = 0; k < VEC; ++k) f[k] = 0.f;
      OpVec<DT, VEC>::store(ys + r * p.ol, f);
    }
  }
}

// ---- backward, pass 1: per channel sum of dz and of dz xhat over a row block
template <int DT, int VEC, int ACT>
__global__ __launch_bounds__(256) void gn_bwd_sums_kernel(const GnParams p) {
  typedef typename OpType<DT>::T T;
  __shared__ float red[256 * 2 * VEC];
  const long long n = blockIdx.x / (unsigned)p.chunks;
  const int chunk = (int)(blockIdx.x % (unsigned)p.chunks);
  const long long len = gn_length(p, n), r0 = (long long)chunk * p.rows;
  const int rows = (int)max(0ll, min((long long)p.rows, len - r0));
  if (rows == 0) return;
  const T* x = (const T*)p.x + n * p.xn + r0 * p.xl;
  const T* dy = (const T*)p.dy + n * p.dn + r0 * p.dl;
  float2* out = (float2*)p.part + (n * p.chunks + chunk) * p.C;
  const int lanes = min(p.cv, 256), rp = 256 / lanes;
  const int tc = threadIdx.x % lanes, tr = threadIdx.x / lanes;
  for (int v0 = 0; v0 < p.cv; v0 += 256) {
    const int v = v0 + tc;
    const bool on = tr < rp && v < p.cv;
    float s[VEC], q[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) s[k] = q[k] = 0.f;
    if (on) {
      float mu[VEC], rs[VEC], w[VEC], b[VEC];
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        const int c = v * VEC + k, g = c / p.cpg;
        mu[k] = p.mean[n * p.G + g];
        rs[k] = p.rstd[n * p.G + g];
        w[k] = gn_param<DT>(p.w, c, p.affine_f32, 1.f);
        b[k] = gn_param<DT>(p.b, c, p.affine_f32, 0.f);
      }
#pragma unroll 2
      for (int r = tr; r < rows; r += rp) {
        float f[VEC], d[VEC];
        OpVec<DT, VEC>::load(x + r * p.xl + (long long)v * VEC, f);
        OpVec<DT, VEC>::load(dy + r * p.dl + (long long)v * VEC, d);
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          const float h = (f[k] - mu[k]) * rs[k];
          float a, g;
          op_act_grad<ACT, DT == 0>(fmaf(h, w[k], b[k]), a, g);
          const float dz = d[k] * g;
          s[k] += dz;
          q[k] = fmaf(dz, h, q[k]);
        }
      }
    }
    if (rp > 1) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < VEC; ++k) { red[threadIdx.x * 2 * VEC + k] = s[k]; red[threadIdx.x * 2 * VEC + VEC + k] = q[k]; }
      __syncthreads();
      if (on && tr == 0)
        for (int o = 1; o < rp; ++o)
#pragma unroll
          for (int k = 0; k < VEC; ++k) {
            s[k] += red[(o * lanes + tc) * 2 * VEC + k];
            q[k] += red[(o * lanes + tc) * 2 * VEC + VEC + k];
          }
    }
    if (on && tr == 0)
#pragma unroll
      for (int k = 0; k < VEC; ++k) out[v * VEC + k] = make_float2(s[k], q[k]);
  }
}

// ---- pass 2: a sample's sums over its row blocks (fp64, 4 threads per channel) and its groups' A / M and B / M; a block per sample
__global__ __launch_bounds__(1024) void gn_bwd_merge_kernel(const GnParams p) {
  __shared__ double2 sh[4][256];
  const long long n = blockIdx.x;
  const long long len = gn_length(p, n);
  const int in = threadIdx.x & 255, slice = threadIdx.x >> 8;
  const int live = (int)min((long long)p.chunks, (len + p.rows - 1) / p.rows);
  for (int c0 = 0; c0 < p.C; c0 += 256) {
    const int c = c0 + in;
    double s = 0.0, q = 0.0;
    if (c < p.C) {
      const float2* part = (const float2*)p.part + n * p.chunks * p.C + c;
#pragma unroll 4
      for (int k = slice; k < live; k += 4) {
        const float2 t = part[(long long)k * p.C];
        s += t.x;
        q += t.y;
      }
    }
    sh[slice][in] = make_double2(s, q);
    __syncthreads();
    if (slice == 0 && c < p.C) {
      for (int i = 1; i < 4; ++i) { s += sh[i][in].x; q += sh[i][in].y; }
      p.sums[(n * p.C + c) * 2] = s;
      p.sums[(n * p.C + c) * 2 + 1] = q;
    }
    __syncthreads();
  }
}
// ... its groups: a wave per group (the blocks above have ended: their sums are visible)
template <int DT>
__global__ __launch_bounds__(256) void gn_bwd_groups_kernel(const GnParams p) {
  const int lane = threadIdx.x & 63;
  const long long i = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);   // n * G + g
  if (i >= p.N * p.G) return;
  const long long n = i / p.G;
  const int g = (int)(i - n * p.G);
  double a = 0.0, b = 0.0;
  for (int c = lane; c < p.cpg; c += 64) {
    const int ch = g * p.cpg + c;
    const double w = gn_param<DT>(p.w, ch, p.affine_f32, 1.f);
    a += w * p.sums[(n * p.C + ch) * 2];
    b += w * p.sums[(n * p.C + ch) * 2 + 1];
  }
  a = wave_sum_d(a);
  b = wave_sum_d(b);
  const double m = (double)gn_length(p, n) * p.cpg;
  if (lane == 0) {
    double* o = p.gsums + i * 2;
    o[0] = m > 0 ? a / m : 0.0;
    o[1] = m > 0 ? b / m : 0.0;
  }
}

// ---- the affine's gradients: sums over the samples, 64 channels by 256 threads (4 per channel), in a fixed order
template <int DT> __device__ __forceinline__ void gn_affine_grads(const GnParams& p, int c0, double2 (*sh)[64]) {
  typedef typename OpType<DT>::T T;
  const int in = threadIdx.x & 63, slice = threadIdx.x >> 6, c = c0 + in;
  double s = 0.0, q = 0.0;
  if (c < p.C)
#pragma unroll 4
    for (long long n = slice; n < p.N; n += 4) {
      s += p.sums[(n * p.C + c) * 2];
      q += p.sums[(n * p.C + c) * 2 + 1];
    }
  sh[slice][in] = make_double2(s, q);
  __syncthreads();
  if (slice || c >= p.C) return;
  for (int i = 1; i < 4; ++i) { s += sh[i][in].x; q += sh[i][in].y; }
  if (p.db) { if (p.affine_f32) ((float*)p.db)[c] = (float)s; else ((T*)p.db)[c] = op_store<DT>((float)s); }
  if (p.dw) { if (p.affine_f32) ((float*)p.dw)[c] = (float)q; else ((T*)p.dw)[c] = op_store<DT>((float)q); }
}
template <int DT>
__global__ __launch_bounds__(256) void gn_affine_grads_kernel(const GnParams p) {
  __shared__ double2 sh[4][64];
  gn_affine_grads<DT>(p, blockIdx.x * 64, sh);
}

// ---- pass 3: dx
template <int DT, int VEC, int ACT>
__global__ __launch_bounds__(256) void gn_bwd_apply_kernel(const GnParams p) {
  typedef typename OpType<DT>::T T;
  __shared__ double2 sh[4][64];
  const unsigned row_blocks = (unsigned)(p.N * p.achunks);
  if (blockIdx.x >= row_blocks) { gn_affine_grads<DT>(p, (int)(blockIdx.x - row_blocks) * 64, sh); return; }
  const unsigned blk = row_blocks - 1 - blockIdx.x;   // see gn_apply_kernel
  const long long n = blk / (unsigned)p.achunks;
  const long long len = gn_length(p, n), r0 = (long long)(blk % (unsigned)p.achunks) * p.arows;
  const int rows = (int)min((long long)p.arows, p.L - r0);
  const int real = (int)max(0ll, min((long long)rows, len - r0));
  const T* x = (const T*)p.x + n * p.xn + r0 * p.xl;
  const T* dy = (const T*)p.dy + n * p.dn + r0 * p.dl;
  T* dx = (T*)p.out + n * p.on + r0 * p.ol;
  const int lanes = min(p.cv, 256), rp = 256 / lanes;
  const int tc = threadIdx.x % lanes, tr = threadIdx.x / lanes;
  if (tr >= rp) return;
  const double* grp = p.gsums + n * p.G * 2;
  for (int v = tc; v < p.cv; v += 256) {
    float mu[VEC], rs[VEC], w[VEC], b[VEC], A[VEC], B[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      const int c = v * VEC + k, g = c / p.cpg;
      mu[k] = p.mean[n * p.G + g];
      rs[k] = p.rstd[n * p.G + g];
      w[k] = gn_param<DT>(p.w, c, p.affine_f32, 1.f);
      b[k] = gn_param<DT>(p.b, c, p.affine_f32, 0.f);
      A[k] = (float)grp[g * 2];
      B[k] = (float)grp[g * 2 + 1];
    }
    int r = tr;
#pragma unroll 2
    for (; r < real; r += rp) {
      float f[VEC], d[VEC];
      OpVec<DT, VEC>::load(x + r * p.xl + (long long)v * VEC, f);
      OpVec<DT, VEC>::load(dy + r * p.dl + (long long)v * VEC, d);
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        const float h = (f[k] - mu[k]) * rs[k];
        float a, g;
        op_act_grad<ACT, DT == 0>(fmaf(h, w[k], b[k]), a, g);
        f[k] = rs[k] * (d[k] * g * w[k] - fmaf(h, B[k], A[k]));
      }
      OpVec<DT, VEC>::store(dx + r * p.ol + (long long)v * VEC, f);
    }
    for (; r < rows; r += rp) {
      float f[VEC];
#pragma unroll
      for (int k = 0; k < VEC; ++k) f[k] = 0.f;
      OpVec<DT, VEC>::store(dx + r * p.ol + (long long)v * VEC, f);
    }
  }
}

// ---- whole samples on chip: one block owns `bc` channels (whole groups, at least 32 B of a row) of one sample and keeps its rows in
// registers, so x (and dy) are read once.  256 threads (backward 512), NV 16-byte vectors each: vector i of thread t is piece
// t + threads * i, piece = row * cvb + channel vector.  Bound: HBM and the activation's VALU work, about equal.  Neighbouring
// blocks share 128-byte lines and run on one XCD (xcd_remap), so the L2 serves the other parts of a line.
template <int DT> struct GnVec {
  static constexpr int VEC = 16 / (int)sizeof(typename OpType<DT>::T);
  static __device__ __forceinline__ void unpack(const u16x8& r, float (&f)[VEC]) {
    if constexpr (DT == 0) {
      const f32x4 v = __builtin_bit_cast(f32x4, r);
#pragma unroll
      for (int k = 0; k < VEC; ++k) f[k] = v[k];
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k) f[k] = from_h16<DT == 1>(r[k]);
    }
  }
  static __device__ __forceinline__ u16x8 pack(const float (&f)[VEC]) {
    if constexpr (DT == 0) return __builtin_bit_cast(u16x8, f32x4{f[0], f[1], f[2], f[3]});
    else {
      u16x8 r;
#pragma unroll
      for (int k = 0; k < VEC; ++k) r[k] = to_h16<DT == 1>(f[k]);
      return r;
    }
  }
};

// sum over the lanes of a row of 16 that hold the same channel vector (lane % cvb), on the VALU (DPP rotations)
__device__ __forceinline__ float gn_row_sum(float v, int cvb) {
  if (cvb <= 1) v = ror_add<0x121>(v);
  if (cvb <= 2) v = ror_add<0x122>(v);
  if (cvb <= 4) v = ror_add<0x124>(v);
  if (cvb <= 8) v = ror_add<0x128>(v);
  return v;
}
constexpr int kGnMaxCvb = 8;
constexpr int kGnSlabThreads = 256, kGnSlabBwdThreads = 512;

// Block sums of NQ values per channel vector: v in every thread on entry, tot[vector * NQ + k] on exit.  Fixed order.
template <int NQ, int THREADS> __device__ __forceinline__ void gn_block_sums(const float (&v)[NQ], int cvb, float* red, float* tot) {
  const int row = threadIdx.x >> 4, in = threadIdx.x & 15, outs = cvb * NQ;   // rows of 16 lanes
#pragma unroll
  for (int k = 0; k < NQ; ++k) {
    const float s = gn_row_sum(v[k], cvb);
    if (in < cvb) red[row * outs + in * NQ + k] = s;
  }
  __syncthreads();
  constexpr int P = THREADS / 128;              // threads per sum (at most 128 sums), 8 rows each
  const int o = threadIdx.x / P, part = threadIdx.x % P;
  float s = 0.f;
  if (o < outs)
#pragma unroll
    for (int r = 0; r < 8; ++r) s += red[(part * 8 + r) * outs + o];
#pragma unroll
  for (int d = 1; d < P; d <<= 1) s += __shfl_xor(s, d);
  if (o < outs && part == 0) tot[o] = s;
  __syncthreads();
}

template <int DT, int NV, int ACT>
__global__ __launch_bounds__(kGnSlabThreads, 4) void gn_slab_kernel(const GnParams p) {
  typedef typename OpType<DT>::T T;
  constexpr int VEC = GnVec<DT>::VEC;
  __shared__ float red[kGnSlabThreads / 16 * kGnMaxCvb * VEC], tot[kGnMaxCvb * VEC], gmean[kGnMaxCvb * VEC], grstd[kGnMaxCvb * VEC];
  const int cvb = p.cvb, bc = cvb * VEC, bundles = p.C / bc;
  const int sh = 31 - __builtin_clz(p.cpg), ngb = bc >> sh;   // groups divide a power of two here: they are powers of two
  const unsigned blk = xcd_remap(blockIdx.x, gridDim.x);
  const long long n = blk / (unsigned)bundles;
  const int c_base = (int)(blk % (unsigned)bundles) * bc;
  const int v = threadIdx.x & (cvb - 1), r0 = threadIdx.x / cvb, dr = kGnSlabThreads / cvb;
  const long long len = gn_length(p, n);
  const int real = (int)len;
  const T* x = (const T*)p.x + n * p.xn + c_base + v * VEC;
  T* y = (T*)p.out + n * p.on + c_base + v * VEC;
  u16x8 data[NV];
  {
    const T* src = x + r0 * p.xl;
#pragma unroll
    for (int i = 0; i < NV; ++i, src += dr * p.xl)
      if (r0 + i * dr < real) data[i] = *(const u16x8*)src;
  }
  // One pass as the rows arrive: sums of x - f and (x - f)^2, f = the thread's own first value.  A set that holds its own shift
  // cancels at most a factor of its size (NV rows), whatever the data; the threads' means and M2 then merge by Chan's formula.
  float s[VEC], q[VEC], first[VEC];
  const int cnt = r0 < real ? (real - r0 + dr - 1) / dr : 0;   // rows of this thread
#pragma unroll
  for (int k = 0; k < VEC; ++k) s[k] = q[k] = first[k] = 0.f;
  if (cnt > 0) GnVec<DT>::unpack(data[0], first);
#pragma unroll
  for (int i = 1; i < NV; ++i)
    if (r0 + i * dr < real) {
      float f[VEC];
      GnVec<DT>::unpack(data[i], f);
#pragma unroll
      for (int k = 0; k < VEC; ++k) { const float d = f[k] - first[k]; s[k] += d; q[k] = fmaf(d, d, q[k]); }
      __builtin_amdgcn_sched_barrier(0);
    }
  const float fc = (float)cnt, ic = cnt > 0 ? 1.f / fc : 0.f;
  float v0[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) v0[k] = 0.f;
  if (cnt > 0) {
    asm volatile("" ::: "memory");   // (read here, not held over the loop)
    GnVec<DT>::unpack(*(const u16x8*)x, v0);   // the channels' values in row 0: the reference of the sums between threads
  }
#pragma unroll
  for (int k = 0; k < VEC; ++k) v0[k] = fmaf(fc, first[k] - v0[k], s[k]);
  gn_block_sums<VEC, kGnSlabThreads>(v0, cvb, red, tot);
  const float inv = real > 0 ? 1.f / ((float)real * (float)p.cpg) : 0.f;
  if ((int)threadIdx.x < ngb) {
    // the group's mean from its first channel's value in row 0 on: fp32 loses nothing to a mean far from zero
    float ref = 0.f, t = 0.f;
    if (real > 0) {
      const T* row0 = (const T*)p.x + n * p.xn + c_base + threadIdx.x * p.cpg;
      const float ir = 1.f / (float)real;
      ref = op_load<DT>(row0[0]);
      for (int c = 0; c < p.cpg; ++c) t += fmaf(tot[threadIdx.x * p.cpg + c], ir, op_load<DT>(row0[c]) - ref);
    }
    gmean[threadIdx.x] = ref + t / (float)p.cpg;
  }
  __syncthreads();
  float mu[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) {
    mu[k] = gmean[(v * VEC + k) >> sh];
    const float d = fmaf(s[k], ic, first[k] - mu[k]);          // the thread's mean, from the group's
    v0[k] = cnt > 0 ? fmaf(fc * d, d, fmaf(-s[k], s[k] * ic, q[k])) : 0.f;
  }
  gn_block_sums<VEC, kGnSlabThreads>(v0, cvb, red, tot);
  if ((int)threadIdx.x < ngb) {
    float t = 0.f;
    for (int c = 0; c < p.cpg; ++c) t += tot[threadIdx.x * p.cpg + c];
    const float rs = real > 0 ? 1.f / sqrtf(fmaf(t, inv, p.eps)) : 0.f;
    grstd[threadIdx.x] = rs;
    const long long g = n * p.G + (c_base >> sh) + threadIdx.x;
    p.mean[g] = gmean[threadIdx.x];
    p.rstd[g] = rs;
  }
  __syncthreads();
  float a[VEC], b[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) {
    const int c = c_base + v * VEC + k;
    a[k] = grstd[(v * VEC + k) >> sh] * gn_param<DT>(p.w, c, p.affine_f32, 1.f);
    b[k] = gn_param<DT>(p.b, c, p.affine_f32, 0.f);
    if constexpr (DT != 0) b[k] = fmaf(-mu[k], a[k], b[k]);   // see gn_apply_kernel
  }
  T* dst = y + r0 * p.ol;
#pragma unroll
  for (int i = 0; i < NV; ++i, dst += dr * p.ol) {
    const int r = r0 + i * dr;
    if (r >= p.L) break;
    float f[VEC];
    if (r < real) {
      GnVec<DT>::unpack(data[i], f);
#pragma unroll
      for (int k = 0; k < VEC; ++k) f[k] = op_act<ACT, DT == 0>(DT == 0 ? fmaf(f[k] - mu[k], a[k], b[k]) : fmaf(f[k], a[k], b[k]));
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k) f[k] = 0.f;
    }
    *(u16x8*)dst = GnVec<DT>::pack(f);
    __builtin_amdgcn_sched_barrier(0);   // one vector at a time: interleaved, their temporaries would not fit beside the data
  }
}

// backward of the same: x stays in registers, and dz in fp32, so the slope is computed once
template <int DT, int NV, int ACT>
__global__ __launch_bounds__(kGnSlabBwdThreads, NV <= 4 ? 4 : 2) void gn_bwd_slab_kernel(const GnParams p) {
  typedef typename OpType<DT>::T T;
  constexpr int VEC = GnVec<DT>::VEC;
  __shared__ float red[kGnSlabBwdThreads / 16 * kGnMaxCvb * 2 * VEC], tot[kGnMaxCvb * 2 * VEC], gA[kGnMaxCvb * VEC], gB[kGnMaxCvb * VEC];
  const int cvb = p.cvb, bc = cvb * VEC, bundles = p.C / bc;
  const int sh = 31 - __builtin_clz(p.cpg), ngb = bc >> sh;   // groups divide a power of two here: they are powers of two
  const unsigned blk = xcd_remap(blockIdx.x, gridDim.x);
  const long long n = blk / (unsigned)bundles;
  const int c_base = (int)(blk % (unsigned)bundles) * bc;
  const int v = threadIdx.x & (cvb - 1), r0 = threadIdx.x / cvb, dr = kGnSlabBwdThreads / cvb;
  const int real = (int)gn_length(p, n);
  const T* x = (const T*)p.x + n * p.xn + c_base + v * VEC;
  const T* dy = (const T*)p.dy + n * p.dn + c_base + v * VEC;
  T* dx = (T*)p.out + n * p.on + c_base + v * VEC;
  u16x8 xd[NV], yd[NV];
  float dzk[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int r = r0 + i * dr;
    if (r < real) {
      xd[i] = *(const u16x8*)(x + r * p.xl);
      yd[i] = *(const u16x8*)(dy + r * p.dl);
    }
  }
  float mu[VEC], rs[VEC], w[VEC], b[VEC], s[2 * VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) {
    const int c = c_base + v * VEC + k, g = c >> sh;
    mu[k] = p.mean[n * p.G + g];
    rs[k] = p.rstd[n * p.G + g];
    w[k] = gn_param<DT>(p.w, c, p.affine_f32, 1.f);
    b[k] = gn_param<DT>(p.b, c, p.affine_f32, 0.f);
    s[k] = s[VEC + k] = 0.f;
  }
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (r0 + i * dr < real) {
      float f[VEC], d[VEC];
      GnVec<DT>::unpack(xd[i], f);
      GnVec<DT>::unpack(yd[i], d);
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        const float h = (f[k] - mu[k]) * rs[k];
        float a, g;
        op_act_grad<ACT, DT == 0>(fmaf(h, w[k], b[k]), a, g);
        const float dz = d[k] * g;
        dzk[i][k] = dz;
        s[k] += dz;
        s[VEC + k] = fmaf(dz, h, s[VEC + k]);
      }
    }
  gn_block_sums<2 * VEC, kGnSlabBwdThreads>(s, cvb, red, tot);
  if ((int)threadIdx.x < bc) {   // a channel's sums: for the affine's gradients, and into its group
    const int vv = threadIdx.x / VEC, k = threadIdx.x % VEC;
    double* o = p.sums + (n * p.C + c_base + threadIdx.x) * 2;
    o[0] = tot[vv * 2 * VEC + k];
    o[1] = tot[vv * 2 * VEC + VEC + k];
  }
  if ((int)threadIdx.x < ngb) {
    const float inv = real > 0 ? 1.f / ((float)real * (float)p.cpg) : 0.f;
    float A = 0.f, B = 0.f;
    for (int i = 0; i < p.cpg; ++i) {
      const int c = threadIdx.x * p.cpg + i, vv = c / VEC, k = c % VEC;
      const float wc = gn_param<DT>(p.w, c_base + c, p.affine_f32, 1.f);
      A = fmaf(wc, tot[vv * 2 * VEC + k], A);
      B = fmaf(wc, tot[vv * 2 * VEC + VEC + k], B);
    }
    gA[threadIdx.x] = A * inv;
    gB[threadIdx.x] = B * inv;
  }
  __syncthreads();
  float A[VEC], B[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) { A[k] = gA[(v * VEC + k) >> sh]; B[k] = gB[(v * VEC + k) >> sh]; }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int r = r0 + i * dr;
    if (r >= p.L) break;
    float f[VEC];
    if (r < real) {
      GnVec<DT>::unpack(xd[i], f);
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        const float h = (f[k] - mu[k]) * rs[k];
        f[k] = rs[k] * fmaf(dzk[i][k], w[k], -fmaf(h, B[k], A[k]));
      }
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k) f[k] = 0.f;
    }
    *(u16x8*)(dx + r * p.ol) = GnVec<DT>::pack(f);
  }
}

}  // namespace vtc
