// Group norm with an activation on channel-last rows (N, L, C), forward and backward.
//
// Mathematics, per sample n and group g of C / G neighbouring channels, over the real rows l < length[n] (all L without lengths):
//   mean, rstd = 1 / sqrt(var + eps);  z = (x - mean) rstd w_c + b_c;  y = act(z).
//   backward: dz = dy act'(z);  db_c = sum dz;  dw_c = sum dz xhat (over n and l);
//   dx = rstd (w_c dz - (A + xhat B) / M),  A = sum w_c dz,  B = sum w_c dz xhat over the group, M = its element count.
// Rows at and behind length[n] are not read; y and dx are zero there.  A sample of length 0 has mean = rstd = 0.
//
// Statistics: every partial is (mean, M2 = sum of squared distances from it) and partials merge by Chan's formula, so a mean
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
  double* sums;                 // backward: [N][C][2] sums over rows, then [N][G][2] (A / M, B / M)
  void *dw, *db;                // gradients of the affine, may be null
  long long N, L;
  int C, G, cpg, cv, rows, chunks;   // cv = C / VEC; rows per row block (chunk)
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

// ---- merge the row blocks of a sample: one thread per group walks them in order
template <int DT>
__global__ __launch_bounds__(64) void gn_finalize_kernel(const GnParams p) {
  const unsigned per = (unsigned)(p.G + 63) / 64;
  const long long n = blockIdx.x / per;
  const int g = (int)(blockIdx.x % per) * 64 + threadIdx.x;
  if (g >= p.G) return;
  const long long len = gn_length(p, n);
  double mean = 0.0, m2 = 0.0, cnt = 0.0;
  const float2* part = (const float2*)p.part + n * p.chunks * p.G + g;
  for (int k = 0; k < p.chunks && (long long)k * p.rows < len; ++k) {
    const float2 t = part[(long long)k * p.G];
    const double c = (double)min((long long)p.rows, len - (long long)k * p.rows) * p.cpg;
    const double d = (double)t.x - mean, tot = cnt + c;
    mean += d * (c / tot);
    m2 += (double)t.y + d * d * (cnt * c / tot);
    cnt = tot;
  }
  p.mean[n * p.G + g] = (float)mean;
  p.rstd[n * p.G + g] = cnt > 0.0 ? (float)(1.0 / sqrt(m2 / cnt + (double)p.eps)) : 0.f;
}

// ---- y = act((x - mean) rstd w + b), row blocks again; rows behind the length become zero
template <int DT, int VEC, int ACT>
__global__ __launch_bounds__(256) void gn_apply_kernel(const GnParams p) {
  typedef typename OpType<DT>::T T;
  const long long n = blockIdx.x / (unsigned)p.chunks;
  const long long len = gn_length(p, n), r0 = (long long)(blockIdx.x % (unsigned)p.chunks) * p.rows;
  const int rows = (int)min((long long)p.rows, p.L - r0);
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
      mu[k] = p.mean[n * p.G + g];
      a[k] = p.rstd[n * p.G + g] * gn_param<DT>(p.w, c, p.affine_f32, 1.f);
      b[k] = gn_param<DT>(p.b, c, p.affine_f32, 0.f);
    }
    const T* xs = x + (long long)v * VEC;
    T* ys = y + (long long)v * VEC;
    int r = tr;
#pragma unroll 4
    for (; r < real; r += rp) {
      float f[VEC];
      OpVec<DT, VEC>::load(xs + r * p.xl, f);
#pragma unroll
      for (int k = 0; k < VEC; ++k) f[k] = op_act<ACT, DT == 0>(fmaf(f[k] - mu[k], a[k], b[k]));
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

// ---- pass 2a: sums over the row blocks of a sample, fp64, a thread per channel
__global__ __launch_bounds__(64) void gn_bwd_merge_kernel(const GnParams p) {
  const unsigned per = (unsigned)(p.C + 63) / 64;
  const long long n = blockIdx.x / per;
  const int c = (int)(blockIdx.x % per) * 64 + threadIdx.x;
  if (c >= p.C) return;
  const long long len = gn_length(p, n);
  const float2* part = (const float2*)p.part + n * p.chunks * p.C + c;
  double s = 0.0, q = 0.0;
  for (int k = 0; k < p.chunks && (long long)k * p.rows < len; ++k) {
    const float2 t = part[(long long)k * p.C];
    s += t.x;
    q += t.y;
  }
  p.sums[(n * p.C + c) * 2] = s;
  p.sums[(n * p.C + c) * 2 + 1] = q;
}

// ---- pass 2b: the group sums of every sample (blocks 0 .. N G / 4 - 1, a wave per group) and the affine's gradients
template <int DT>
__global__ __launch_bounds__(256) void gn_bwd_groups_kernel(const GnParams p, long long group_blocks) {
  typedef typename OpType<DT>::T T;
  const int lane = threadIdx.x & 63;
  if ((long long)blockIdx.x < group_blocks) {
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
      double* o = p.sums + p.N * p.C * 2 + i * 2;
      o[0] = m > 0 ? a / m : 0.0;
      o[1] = m > 0 ? b / m : 0.0;
    }
    return;
  }
  const int c = (int)(((long long)blockIdx.x - group_blocks) * 256 + threadIdx.x);
  if (c >= p.C) return;
  double s = 0.0, q = 0.0;
  for (long long n = 0; n < p.N; ++n) {
    s += p.sums[(n * p.C + c) * 2];
    q += p.sums[(n * p.C + c) * 2 + 1];
  }
  if (p.db) { if (p.affine_f32) ((float*)p.db)[c] = (float)s; else ((T*)p.db)[c] = op_store<DT>((float)s); }
  if (p.dw) { if (p.affine_f32) ((float*)p.dw)[c] = (float)q; else ((T*)p.dw)[c] = op_store<DT>((float)q); }
}

// ---- pass 3: dx
template <int DT, int VEC, int ACT>
__global__ __launch_bounds__(256) void gn_bwd_apply_kernel(const GnParams p) {
  typedef typename OpType<DT>::T T;
  const long long n = blockIdx.x / (unsigned)p.chunks;
  const long long len = gn_length(p, n), r0 = (long long)(blockIdx.x % (unsigned)p.chunks) * p.rows;
  const int rows = (int)min((long long)p.rows, p.L - r0);
  const int real = (int)max(0ll, min((long long)rows, len - r0));
  const T* x = (const T*)p.x + n * p.xn + r0 * p.xl;
  const T* dy = (const T*)p.dy + n * p.dn + r0 * p.dl;
  T* dx = (T*)p.out + n * p.on + r0 * p.ol;
  const int lanes = min(p.cv, 256), rp = 256 / lanes;
  const int tc = threadIdx.x % lanes, tr = threadIdx.x / lanes;
  if (tr >= rp) return;
  const double* grp = p.sums + p.N * p.C * 2 + n * p.G * 2;
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

}  // namespace vtc
