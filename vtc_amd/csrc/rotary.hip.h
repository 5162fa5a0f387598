// Rotary positions on the heads of q and k (interleaved or half layout, part of the head), one launch for both tensors.
//
// Mathematics: a pair (a, b) of a head at position p turns by theta = p * f_j:  (a cos - b sin, a sin + b cos), times an
// amplitude; the inverse (the gradient's direction) turns by -theta.  Pair j is elements (j, j + R/2) or (2j, 2j + 1).
//
// Precision: the angle is kept in TURNS in fp64 (f_j / 2 pi comes from the host), the product p * f_j as a two-term sum (fma),
// so the whole turns drop out exactly and what is left is good to ~1e-16 x (number of turns); fp32 angles would be off by
// 0.06 rad a million frames into a recording.  After the reduction to an eighth of a turn either way, sin and cos are Taylor
// polynomials in fp32 (|x| <= pi/4: remainders x^13/13! = 7e-12 and x^12/12! = 1.2e-10, below half an ulp of fp32).
//
// Bound: HBM (x read once, y written once).  A block takes `tpb` tokens: first the angles of its (token, pair) entries go to
// LDS, once for all heads of q and k (24 heads share one fp64 reduction), then its threads walk the (token, head, piece)
// items.  An item is 2 x VEC elements in two vector accesses (16 B each where sizes and alignment allow).
//
// Measured: fp32, 60001 x (16 + 4) x 128, 1.23 GB in and out: 245 us, 5.0 TB/s, the rate of a plain copy of that size; f16, 64 x 499
// x 24 x 64, 196 MB: 31 us where the last-level cache holds it (6.2 TB/s), 44 us among other work; 8 single frames 3.8 us (latency).
#pragma once
#include "common.hip.h"

namespace vtc {

constexpr int kRotMaxDim = 512;          // rotary_dim: the frequency table travels in the kernel arguments (2 KiB)
constexpr int kRotTableEntries = 2048;   // (cos, sin) entries of a block in LDS: 16 KiB

struct RotaryTensor {
  const void* x;
  void* y;
  long long xb, xt, xh, yb, yt, yh;   // element strides of batch, token, head (elements of a head are contiguous)
  int heads;
};
struct RotaryParams {
  RotaryTensor t[2];
  const void* pos;        // int32 / int64 positions, or null: offset + token index
  long long pb, pt;       // element strides of pos
  long long offset;
  long long tokens;       // batch * T
  int T, pos64, half, tail, heads, tpb, inverse;   // tail: elements behind the rotated part that have to be copied (0 in place)
  int vec_half, items;    // VEC-sized pieces of half, items per head (rotated + tail)
  float amp;
  double turns[kRotMaxDim / 2];   // f_j / 2 pi
};

template <int DT> struct OpType;
template <> struct OpType<0> { typedef float T; };
template <> struct OpType<1> { typedef h16 T; };
template <> struct OpType<2> { typedef h16 T; };

template <int DT> __device__ __forceinline__ float op_load(const typename OpType<DT>::T v) {
  if constexpr (DT == 0) return v;
  else return from_h16<DT == 1>(v);
}
template <int DT> __device__ __forceinline__ typename OpType<DT>::T op_store(float v) {
  if constexpr (DT == 0) return v;
  else return to_h16<DT == 1>(v);
}
// VEC consecutive elements as fp32; one access of VEC * sizeof(T) bytes (the host checked the alignment)
template <int DT, int VEC> struct OpVec {
  typedef typename OpType<DT>::T T;
  struct alignas(sizeof(T) * VEC) Raw { T v[VEC]; };
  static __device__ __forceinline__ void load(const T* p, float (&f)[VEC]) {
    const Raw r = *(const Raw*)p;
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = op_load<DT>(r.v[i]);
  }
  static __device__ __forceinline__ void store(T* p, const float (&f)[VEC]) {
    Raw r;
#pragma unroll
    for (int i = 0; i < VEC; ++i) r.v[i] = op_store<DT>(f[i]);
    *(Raw*)p = r;
  }
};

// cos and sin of 2 pi (p * f): see the head of the file
__device__ __forceinline__ float2 turn_cos_sin(double p, double f) {
  const double hi = p * f, lo = fma(p, f, -hi);
  double r = (hi - rint(hi)) + lo;                      // |r| <= 1/2 (+ rounding)
  const double q = rint(r * 4.0);
  const float x = (float)((r - q * 0.25) * 6.283185307179586476925);
  const float z = x * x;
  float s = fmaf(z, -2.50521084e-8f, 2.75573192e-6f);   // -1/11!, 1/9!
  s = fmaf(z, s, -1.98412698e-4f);                      // -1/7!
  s = fmaf(z, s, 8.33333333e-3f);
  s = fmaf(z, s, -1.66666667e-1f);
  s = fmaf(z * x, s, x);
  float c = fmaf(z, -2.75573192e-7f, 2.48015873e-5f);   // -1/10!, 1/8!
  c = fmaf(z, c, -1.38888889e-3f);
  c = fmaf(z, c, 4.16666667e-2f);
  c = fmaf(z, c, -0.5f);
  c = fmaf(z, c, 1.0f);
  const int k = (int)q & 3;
  const float cc = (k & 1) ? s : c, ss = (k & 1) ? c : s;
  return make_float2((k == 1 || k == 2) ? -cc : cc, (k & 2) ? -ss : ss);
}

template <int DT, int VEC, bool HALF>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryParams p) {
  typedef typename OpType<DT>::T T;
  __shared__ float2 table[kRotTableEntries];
  const long long tok0 = (long long)blockIdx.x * p.tpb;
  const int ntok = (int)min((long long)p.tpb, p.tokens - tok0);
  for (int i = threadIdx.x; i < ntok * p.half; i += 256) {
    const int tk = i / p.half, j = i - tk * p.half;
    const long long tok = tok0 + tk, b = tok / p.T, t = tok - b * p.T;
    long long pos = p.offset + t;
    if (p.pos) {
      const long long at = b * p.pb + t * p.pt;
      pos = p.offset + (p.pos64 ? ((const long long*)p.pos)[at] : (long long)((const int*)p.pos)[at]);
    }
    float2 cs = turn_cos_sin((double)pos, p.turns[j]);
    cs.x *= p.amp;
    cs.y *= p.inverse ? -p.amp : p.amp;
    table[i] = cs;
  }
  __syncthreads();
  const unsigned per_tok = (unsigned)(p.heads * p.items), n = (unsigned)ntok * per_tok;
  for (unsigned i = threadIdx.x; i < n; i += 256) {
    const unsigned tk = i / per_tok, r = i - tk * per_tok;
    const int head = (int)(r / (unsigned)p.items), it = (int)(r - (unsigned)head * (unsigned)p.items);
    const long long tok = tok0 + tk, b = tok / p.T, t = tok - b * p.T;
    const bool second = head >= p.t[0].heads;
    const int h = second ? head - p.t[0].heads : head;
    // both tensors' fields as scalars, selected per lane (an index into the kernel arguments would be a load per field)
    const T* x = (const T*)(second ? p.t[1].x : p.t[0].x);
    T* y = (T*)(second ? p.t[1].y : p.t[0].y);
    x += b * (second ? p.t[1].xb : p.t[0].xb) + t * (second ? p.t[1].xt : p.t[0].xt) + h * (second ? p.t[1].xh : p.t[0].xh);
    y += b * (second ? p.t[1].yb : p.t[0].yb) + t * (second ? p.t[1].yt : p.t[0].yt) + h * (second ? p.t[1].yh : p.t[0].yh);
    if (it < p.vec_half) {
      const int j = it * VEC;
      const int e0 = HALF ? j : 2 * j, e1 = HALF ? p.half + j : 2 * j + VEC;
      float u[VEC], v[VEC];
      OpVec<DT, VEC>::load(x + e0, u);
      OpVec<DT, VEC>::load(x + e1, v);
      const float2* cs = table + tk * p.half + j;
      if constexpr (HALF) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          const float2 a = cs[k];
          const float u0 = u[k], v0 = v[k];
          u[k] = fmaf(-v0, a.y, u0 * a.x);
          v[k] = fmaf(v0, a.x, u0 * a.y);
        }
      } else {
        float w2[2 * VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) { w2[k] = u[k]; w2[VEC + k] = v[k]; }
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          const float2 a = cs[k];
          const float u0 = w2[2 * k], v0 = w2[2 * k + 1];
          w2[2 * k] = fmaf(-v0, a.y, u0 * a.x);
          w2[2 * k + 1] = fmaf(v0, a.x, u0 * a.y);
        }
#pragma unroll
        for (int k = 0; k < VEC; ++k) { u[k] = w2[k]; v[k] = w2[VEC + k]; }
      }
      OpVec<DT, VEC>::store(y + e0, u);
      OpVec<DT, VEC>::store(y + e1, v);
    } else {   // the part of the head behind the rotation, copied as it is
      const int o = (it - p.vec_half) * 2 * VEC;
      typedef typename OpVec<DT, VEC>::Raw Raw;
      const T* xs = x + 2 * p.half + o;
      T* ys = y + 2 * p.half + o;
      *(Raw*)ys = *(const Raw*)xs;
      if (o + VEC < p.tail) *(Raw*)(ys + VEC) = *(const Raw*)(xs + VEC);
    }
  }
}

}  // namespace vtc
