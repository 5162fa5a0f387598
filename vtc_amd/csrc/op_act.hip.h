// Activations of the stand-alone operators and their derivatives, on fp32 values.
//
// gelu(x) = x Phi(x), gelu'(x) = Phi(x) + x phi(x).  For 16-bit results Phi is sigmoid(x P(x^2)): logit(Phi(x)) is odd and
// smooth; P is a degree-6 minimax fit of that logit with the allowed error growing from 1e-4 (|x| <= 3) as exp(1.4 (|x| - 3)),
// so that the negative tail keeps its RELATIVE accuracy: 1.4e-4 for |x| <= 3, 5.8e-4 to |x| = 4 (values of 1e-4), and
// 1.7e-5 absolute on gelu everywhere, 1/28 of an fp16 ulp at 1.  (common.hip.h's gelu_f is tighter in the middle and off by
// 3 % of the value at x = -4, which its only use, an activation stored at scale 1, does not see.)  fp32 results use erfc.
// Both saturate without NaN for every finite x.
#pragma once
#include "common.hip.h"
#include "ops.h"

namespace vtc {

__device__ __forceinline__ float sigmoid_fast(float x) {   // v_exp_f32 + v_rcp_f32: ~2 ulp + the rounding of x log2(e)
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504088896f * x));
}
__device__ __forceinline__ float phi_fast(float x) {
  const float s = x * x;
  float p = fmaf(-1.097430923913123e-09f, s, 1.216908600554234e-07f);
  p = fmaf(p, s, -5.072588010079926e-06f);
  p = fmaf(p, s, 8.63231616676785e-05f);
  p = fmaf(p, s, 0.0004971091402694583f);
  p = fmaf(p, s, -0.10577518492937088f);
  p = fmaf(p, s, -2.301586389541626f);
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * p));
}

// EXACT: results are stored in fp32
template <bool EXACT> __device__ __forceinline__ float op_sigmoid(float x) {
  if constexpr (EXACT) return 1.0f / (1.0f + expf(-x));
  else return sigmoid_fast(x);
}
template <bool EXACT> __device__ __forceinline__ float op_phi(float x) {
  if constexpr (EXACT) return 0.5f * erfcf(x * -0.70710678118654752f);
  else return phi_fast(x);
}

template <int ACT, bool EXACT> __device__ __forceinline__ float op_act(float z) {
  if constexpr (ACT == ACT_GELU) return z * op_phi<EXACT>(z);
  else if constexpr (ACT == ACT_SILU) return z * op_sigmoid<EXACT>(z);
  else if constexpr (ACT == ACT_SIGMOID) return op_sigmoid<EXACT>(z);
  else return z;
}
// value and derivative together
template <int ACT, bool EXACT> __device__ __forceinline__ void op_act_grad(float z, float& a, float& d) {
  if constexpr (ACT == ACT_GELU) {
    const float p = op_phi<EXACT>(z);
    const float e = -0.5f * z * z;
    const float g = EXACT ? expf(e) : __builtin_amdgcn_exp2f(e * 1.44269504088896f);
    a = z * p;
    d = fmaf(z * 0.39894228040143268f, g, p);
  } else if constexpr (ACT == ACT_SILU) {
    const float s = op_sigmoid<EXACT>(z);
    a = z * s;
    d = s * fmaf(z, 1.0f - s, 1.0f);
  } else if constexpr (ACT == ACT_SIGMOID) {
    const float s = op_sigmoid<EXACT>(z);
    a = s;
    d = s * (1.0f - s);
  } else {
    a = z;
    d = 1.0f;
  }
}

}  // namespace vtc
