// What vtc_ops.hip (the stand-alone operators) and vtc_api.hip (the model) share: argument structs of the operators' host
// code, which both the C entry points and the model's forward pass call, and the error message of handle-less calls.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace vtc {

enum OpDtype : int { OP_F32 = 0, OP_F16 = 1, OP_BF16 = 2 };
enum OpAct : int { ACT_NONE = 0, ACT_GELU = 1, ACT_SILU = 2, ACT_SIGMOID = 3 };

// message of the last failed handle-less call on this thread (vtc_last_error(NULL)); returns `code`
int fail_handleless(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));

// h = act(x Wg^T + bg) * (x Wu^T + bu) of the gated feed-forward block, for the model's own layers: x [M][K], Wg and Wu [F][K], h
// [M][F] dense 16-bit rows (dtype OP_F16 / OP_BF16), K and F multiples of 8, 16-byte aligned, fp32 biases.  On the current device.
void launch_gated_up(int dtype, int64_t M, int K, int F, const unsigned short* x, const unsigned short* wg, const unsigned short* wu, const float* bg,
                     const float* bu, int act, unsigned short* h, hipStream_t s);

}  // namespace vtc
