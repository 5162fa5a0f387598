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

}  // namespace vtc
