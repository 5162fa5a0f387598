// Stand-alone operators of libvtc_amd.so (include/vtc_amd.h, "Operators"): argument checks, launch shapes, dispatch.
// They take no model handle; errors are reported as for the other handle-less calls.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>

#include "../../include/vtc_amd.h"
#include "groupnorm.hip.h"
#include "ops.h"
#include "rotary.hip.h"

using namespace vtc;

namespace {

// Makes `device` current for the call and puts the caller's device back; refuses what is not a gfx950 GPU.
struct DeviceGuard {
  int before = -1, rc = VTC_OK;
  explicit DeviceGuard(int device) {
    static int known[64] = {0};   // 0 = not looked at, 1 = gfx950 (a word per device, written with one value only)
    int n = 0;
    if (hipGetDeviceCount(&n) != hipSuccess || n < 1) { rc = fail_handleless(VTC_ERR_NO_GPU, "no HIP device visible"); return; }
    if (device < 0 || device >= n || device >= 64) { rc = fail_handleless(VTC_ERR_ARG, "device %d out of range (%d visible)", device, n); return; }
    if (!__atomic_load_n(&known[device], __ATOMIC_RELAXED)) {
      hipDeviceProp_t prop;
      if (hipGetDeviceProperties(&prop, device) != hipSuccess) { rc = fail_handleless(VTC_ERR_HIP, "hipGetDeviceProperties failed"); return; }
      if (strncmp(prop.gcnArchName, "gfx950", 6) != 0) {
        rc = fail_handleless(VTC_ERR_NO_GPU, "device %d is %s; this library is built for gfx950 only", device, prop.gcnArchName);
        return;
      }
      __atomic_store_n(&known[device], 1, __ATOMIC_RELAXED);
    }
    if (hipGetDevice(&before) != hipSuccess) { before = -1; rc = fail_handleless(VTC_ERR_HIP, "hipGetDevice failed"); return; }
    if (before == device) { before = -1; return; }
    if (hipSetDevice(device) != hipSuccess) { before = -1; rc = fail_handleless(VTC_ERR_HIP, "hipSetDevice(%d) failed", device); }
  }
  ~DeviceGuard() { if (before >= 0) (void)hipSetDevice(before); }
};

int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? VTC_OK : fail_handleless(VTC_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

int esize(int dt) { return dt == OP_F32 ? 4 : 2; }
bool dtype_ok(int dt) { return dt >= OP_F32 && dt <= OP_BF16; }

// One past the last byte a strided tensor touches (all strides >= 0).
const char* end_of(const void* p, std::initializer_list<std::pair<long long, long long>> dims, long long inner, int es) {
  long long last = 0;
  for (auto& d : dims) last += (d.first - 1) * d.second;
  return (const char*)p + (last + inner) * es;
}
bool overlap(const void* a, const char* a_end, const void* b, const char* b_end) { return (const char*)a < b_end && (const char*)b < a_end; }

// Largest of 16 B / 8 B / .. pieces that divides every stride, size and address given (as a count of elements).
int vec_of(int dt, std::initializer_list<long long> counts, std::initializer_list<const void*> ptrs) {
  int v = 16 / esize(dt);
  while (v > 1) {
    bool ok = true;
    for (long long c : counts) ok = ok && c % v == 0;
    for (const void* p : ptrs) ok = ok && ((uintptr_t)p % (v * esize(dt))) == 0;
    if (ok) break;
    v >>= 1;
  }
  return v;
}

// f(integral_constant<DT>, integral_constant<VEC>) for the run-time pair
template <typename F> void by_vec(int dt, int vec, F&& f) {
  auto v = [&](auto d) {
    switch (vec) {
      case 8: if constexpr (decltype(d)::value != OP_F32) { f(d, std::integral_constant<int, 8>{}); } break;
      case 4: f(d, std::integral_constant<int, 4>{}); break;
      case 2: f(d, std::integral_constant<int, 2>{}); break;
      default: f(d, std::integral_constant<int, 1>{}); break;
    }
  };
  if (dt == OP_F32) v(std::integral_constant<int, OP_F32>{});
  else if (dt == OP_F16) v(std::integral_constant<int, OP_F16>{});
  else v(std::integral_constant<int, OP_BF16>{});
}
template <typename F> void by_act(int act, F&& f) {
  switch (act) {
    case ACT_GELU: f(std::integral_constant<int, ACT_GELU>{}); break;
    case ACT_SILU: f(std::integral_constant<int, ACT_SILU>{}); break;
    case ACT_SIGMOID: f(std::integral_constant<int, ACT_SIGMOID>{}); break;
    default: f(std::integral_constant<int, ACT_NONE>{}); break;
  }
}

}  // namespace

// ===================================================================================== rotary
namespace {

int rotary_check_tensor(const char* name, const vtc_heads& t, const vtc_rotary& r, long long B, long long T, int dt, bool* in_place) {
  if (!t.x || !t.y) return fail_handleless(VTC_ERR_ARG, "rotary: %s is null", name);
  if (t.heads < 1 || t.heads > 65536) return fail_handleless(VTC_ERR_ARG, "rotary: %s has %d heads", name, t.heads);
  for (long long s : {t.x_batch, t.x_row, t.x_head, t.y_batch, t.y_row, t.y_head})
    if (s < 0) return fail_handleless(VTC_ERR_ARG, "rotary: %s has a negative stride", name);
  if ((uintptr_t)t.x % esize(dt) || (uintptr_t)t.y % esize(dt)) return fail_handleless(VTC_ERR_ARG, "rotary: %s is not aligned to its type", name);
  // the output's elements must be distinct: strides, from the smallest, step over all that lies inside them
  std::pair<long long, long long> d[3] = {{t.y_batch, B}, {t.y_row, T}, {t.y_head, t.heads}};
  std::sort(d, d + 3);
  long long span = r.head_dim;
  for (auto& e : d) {
    if (e.second == 1) continue;
    if (e.first < span) return fail_handleless(VTC_ERR_ARG, "rotary: the output %s overlaps itself", name);
    span = e.first * (e.second - 1) + span;
  }
  *in_place = t.x == t.y && (B == 1 || t.x_batch == t.y_batch) && (T == 1 || t.x_row == t.y_row) && (t.heads == 1 || t.x_head == t.y_head);
  return VTC_OK;
}

// No element in common: ranges that do not meet, or columns apart in rows of one pitch (q and k inside a fused projection's rows).
bool apart(const void* a, const char* a_end, long long a_batch, long long a_row, long long a_width, const void* b, const char* b_end,
           long long b_batch, long long b_row, long long b_width, long long batch, int es) {
  if (!overlap(a, a_end, b, b_end)) return true;
  if (a_row != b_row || a_row < 1 || (batch > 1 && (a_batch % a_row || b_batch % a_row))) return false;
  const long long bytes = (const char*)b - (const char*)a;
  if (bytes % es) return false;
  const long long d = ((bytes / es) % a_row + a_row) % a_row;
  return d >= a_width && d + b_width <= a_row;
}

}  // namespace

extern "C" int vtc_rotary_heads(int device, int dtype, const vtc_rotary* r, int64_t batch, int64_t length, const vtc_heads* tensors,
                                int32_t n_tensors, const void* positions, int32_t positions64, int64_t pos_batch, int64_t pos_row,
                                int64_t offset, int32_t inverse, void* stream) {
  if (!r || !tensors || n_tensors < 1 || n_tensors > 2) return fail_handleless(VTC_ERR_ARG, "rotary: one or two tensors, got %d", n_tensors);
  if (!dtype_ok(dtype)) return fail_handleless(VTC_ERR_ARG, "rotary: unknown type %d", dtype);
  if (batch < 0 || length < 0) return fail_handleless(VTC_ERR_ARG, "rotary: negative size");
  if (r->head_dim < 2 || r->head_dim > 65536) return fail_handleless(VTC_ERR_ARG, "rotary: head_dim %d not in 2..65536", r->head_dim);
  if (r->rotary_dim < 2 || r->rotary_dim % 2 || r->rotary_dim > r->head_dim || r->rotary_dim > kRotMaxDim)
    return fail_handleless(VTC_ERR_ARG, "rotary: rotary_dim %d must be even and in 2..min(head_dim = %d, %d)", r->rotary_dim, r->head_dim, kRotMaxDim);
  if (r->layout != VTC_ROTARY_HALF && r->layout != VTC_ROTARY_INTERLEAVED) return fail_handleless(VTC_ERR_ARG, "rotary: unknown layout %d", r->layout);
  if (!r->frequency) return fail_handleless(VTC_ERR_ARG, "rotary: no frequencies");
  if (!std::isfinite(r->amplitude)) return fail_handleless(VTC_ERR_ARG, "rotary: the amplitude is not finite");
  if (pos_batch < 0 || pos_row < 0) return fail_handleless(VTC_ERR_ARG, "rotary: negative position stride");
  if (positions && (uintptr_t)positions % (positions64 ? 8 : 4)) return fail_handleless(VTC_ERR_ARG, "rotary: positions are not aligned to their type");
  RotaryParams p{};
  const int half = r->rotary_dim / 2;
  for (int j = 0; j < half; ++j) {
    if (!std::isfinite(r->frequency[j])) return fail_handleless(VTC_ERR_ARG, "rotary: frequency %d is not finite", j);
    p.turns[j] = r->frequency[j] / 6.283185307179586476925286766559;
  }
  if (batch == 0 || length == 0) return VTC_OK;
  if (length > 0x7fffffff || batch > 0x7fffffffffffll / length) return fail_handleless(VTC_ERR_ARG, "rotary: too many rows");
  int vec = 16 / esize(dtype);
  bool copy_tail = false;
  const char* ends[2][2];
  for (int i = 0; i < n_tensors; ++i) {
    const vtc_heads& t = tensors[i];
    const char* name = i ? "second tensor" : "first tensor";
    bool in_place = false;
    if (int rc = rotary_check_tensor(name, t, *r, batch, length, dtype, &in_place)) return rc;
    ends[i][0] = end_of(t.x, {{batch, t.x_batch}, {length, t.x_row}, {t.heads, t.x_head}}, r->head_dim, esize(dtype));
    ends[i][1] = end_of(t.y, {{batch, t.y_batch}, {length, t.y_row}, {t.heads, t.y_head}}, r->head_dim, esize(dtype));
    if (!in_place && overlap(t.x, ends[i][0], t.y, ends[i][1]))
      return fail_handleless(VTC_ERR_ARG, "rotary: input and output of the %s overlap without being the same", name);
    copy_tail = copy_tail || !in_place;
    p.t[i] = RotaryTensor{t.x, t.y, t.x_batch, t.x_row, t.x_head, t.y_batch, t.y_row, t.y_head, t.heads};
    p.heads += t.heads;
    auto eff = [](long long stride, long long count) { return count > 1 ? stride : 0ll; };
    vec = std::min(vec, vec_of(dtype, {half, r->head_dim - r->rotary_dim, eff(t.x_batch, batch), eff(t.x_row, length), eff(t.x_head, t.heads),
                                       eff(t.y_batch, batch), eff(t.y_row, length), eff(t.y_head, t.heads)}, {t.x, t.y}));
  }
  for (int i = 0; n_tensors == 2 && i < 2; ++i) {   // what one tensor's blocks write, the other's must not read or write
    const vtc_heads &a = tensors[i], &b = tensors[1 - i];
    if (!apart(a.y, ends[i][1], a.y_batch, a.y_row, (a.heads - 1) * a.y_head + r->head_dim, b.x, ends[1 - i][0], b.x_batch, b.x_row,
               (b.heads - 1) * b.x_head + r->head_dim, batch, esize(dtype)) ||
        !apart(a.y, ends[i][1], a.y_batch, a.y_row, (a.heads - 1) * a.y_head + r->head_dim, b.y, ends[1 - i][1], b.y_batch, b.y_row,
               (b.heads - 1) * b.y_head + r->head_dim, batch, esize(dtype)))
      return fail_handleless(VTC_ERR_ARG, "rotary: an output shares memory with the other tensor");
  }
  DeviceGuard guard(device);
  if (guard.rc) return guard.rc;
  p.pos = positions; p.pos64 = positions64 ? 1 : 0; p.pb = pos_batch; p.pt = pos_row; p.offset = offset;
  p.tokens = (long long)batch * length; p.T = (int)length;
  p.half = half; p.tail = copy_tail ? r->head_dim - r->rotary_dim : 0;
  p.amp = (float)r->amplitude; p.inverse = inverse ? 1 : 0;
  p.vec_half = half / vec;
  p.items = p.vec_half + (p.tail + 2 * vec - 1) / (2 * vec);
  // tokens of a block: ~4 items per thread, the angle table within its LDS, and at least ~1000 blocks where there are rows for it
  const long long per_tok = (long long)p.heads * p.items;
  long long tpb = std::max<long long>(1, 1024 / per_tok);
  tpb = std::min<long long>(tpb, kRotTableEntries / half);
  tpb = std::min<long long>(tpb, std::max<long long>(1, p.tokens / 1024));
  p.tpb = (int)tpb;
  const long long blocks = (p.tokens + tpb - 1) / tpb;
  if (blocks > 0x7fffffff || per_tok * tpb > 0x7fffffff) return fail_handleless(VTC_ERR_ARG, "rotary: too many rows");
  by_vec(dtype, vec, [&](auto d, auto v) {
    constexpr int DT = decltype(d)::value, VEC = decltype(v)::value;
    if (r->layout == VTC_ROTARY_HALF)
      hipLaunchKernelGGL((rotary_kernel<DT, VEC, true>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, p);
    else
      hipLaunchKernelGGL((rotary_kernel<DT, VEC, false>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, p);
  });
  return launched("rotary");
}

// ===================================================================================== group norm + activation
namespace {

size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

// Rows of a block: enough blocks to fill 256 CUs several times over, enough rows to pay for a block's reduction.
void gn_shape(long long N, long long L, int* rows, int* chunks) {
  long long want = std::max<long long>(1, 4096 / std::max<long long>(1, N));   // row blocks per sample
  long long r = (L + want - 1) / want;
  r = std::max<long long>(r, 32);
  r = std::min<long long>(r, 256);
  *rows = (int)r;
  *chunks = (int)std::max<long long>(1, (L + r - 1) / r);
}

int gn_check(const char* what, int dtype, int affine_f32, const vtc_rows3* const* ts, int n_t, int64_t N, int64_t L, int C, int G, int act) {
  if (!dtype_ok(dtype)) return fail_handleless(VTC_ERR_ARG, "%s: unknown type %d", what, dtype);
  if (affine_f32 != 0 && affine_f32 != 1) return fail_handleless(VTC_ERR_ARG, "%s: affine_f32 must be 0 or 1", what);
  if (act != ACT_NONE && act != ACT_GELU && act != ACT_SILU) return fail_handleless(VTC_ERR_ARG, "%s: unknown activation %d", what, act);
  if (N < 0 || L < 0) return fail_handleless(VTC_ERR_ARG, "%s: negative size", what);
  if (C < 1 || C > kGnMaxChannels) return fail_handleless(VTC_ERR_ARG, "%s: %d channels not in 1..%d", what, C, kGnMaxChannels);
  if (G < 1 || C % G) return fail_handleless(VTC_ERR_ARG, "%s: %d channels do not divide into %d groups", what, C, G);
  if (N == 0 || L == 0) return VTC_OK;
  if (L > (1ll << 40) || N > (1ll << 40) / L) return fail_handleless(VTC_ERR_ARG, "%s: too many rows", what);
  int rows, chunks;
  if (L > (long long)256 * 0x7ffffff) return fail_handleless(VTC_ERR_ARG, "%s: too many rows", what);
  gn_shape(N, L, &rows, &chunks);
  if (N * (long long)chunks > 0x7fffffff || N * (long long)((C + 63) / 64) > 0x7fffffff) return fail_handleless(VTC_ERR_ARG, "%s: too many rows", what);
  for (int i = 0; i < n_t; ++i) {
    const vtc_rows3& t = *ts[i];
    if (!t.p) return fail_handleless(VTC_ERR_ARG, "%s: null tensor", what);
    if (t.batch < 0 || t.row < 0) return fail_handleless(VTC_ERR_ARG, "%s: negative stride", what);
    if ((uintptr_t)t.p % esize(dtype)) return fail_handleless(VTC_ERR_ARG, "%s: a tensor is not aligned to its type", what);
  }
  // the last one is written: its rows must be distinct
  const vtc_rows3& o = *ts[n_t - 1];
  std::pair<long long, long long> d[2] = {{o.batch, N}, {o.row, L}};
  std::sort(d, d + 2);
  long long span = C;
  for (auto& e : d) {
    if (e.second == 1) continue;
    if (e.first < span) return fail_handleless(VTC_ERR_ARG, "%s: the output overlaps itself", what);
    span = e.first * (e.second - 1) + span;
  }
  const char* o_end = end_of(o.p, {{N, o.batch}, {L, o.row}}, C, esize(dtype));
  for (int i = 0; i + 1 < n_t; ++i) {
    const vtc_rows3& t = *ts[i];
    const bool same = t.p == o.p && (N == 1 || t.batch == o.batch) && (L == 1 || t.row == o.row);
    if (!same && overlap(t.p, end_of(t.p, {{N, t.batch}, {L, t.row}}, C, esize(dtype)), o.p, o_end))
      return fail_handleless(VTC_ERR_ARG, "%s: an input and the output overlap without being the same", what);
  }
  return VTC_OK;
}

size_t gn_forward_bytes(int64_t N, int64_t L, int G) {
  int rows, chunks;
  gn_shape(N, L, &rows, &chunks);
  return align256((size_t)N * chunks * G * 8);
}
size_t gn_backward_bytes(int64_t N, int64_t L, int C, int G) {
  int rows, chunks;
  gn_shape(N, L, &rows, &chunks);
  return align256((size_t)N * chunks * C * 8) + align256((size_t)N * (C + G) * 16);
}

GnParams gn_params(int64_t N, int64_t L, int C, int G, const void* w, const void* b, int affine_f32, const int32_t* lengths) {
  GnParams p{};
  p.N = N; p.L = L; p.C = C; p.G = G; p.cpg = C / G;
  p.w = w; p.b = b; p.affine_f32 = affine_f32; p.length = lengths;
  gn_shape(N, L, &p.rows, &p.chunks);
  return p;
}
long long eff(long long stride, long long count) { return count > 1 ? stride : 0; }

}  // namespace

extern "C" int64_t vtc_group_norm_act_workspace(int64_t batch, int64_t length, int32_t channels, int32_t groups, int32_t backward) {
  if (batch < 0 || length < 0 || channels < 1 || groups < 1 || channels > kGnMaxChannels) {
    fail_handleless(VTC_ERR_ARG, "group norm: bad sizes");
    return VTC_ERR_ARG;
  }
  if (batch == 0 || length == 0) return 0;
  return (int64_t)(backward ? gn_backward_bytes(batch, length, channels, groups) : gn_forward_bytes(batch, length, groups));
}

extern "C" int vtc_group_norm_act(int device, int dtype, const vtc_rows3* x, const vtc_rows3* y, int64_t batch, int64_t length,
                                  int32_t channels, int32_t groups, const void* weight, const void* bias, int32_t affine_f32, double eps,
                                  int32_t act, const int32_t* lengths, float* mean, float* rstd, void* workspace, int64_t workspace_bytes,
                                  void* stream) {
  if (!x || !y) return fail_handleless(VTC_ERR_ARG, "group norm: null argument");
  const vtc_rows3* ts[2] = {x, y};
  if (int rc = gn_check("group norm", dtype, affine_f32, ts, 2, batch, length, channels, groups, act)) return rc;
  if (!(eps >= 0.0) || !std::isfinite(eps)) return fail_handleless(VTC_ERR_ARG, "group norm: eps must be finite and not negative");
  if (batch == 0 || length == 0) return VTC_OK;
  if (!mean || !rstd) return fail_handleless(VTC_ERR_ARG, "group norm: mean and rstd are needed");
  const size_t need = gn_forward_bytes(batch, length, groups);
  if (!workspace || workspace_bytes < (int64_t)need) return fail_handleless(VTC_ERR_CAPACITY, "group norm: the workspace holds %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
  if ((uintptr_t)workspace % 256) return fail_handleless(VTC_ERR_ARG, "group norm: the workspace is not aligned to 256 bytes");
  DeviceGuard guard(device);
  if (guard.rc) return guard.rc;
  GnParams p = gn_params(batch, length, channels, groups, weight, bias, affine_f32, lengths);
  p.x = x->p; p.xn = x->batch; p.xl = x->row;
  p.out = (void*)y->p; p.on = y->batch; p.ol = y->row;
  p.mean = mean; p.rstd = rstd; p.part = (float*)workspace; p.eps = (float)eps;
  const int vec = vec_of(dtype, {channels, eff(x->batch, batch), eff(x->row, length), eff(y->batch, batch), eff(y->row, length)}, {x->p, y->p});
  p.cv = channels / vec;
  hipStream_t s = (hipStream_t)stream;
  const unsigned blocks = (unsigned)(batch * p.chunks);
  by_vec(dtype, vec, [&](auto d, auto v) {
    constexpr int DT = decltype(d)::value, VEC = decltype(v)::value;
    const size_t lds = ((size_t)2 * channels + 256 * 2 * VEC) * 4;
    hipLaunchKernelGGL((gn_stats_kernel<DT, VEC>), dim3(blocks), dim3(256), lds, s, p);
    hipLaunchKernelGGL((gn_finalize_kernel<DT>), dim3((unsigned)(batch * ((groups + 63) / 64))), dim3(64), 0, s, p);
    by_act(act, [&](auto a) {
      hipLaunchKernelGGL((gn_apply_kernel<DT, VEC, decltype(a)::value>), dim3(blocks), dim3(256), 0, s, p);
    });
  });
  return launched("group norm");
}

extern "C" int vtc_group_norm_act_backward(int device, int dtype, const vtc_rows3* dy, const vtc_rows3* x, const vtc_rows3* dx, int64_t batch,
                                           int64_t length, int32_t channels, int32_t groups, const void* weight, const void* bias,
                                           int32_t affine_f32, int32_t act, const int32_t* lengths, const float* mean, const float* rstd,
                                           void* dweight, void* dbias, void* workspace, int64_t workspace_bytes, void* stream) {
  if (!x || !dy || !dx) return fail_handleless(VTC_ERR_ARG, "group norm backward: null argument");
  const vtc_rows3* ts[3] = {x, dy, dx};
  if (int rc = gn_check("group norm backward", dtype, affine_f32, ts, 3, batch, length, channels, groups, act)) return rc;
  DeviceGuard guard(device);
  if (guard.rc) return guard.rc;
  GnParams p = gn_params(batch, length, channels, groups, weight, bias, affine_f32, lengths);
  p.dw = dweight; p.db = dbias;
  hipStream_t s = (hipStream_t)stream;
  const unsigned grad_blocks = (unsigned)((channels + 255) / 256);
  if (batch == 0 || length == 0) {   // the affine's gradients are sums over nothing
    p.N = 0;
    if (dweight || dbias) by_vec(dtype, 1, [&](auto d, auto) {
      hipLaunchKernelGGL((gn_bwd_groups_kernel<decltype(d)::value>), dim3(grad_blocks), dim3(256), 0, s, p, 0ll);
    });
    return launched("group norm backward");
  }
  if (!mean || !rstd) return fail_handleless(VTC_ERR_ARG, "group norm backward: mean and rstd of the forward pass are needed");
  const size_t need = gn_backward_bytes(batch, length, channels, groups);
  if (!workspace || workspace_bytes < (int64_t)need) return fail_handleless(VTC_ERR_CAPACITY, "group norm backward: the workspace holds %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
  if ((uintptr_t)workspace % 256) return fail_handleless(VTC_ERR_ARG, "group norm backward: the workspace is not aligned to 256 bytes");
  p.x = x->p; p.xn = x->batch; p.xl = x->row;
  p.dy = dy->p; p.dn = dy->batch; p.dl = dy->row;
  p.out = (void*)dx->p; p.on = dx->batch; p.ol = dx->row;
  p.mean = (float*)mean; p.rstd = (float*)rstd;
  p.part = (float*)workspace;
  p.sums = (double*)((char*)workspace + align256((size_t)batch * p.chunks * channels * 8));
  const int vec = vec_of(dtype, {channels, eff(x->batch, batch), eff(x->row, length), eff(dy->batch, batch), eff(dy->row, length),
                                 eff(dx->batch, batch), eff(dx->row, length)}, {x->p, dy->p, dx->p});
  p.cv = channels / vec;
  const unsigned blocks = (unsigned)(batch * p.chunks);
  const long long group_blocks = ((long long)batch * groups + 3) / 4;
  by_vec(dtype, vec, [&](auto d, auto v) {
    constexpr int DT = decltype(d)::value, VEC = decltype(v)::value;
    by_act(act, [&](auto a) {
      constexpr int ACT = decltype(a)::value;
      if constexpr (ACT != ACT_SIGMOID) {
        hipLaunchKernelGGL((gn_bwd_sums_kernel<DT, VEC, ACT>), dim3(blocks), dim3(256), 0, s, p);
        hipLaunchKernelGGL(gn_bwd_merge_kernel, dim3((unsigned)(batch * ((channels + 63) / 64))), dim3(64), 0, s, p);
        hipLaunchKernelGGL((gn_bwd_groups_kernel<DT>), dim3((unsigned)(group_blocks + grad_blocks)), dim3(256), 0, s, p, group_blocks);
        hipLaunchKernelGGL((gn_bwd_apply_kernel<DT, VEC, ACT>), dim3(blocks), dim3(256), 0, s, p);
      }
    });
  });
  return launched("group norm backward");
}
