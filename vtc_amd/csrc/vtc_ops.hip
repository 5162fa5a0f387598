// Stand-alone operators of libvtc_amd.so (include/vtc_amd.h, "Operators"): argument checks, launch shapes, dispatch.
// They take no model handle; errors are reported as for the other handle-less calls.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>

#include "../../include/vtc_amd.h"
#include "gated_ffn.hip.h"
#include "groupnorm.hip.h"
#include "op_plan.h"
#include "ops.h"
#include "rotary.hip.h"

using namespace vtc;

namespace {

// Makes `device` current for the call and puts the caller's device back; refuses what is not a gfx950 GPU.
struct DeviceGuard {
  int before = -1, rc = VTC_OK;
  explicit DeviceGuard(int device) {
    static int known[64] = {0};   // 0 = not looked at, 1 = gfx950 (a word per device, written with one value only)
    if (device < 0 || device >= 64 || !__atomic_load_n(&known[device], __ATOMIC_RELAXED)) {   // the first call on a device looks at it
      int n = 0;
      if (hipGetDeviceCount(&n) != hipSuccess || n < 1) { rc = fail_handleless(VTC_ERR_NO_GPU, "no HIP device visible"); return; }
      if (device < 0 || device >= n || device >= 64) { rc = fail_handleless(VTC_ERR_ARG, "device %d out of range (%d visible)", device, n); return; }
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
template <typename F> void by_type(int dt, F&& f) {
  if (dt == OP_F32) f(std::integral_constant<int, OP_F32>{});
  else if (dt == OP_F16) f(std::integral_constant<int, OP_F16>{});
  else f(std::integral_constant<int, OP_BF16>{});
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

// One side of a tensor: (batch, length, heads) blocks of `width` contiguous elements
struct Blocks {
  const void* p;
  long long stride[3], count[3];
  int width;
  const char* end(int es) const { return end_of(p, {{count[0], stride[0]}, {count[1], stride[1]}, {count[2], stride[2]}}, width, es); }
};
// Whether two sets of blocks of the same strides, `delta` elements apart, share an element: delta = sum of q_i stride_i + e for steps
// lo_i <= q_i <= hi_i and |e| < width.  From the largest stride on; what lies inside a stride rarely reaches past the next
// multiple, so two or three steps come into question each.  Many of them (strides that are not nested) count as shared.
struct Step { long long stride, lo, hi; };
bool steps_meet(const Step* d, int n, long long delta, int width) {
  if (n == 0) return std::abs(delta) < width;
  long long reach = width - 1;
  for (int i = 1; i < n; ++i) reach += d[i].stride * std::max(-d[i].lo, d[i].hi);
  auto floor_div = [](long long a, long long b) { return a / b - (a % b < 0); };
  const long long from = std::max(d->lo, -floor_div(reach - delta, d->stride)), to = std::min(d->hi, floor_div(delta + reach, d->stride));
  if (to - from >= 8) return true;
  for (long long q = from; q <= to; ++q)
    if (steps_meet(d + 1, n - 1, delta - q * d->stride, width)) return true;
  return false;
}
// No element in common: ranges that do not meet; blocks between each other's, at the same strides (q and k inside a fused projection, in
// any order of its dimensions); or columns apart in rows of one pitch.
bool apart(const Blocks& a, const Blocks& b, int es) {
  if (!overlap(a.p, a.end(es), b.p, b.end(es))) return true;
  const long long bytes = (const char*)b.p - (const char*)a.p;
  if (bytes % es) return false;
  bool same = true;
  int n = 0;
  Step d[3];
  for (int i = 0; i < 3; ++i) {
    const long long s = a.count[i] > 1 ? a.stride[i] : b.stride[i];
    if (a.count[i] > 1 && b.count[i] > 1 && a.stride[i] != b.stride[i]) same = false;
    if ((a.count[i] > 1 || b.count[i] > 1) && s > 0) d[n++] = Step{s, -(b.count[i] - 1), a.count[i] - 1};
  }
  std::sort(d, d + n, [](const Step& x, const Step& y) { return x.stride > y.stride; });
  if (same && !steps_meet(d, n, bytes / es, a.width)) return true;
  const long long row = a.stride[1], a_width = (a.count[2] - 1) * a.stride[2] + a.width, b_width = (b.count[2] - 1) * b.stride[2] + b.width;
  if (row != b.stride[1] || row < 1 || (a.count[0] > 1 && (a.stride[0] % row || b.stride[0] % row))) return false;
  const long long at = ((bytes / es) % row + row) % row;
  return at >= a_width && at + b_width <= row;
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
  Blocks xs[2], ys[2];
  for (int i = 0; i < n_tensors; ++i) {
    const vtc_heads& t = tensors[i];
    const char* name = i ? "second tensor" : "first tensor";
    bool in_place = false;
    if (int rc = rotary_check_tensor(name, t, *r, batch, length, dtype, &in_place)) return rc;
    xs[i] = Blocks{t.x, {t.x_batch, t.x_row, t.x_head}, {batch, length, t.heads}, r->head_dim};
    ys[i] = Blocks{t.y, {t.y_batch, t.y_row, t.y_head}, {batch, length, t.heads}, r->head_dim};
    if (!in_place && !apart(xs[i], ys[i], esize(dtype)))
      return fail_handleless(VTC_ERR_ARG, "rotary: input and output of the %s overlap without being the same", name);
    copy_tail = copy_tail || !in_place;
    p.t[i] = RotaryTensor{t.x, t.y, t.x_batch, t.x_row, t.x_head, t.y_batch, t.y_row, t.y_head, t.heads};
    p.heads += t.heads;
    auto eff = [](long long stride, long long count) { return count > 1 ? stride : 0ll; };
    vec = std::min(vec, vec_of(dtype, {half, r->head_dim - r->rotary_dim, eff(t.x_batch, batch), eff(t.x_row, length), eff(t.x_head, t.heads),
                                       eff(t.y_batch, batch), eff(t.y_row, length), eff(t.y_head, t.heads)}, {t.x, t.y}));
  }
  for (int i = 0; n_tensors == 2 && i < 2; ++i)   // what one tensor's blocks write, the other's must not read or write
    if (!apart(ys[i], xs[1 - i], esize(dtype)) || !apart(ys[i], ys[1 - i], esize(dtype)))
      return fail_handleless(VTC_ERR_ARG, "rotary: an output shares memory with the other tensor");
  DeviceGuard guard(device);
  if (guard.rc) return guard.rc;
  p.pos = positions; p.pos64 = positions64 ? 1 : 0; p.pb = pos_batch; p.pt = pos_row; p.offset = offset;
  p.tokens = (long long)batch * length; p.T = (int)length;
  p.half = half; p.tail = copy_tail ? r->head_dim - r->rotary_dim : 0;
  p.amp = (float)r->amplitude; p.inverse = inverse ? 1 : 0;
  p.vec_half = half / vec;
  p.items = p.vec_half + (p.tail + 2 * vec - 1) / (2 * vec);
  const long long per_tok = (long long)p.heads * p.items;
  p.tpb = rotary_tokens_per_block(p.tokens, per_tok, kRotTableEntries / half);
  const long long blocks = (p.tokens + p.tpb - 1) / p.tpb;
  if (blocks > kMaxBlocks || per_tok * p.tpb > 0x7fffffff) return fail_handleless(VTC_ERR_ARG, "rotary: too many rows");
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

// Rows of a block, by the length and the channels alone: a sample's result must not depend on how many samples share the call.  Blocks of
// many rows pay their joins less often, blocks of few fill the chip with few samples: 64 x 3999 x 512 f16 + GELU forward takes 213 us
// with 128 blocks of a sample, 194 with 64, 178 with 32, 178 with 16; one such sample 21, 21, 23, 29; 64 x 7999 340, 312, 323, 326.
// Channels that are no whole vectors go one per thread, with fewer rows side by side.
void gn_shape(long long L, int C, int* rows, int* chunks) {
  const int split = C % 8 == 0 ? 32 : 64;
  const long long r = std::min<long long>(std::max<long long>((L + split - 1) / split, 16), 128);
  *rows = (int)r;
  *chunks = (int)std::max<long long>(1, (L + r - 1) / r);
}
// Most 16-byte vectors of a whole-sample block.  Measured, f16 + GELU, 512 channels in 32 groups, whole-sample blocks against the
// streaming kernels (us): forward 64 x 499 rows 26 / 46, 64 x 999 43 / 59, 64 x 1999 83 / 89; 64 x 3999 (blocks of twice this size)
// 206 / 182, where 8 x 3999 would take 26 / 42 and 1 x 3999 19 / 24 (the large batch decides: the choice must not look at it).  Backward 64 x 499 51 / 64, 64 x 999 70 / 87, 24 x 1999 in 512
// groups 62 / 99, 64 x 1999 199 / 162 (beyond the last-level cache), 64 x 3999 444 / 305.
constexpr long long kGnSlabVectors = 4096;
// Channel vectors of a whole-sample block (0: the sample does not fit, or its groups do not divide into such blocks).
// 2 vectors are 32 bytes of a row, the least that a fetch of a 64-byte half line uses well; wider groups take 4 or 8.
int gn_slab(int dtype, int vec, long long L, int C, int cpg) {
  const int v16 = 16 / esize(dtype);
  if (vec != v16) return 0;
  for (int cvb = 2; cvb <= kGnMaxCvb; cvb *= 2)
    if ((cvb * v16) % cpg == 0 && C % (cvb * v16) == 0) return L * cvb <= kGnSlabVectors ? cvb : 0;
  return 0;
}

// Many samples go in several launches of each kernel, one after the other (a sample's result does not depend on them).  threads: the
// most that one sample takes in any kernel of the call; what kLaunchThreads leaves of 2^32 is room for blocks that are not a sample's (the
// affine's gradients) and for counts rounded up.
constexpr long long kGnMaxLength = (1 << 30) - (1 << 17);   // 64 rows in a block of 256 where there are that many: one sample fits a launch
long long gn_slice(long long N, long long threads) { return std::min(N, std::max(1ll, kLaunchThreads / threads)); }
GnParams gn_from(GnParams p, int dtype, long long n0, long long count) {   // the same call on `count` samples from n0 on
  const long long es = esize(dtype);
  auto on = [&](const void* t, long long stride) -> const void* { return t ? (const char*)t + n0 * stride * es : nullptr; };
  p.N = count;
  p.x = on(p.x, p.xn); p.dy = on(p.dy, p.dn); p.out = (void*)on(p.out, p.on);
  p.mean += n0 * p.G; p.rstd += n0 * p.G;
  if (p.length) p.length += n0;
  if (p.sums) { p.sums += n0 * p.C * 2; p.gsums += n0 * p.G * 2; }
  return p;
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
  if (L > kGnMaxLength) return fail_handleless(VTC_ERR_ARG, "%s: too many rows", what);
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

size_t gn_forward_bytes(int64_t N, int64_t L, int C, int G) {
  int rows, chunks;
  gn_shape(L, C, &rows, &chunks);
  return align256((size_t)N * chunks * G * 8);
}
size_t gn_backward_bytes(int64_t N, int64_t L, int C, int G) {
  int rows, chunks;
  gn_shape(L, C, &rows, &chunks);
  return align256((size_t)N * chunks * C * 8) + align256((size_t)N * (C + G) * 16);
}

GnParams gn_params(int64_t N, int64_t L, int C, int G, const void* w, const void* b, int affine_f32, const int32_t* lengths) {
  GnParams p{};
  p.N = N; p.L = L; p.C = C; p.G = G; p.cpg = C / G;
  p.w = w; p.b = b; p.affine_f32 = affine_f32; p.length = lengths;
  gn_shape(L, C, &p.rows, &p.chunks);
  // the elementwise pass: ~2000 blocks where there are rows for it, at least 4 rows and at most 64
  p.arows = (int)std::min<long long>(64, std::max<long long>(4, N * L / 2048));
  p.achunks = (int)((L + p.arows - 1) / p.arows);
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
  return (int64_t)(backward ? gn_backward_bytes(batch, length, channels, groups) : gn_forward_bytes(batch, length, channels, groups));
}

extern "C" int vtc_group_norm_act(int device, int dtype, const vtc_rows3* x, const vtc_rows3* y, int64_t batch, int64_t length,
                                  int32_t channels, int32_t groups, const void* weight, const void* bias, int32_t affine_f32, double eps,
                                  int32_t act, const int32_t* lengths, float* mean, float* rstd, void* workspace, int64_t workspace_bytes,
                                  void* stream) {
  if (!x || !y) return fail_handleless(VTC_ERR_ARG, "group norm: null argument");
  const vtc_rows3* ts[2] = {x, y};
  if (int rc = gn_check("group norm", dtype, affine_f32, ts, 2, batch, length, channels, groups, act)) return rc;
  if (!(eps >= 0.0) || !std::isfinite(eps)) return fail_handleless(VTC_ERR_ARG, "group norm: eps must be finite and not negative");
  if (batch == 0) return VTC_OK;
  if (!mean || !rstd) return fail_handleless(VTC_ERR_ARG, "group norm: mean and rstd are needed");
  if (length == 0) {   // samples without rows: mean = rstd = 0
    DeviceGuard guard(device);
    if (guard.rc) return guard.rc;
    GnParams p = gn_params(batch, 0, channels, groups, nullptr, nullptr, 0, nullptr);
    p.mean = mean; p.rstd = rstd;
    const int per16 = (groups + 15) / 16;
    const long long slice = gn_slice(batch, 256ll * per16);
    for (long long n0 = 0; n0 < batch; n0 += slice) {
      const GnParams q = gn_from(p, dtype, n0, std::min(slice, batch - n0));
      hipLaunchKernelGGL(gn_finalize_kernel, dim3((unsigned)(q.N * per16)), dim3(256), 0, (hipStream_t)stream, q);
    }
    return launched("group norm");
  }
  const size_t need = gn_forward_bytes(batch, length, channels, groups);
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
  if ((p.cvb = gn_slab(dtype, vec, length, channels, p.cpg))) {
    const int per = channels / (p.cvb * vec);   // blocks of a sample
    const long long slice = gn_slice(batch, (long long)per * kGnSlabThreads);
    for (long long n0 = 0; n0 < batch; n0 += slice) {
      const GnParams q = gn_from(p, dtype, n0, std::min(slice, batch - n0));
      const dim3 grid((unsigned)(q.N * per));
      by_type(dtype, [&](auto d) { by_act(act, [&](auto a) {
        constexpr int DT = decltype(d)::value, ACT = decltype(a)::value;
        if constexpr (ACT != ACT_SIGMOID) {
          if (length * p.cvb <= 256 * 4) hipLaunchKernelGGL((gn_slab_kernel<DT, 4, ACT>), grid, dim3(kGnSlabThreads), 0, s, q);
          else hipLaunchKernelGGL((gn_slab_kernel<DT, 16, ACT>), grid, dim3(kGnSlabThreads), 0, s, q);
        }
      }); });
    }
    return launched("group norm");
  }
  // few partials and few blocks to repeat it in: the elementwise pass merges them itself, a launch less (5 x 1531 rows, 3 groups:
  // 12 us instead of 6 + 9; with 63 row blocks of 32 groups it would cost 64 x 3999 rows 20 us)
  p.merge_here = groups <= kGnMergeHere && p.chunks * groups <= 256 && batch * p.achunks <= 4096;
  const int per16 = (groups + 15) / 16;
  const long long slice = gn_slice(batch, 256ll * std::max({p.chunks, p.achunks, per16}));
  for (long long n0 = 0; n0 < batch; n0 += slice) {
    const GnParams q = gn_from(p, dtype, n0, std::min(slice, batch - n0));
    by_vec(dtype, vec, [&](auto d, auto v) {
      constexpr int DT = decltype(d)::value, VEC = decltype(v)::value;
      const size_t lds = ((size_t)2 * channels + 256 * 2 * VEC) * 4;
      hipLaunchKernelGGL((gn_stats_kernel<DT, VEC>), dim3((unsigned)(q.N * q.chunks)), dim3(256), lds, s, q);
      if (!q.merge_here) hipLaunchKernelGGL(gn_finalize_kernel, dim3((unsigned)(q.N * per16)), dim3(256), 0, s, q);
      by_act(act, [&](auto a) {
        if constexpr (decltype(a)::value != ACT_SIGMOID)
          hipLaunchKernelGGL((gn_apply_kernel<DT, VEC, decltype(a)::value>), dim3((unsigned)(q.N * q.achunks)), dim3(256), 0, s, q);
      });
    });
  }
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
  const unsigned grad_blocks = (unsigned)((channels + 63) / 64);
  if (batch == 0 || length == 0) {   // the affine's gradients are sums over nothing
    p.N = 0;
    if (dweight || dbias) by_vec(dtype, 1, [&](auto d, auto) {
      hipLaunchKernelGGL((gn_affine_grads_kernel<decltype(d)::value>), dim3(grad_blocks), dim3(256), 0, s, p);
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
  p.gsums = p.sums + batch * channels * 2;
  const int vec = vec_of(dtype, {channels, eff(x->batch, batch), eff(x->row, length), eff(dy->batch, batch), eff(dy->row, length),
                                 eff(dx->batch, batch), eff(dx->row, length)}, {x->p, dy->p, dx->p});
  p.cv = channels / vec;
  if ((p.cvb = gn_slab(dtype, vec, length, channels, p.cpg))) {
    const int per = channels / (p.cvb * vec);   // blocks of a sample
    const int nv = (int)((length * p.cvb + kGnSlabBwdThreads - 1) / kGnSlabBwdThreads);
    const long long slice = gn_slice(batch, (long long)per * kGnSlabBwdThreads);
    by_type(dtype, [&](auto d) { by_act(act, [&](auto a) {
      constexpr int DT = decltype(d)::value, ACT = decltype(a)::value;
      for (long long n0 = 0; n0 < batch; n0 += slice) {
        const GnParams q = gn_from(p, dtype, n0, std::min(slice, batch - n0));
        const dim3 grid((unsigned)(q.N * per)), block(kGnSlabBwdThreads);
        if constexpr (ACT != ACT_SIGMOID) {
          if (nv <= 2) hipLaunchKernelGGL((gn_bwd_slab_kernel<DT, 2, ACT>), grid, block, 0, s, q);
          else if (nv <= 4) hipLaunchKernelGGL((gn_bwd_slab_kernel<DT, 4, ACT>), grid, block, 0, s, q);
          else hipLaunchKernelGGL((gn_bwd_slab_kernel<DT, 8, ACT>), grid, block, 0, s, q);
        }
      }
      if (dweight || dbias) hipLaunchKernelGGL((gn_affine_grads_kernel<DT>), dim3(grad_blocks), dim3(256), 0, s, p);
    }); });
    return launched("group norm backward");
  }
  const long long slice = gn_slice(batch, std::max({256ll * p.chunks, 256ll * p.achunks, 1024ll, 64ll * groups}));
  const bool sliced = slice < batch, affine = dweight || dbias;
  by_vec(dtype, vec, [&](auto d, auto v) {
    constexpr int DT = decltype(d)::value, VEC = decltype(v)::value;
    by_act(act, [&](auto a) {
      constexpr int ACT = decltype(a)::value;
      if constexpr (ACT != ACT_SIGMOID) {
        for (long long n0 = 0; n0 < batch; n0 += slice) {
          const GnParams q = gn_from(p, dtype, n0, std::min(slice, batch - n0));
          hipLaunchKernelGGL((gn_bwd_sums_kernel<DT, VEC, ACT>), dim3((unsigned)(q.N * q.chunks)), dim3(256), 0, s, q);
          hipLaunchKernelGGL(gn_bwd_merge_kernel, dim3((unsigned)q.N), dim3(1024), 0, s, q);
          hipLaunchKernelGGL((gn_bwd_groups_kernel<DT>), dim3((unsigned)((q.N * groups + 3) / 4)), dim3(256), 0, s, q);
          // the blocks behind the rows' sum the affine's gradients
          hipLaunchKernelGGL((gn_bwd_apply_kernel<DT, VEC, ACT>), dim3((unsigned)(q.N * q.achunks + (affine && !sliced ? grad_blocks : 0))), dim3(256), 0, s, q);
        }
        if (affine && sliced) hipLaunchKernelGGL((gn_affine_grads_kernel<DT>), dim3(grad_blocks), dim3(256), 0, s, p);
      }
    });
  });
  return launched("group norm backward");
}

// ===================================================================================== gated feed-forward
namespace {

constexpr int64_t kFfnMaxDim = 1 << 18;   // width, inner width: tile offsets stay far below 2^31 bytes
// Most rows of skinny_kernel.  A forward pass, bf16, skinny / tiles (us): 768 x 2048, 1 row 8.3 / 15.0, 16 10.2 / 15.4, 32 13.0 / 15.8, 48 18.3 /
// 16.2, 64 19.5 / 16.5; 256 x 512, 64 rows 9.9 / 11.0; 2048 x 8192, 16 rows 30.0 / 30.5, 32 40 / 31, 64 64 / 33: every
// block of 16 columns reads all rows of x.
constexpr int kSkinnyRows = 32;

// Carves a workspace; with base == null it only measures.
struct Arena {
  char* base;
  size_t used = 0;
  template <typename T> T* take(size_t n) {
    T* p = base ? (T*)(base + used) : nullptr;
    used += align256(n * sizeof(T));
    return p;
  }
};
int up8(int64_t n) { return (int)((n + 7) & ~(int64_t)7); }

struct FfnArgs {
  int dtype, act, bias_f32;
  int64_t M;
  int K, F, N;
  const vtc_mat *x, *wg, *wu, *wd;
  const void *bg, *bu, *bd;
};

int ffn_check_mat(const char* what, const char* name, const vtc_mat* m, int64_t rows, int cols) {
  if (!m || !m->p) return fail_handleless(VTC_ERR_ARG, "%s: %s is null", what, name);
  if (rows > 1 && (m->row < cols || m->row > kMaxPitch))
    return fail_handleless(VTC_ERR_ARG, "%s: %s has a row pitch of %lld for %d columns (at most %d)", what, name, (long long)m->row, cols, kMaxPitch);
  if ((uintptr_t)m->p % 2) return fail_handleless(VTC_ERR_ARG, "%s: %s is not aligned to its type", what, name);
  return VTC_OK;
}
// A single row has no pitch: whatever the caller's says (the newest frame of a recording lies a whole recording from the next one's),
// what follows sees its width.
struct OneRow {
  vtc_mat m{};
  void narrow(const vtc_mat*& at, int64_t rows, int cols) {
    if (!at || rows > 1) return;
    m = vtc_mat{at->p, cols};
    at = &m;
  }
};
int ffn_check(const char* what, const FfnArgs& a) {
  if (a.dtype != OP_F16 && a.dtype != OP_BF16) return fail_handleless(VTC_ERR_ARG, "%s: operands are f16 or bf16 (matrix instructions with fp32 sums), got type %d", what, a.dtype);
  if (a.act < ACT_NONE || a.act > ACT_SIGMOID) return fail_handleless(VTC_ERR_ARG, "%s: unknown activation %d", what, a.act);
  if (a.bias_f32 != 0 && a.bias_f32 != 1) return fail_handleless(VTC_ERR_ARG, "%s: bias_f32 must be 0 or 1", what);
  if (a.M < 0 || a.M > (1ll << 31) - 256) return fail_handleless(VTC_ERR_ARG, "%s: %lld rows not in 0..2^31 - 256", what, (long long)a.M);
  for (int64_t d : {(int64_t)a.K, (int64_t)a.F, (int64_t)a.N})
    if (d < 1 || d > kFfnMaxDim) return fail_handleless(VTC_ERR_ARG, "%s: width %lld not in 1..%lld", what, (long long)d, (long long)kFfnMaxDim);
  // tiles of a launch are counted in 32 bits (the smallest are 128 x 32; with two sides at the limit of 2^18 rows are limited too)
  const int64_t widest = std::max({a.K, a.F, a.N});
  if ((a.M / 128 + 1) * (widest / 32 + 1) > (1ll << 30) || 3 * (widest / 128 + 1) * (widest / 64 + 1) > (1ll << 25))
    return fail_handleless(VTC_ERR_ARG, "%s: %lld rows of width %lld are too many", what, (long long)a.M, (long long)widest);
  for (const void* b : {a.bg, a.bu, a.bd})
    if ((uintptr_t)b % (a.bias_f32 ? 4 : 2)) return fail_handleless(VTC_ERR_ARG, "%s: a bias is not aligned to its type", what);
  if (int rc = ffn_check_mat(what, "x", a.x, a.M, a.K)) return rc;
  if (int rc = ffn_check_mat(what, "w_gate", a.wg, a.F, a.K)) return rc;
  if (int rc = ffn_check_mat(what, "w_up", a.wu, a.F, a.K)) return rc;
  if (int rc = ffn_check_mat(what, "w_down", a.wd, a.N, a.F)) return rc;
  return VTC_OK;
}
// What a call writes (all of `outs`) shares no memory with what it reads, nor with the rest of what it writes.
struct Span { const char* name; const void* p; const char* end; };
int ffn_apart(const char* what, std::initializer_list<Span> outs, std::initializer_list<Span> ins) {
  for (auto o = outs.begin(); o != outs.end(); ++o) {
    if (!o->p) continue;
    for (auto i = ins.begin(); i != ins.end(); ++i)
      if (i->p && overlap(o->p, o->end, i->p, i->end)) return fail_handleless(VTC_ERR_ARG, "%s: %s overlaps %s", what, o->name, i->name);
    for (auto i = outs.begin(); i != o; ++i)
      if (i->p && overlap(o->p, o->end, i->p, i->end)) return fail_handleless(VTC_ERR_ARG, "%s: %s overlaps %s", what, o->name, i->name);
  }
  return VTC_OK;
}
Span span(const char* name, const void* p, long long rows, long long pitch, long long cols, int es) { return {name, p, p ? end_of(p, {{rows, pitch}}, cols, es) : nullptr}; }
Span span(const char* name, const vtc_mat* m, long long rows, long long cols) { return span(name, m->p, rows, m->row, cols, 2); }

bool pieces_ok(const vtc_mat* m, int cols) { return cols % 8 == 0 && m->row % 8 == 0 && (uintptr_t)m->p % 16 == 0; }

// Operands made of aligned 16-byte pieces: the caller's memory where it is, padded copies in the workspace where it is not.
struct Operands {
  Arena& ar;
  PadParams p{};
  int n = 0;
  long long most = 0;   // pieces of the largest copy
  OpMat get(const vtc_mat* m, int64_t rows, int cols, bool force = false) {
    if (!force && pieces_ok(m, cols)) return OpMat{(const h16*)m->p, m->row};
    const int d = up8(cols);
    h16* c = ar.take<h16>((size_t)rows * d);
    p.j[n++] = PadJob{(const h16*)m->p, c, m->row, rows, cols, d};
    most = std::max<long long>(most, rows * (d / 8));
    return OpMat{c, d};
  }
  void copy(hipStream_t s) const {
    if (most) hipLaunchKernelGGL(pad_copy_kernel, dim3((unsigned)std::min<long long>((most + 255) / 256, 65536), (unsigned)n), dim3(256), 0, s, p);
  }
};

// Column-group width of a product's tile order: see launch_gemm256
int group_of(int tiles_m, int tiles_n, double a_bytes, double w_bytes, double w_group_bytes) {
  const double rounds = (double)tiles_m * tiles_n / 256.0;
  double best = 1e300;
  int r = tiles_n;
  for (int g = 1; g <= tiles_n; ++g) {
    if (tiles_n % g) continue;
    const bool fits = g * w_group_bytes <= 2.5e6;
    const double est = a_bytes * (tiles_n / g) + w_bytes * 8.0 * (fits ? 1.0 : (rounds > 1.0 ? rounds : 1.0));
    if (est < best) { best = est; r = g; }
  }
  return r;
}


void finish_prob(OpProb& q, bool small, int bm, int bn, int K, int tile0, int w_rows = 0) {   // w_rows: rows of B behind a tile, if not bn
  q.tiles_m = div_up(q.M, bm);
  q.tiles_n = div_up(q.N, bn);
  q.group_n = small ? q.tiles_n : group_of(q.tiles_m, q.tiles_n, 2.0 * q.M * K, 2.0 * q.N * K, 2.0 * (w_rows ? w_rows : bn) * K);
  q.tile0 = tile0;
}
void set_k(OpGemmParams& p, const OgPlan& plan, int k0, int k1 = 0) {
  p.K[0] = k0; p.K[1] = k1;
  p.nk = div_up(k0, 64) + div_up(k1, 64);
  if (!plan.small) p.nk = (p.nk + 1) & ~1;   // op_gemm_kernel takes K-tiles in pairs; one behind the end reads as zero
  p.splits = plan.splits; p.kps = plan.splits == 1 ? p.nk : plan.kps;
}
template <bool F16, bool AKS, bool BKS, int EPI, int BN> void launch_og(const OpGemmParams& p, bool small, hipStream_t s) {
  const int units = p.ntiles * p.splits;
  if (small) hipLaunchKernelGGL((op_small_kernel<F16, AKS, BKS, EPI>), dim3((unsigned)units), dim3(256), 0, s, p);
  else if constexpr (EPI != OG_PART || AKS)   // 256-wide tiles are split over K for the weights' gradients only
    hipLaunchKernelGGL((op_gemm_kernel<F16, AKS, BKS, EPI, BN>), dim3((unsigned)std::min(units, 256)), dim3(512), 0, s, p);
}
template <bool F16> void launch_reduce(const ReduceParams& r, hipStream_t s) {
  if (r.nr + r.nc == 0) return;
  long long most = 1;   // blocks in x
  for (int i = 0; i < r.nr; ++i) most = std::max(most, std::min<long long>((r.r[i].rows * (r.r[i].pitch / 4) + 255) / 256, 16384));
  for (int i = 0; i < r.nc; ++i) most = std::max<long long>(most, (r.c[i].cols + 15) / 16);
  hipLaunchKernelGGL((reduce_kernel<F16>), dim3((unsigned)most, (unsigned)(r.nr + r.nc)), dim3(256), 0, s, r);
}
template <bool F16, bool GATE> void launch_skinny(const SkinnyParams& p, hipStream_t s) {
  const dim3 grid((unsigned)((p.N + 15) / 16)), block(512);
  if (p.M <= 16) hipLaunchKernelGGL((skinny_kernel<F16, 1, GATE>), grid, block, 0, s, p);
  else hipLaunchKernelGGL((skinny_kernel<F16, 2, GATE>), grid, block, 0, s, p);
}
template <typename F> void by_f16(int dtype, F&& f) {
  if (dtype == OP_F16) f(std::true_type{});
  else f(std::false_type{});
}

struct GateOut { h16* h; Saved24 s, a; };   // s.hi: null where no backward pass follows
template <bool F16> void gate_up(int64_t M, int K, int F, OpMat x, OpMat wg, OpMat wu, const void* bg, const void* bu, int bias_f32, int act, GateOut o,
                                 bool skinny, hipStream_t s) {
  const int F8 = up8(F);
  if (skinny) {
    SkinnyParams p{};
    p.x = x.p; p.ldx = x.ld; p.w0 = wg.p; p.w1 = wu.p; p.ldw = wg.ld;
    p.M = (int)M; p.K = K; p.N = F8; p.Nb = F; p.b0 = bg; p.b1 = bu; p.bias_f32 = bias_f32; p.act = act;
    p.out = o.h; p.s = o.s; p.a = o.a; p.ldo = F8;
    launch_skinny<F16, true>(p, s);
    return;
  }
  const bool save = o.s.hi != nullptr;
  const OgPlan plan = plan_gate(M, K, F8, save);
  OpGemmParams p{};
  p.nprob = 1;
  OpProb& q = p.prob[0];
  q.a[0] = x; q.b[0] = wg; q.b[1] = wu; q.c = o.h; q.ldc = F8; q.M = (int)M; q.N = F8; q.Nb = F; q.cvec = 1;
  finish_prob(q, plan.small, plan.small ? 128 : 256, plan.small ? 32 : 128, K, 0, 256);
  p.ntiles = q.tiles_m * q.tiles_n;
  set_k(p, plan, K);
  p.bias = bg; p.bias2 = bu; p.bias_f32 = bias_f32; p.act = act; p.s = o.s; p.a = o.a; p.ldg = F8;
  if (save) launch_og<F16, false, false, OG_GATE_SAVE, 256>(p, plan.small, s);
  else launch_og<F16, false, false, OG_GATE, 256>(p, plan.small, s);
}

// C = A B^T (+ bias) in 16 bits for one or two operand pairs; with few tiles in K splits whose partials lie in the workspace
struct OutPlan { OgPlan plan; int N8; float* part; };
OutPlan plan_out(Arena& ar, int64_t M, int N, int nk) {
  OutPlan o{plan_rows(M, N, nk), up8(N), nullptr};
  if (o.plan.splits > 1) o.part = ar.take<float>((size_t)o.plan.splits * M * o.N8);
  return o;
}
struct OutProduct { const OpMat *a, *b; const int* k; int segs; const void* bias; int bias_f32; void* c; long long ldc; };
OpGemmParams out_params(const OutPlan& o, int64_t M, int N, const OutProduct& x) {
  const bool small = o.plan.small;
  OpGemmParams p{};
  p.nprob = 1;
  OpProb& q = p.prob[0];
  for (int i = 0; i < x.segs; ++i) { q.a[i] = x.a[i]; q.b[i] = x.b[i]; }
  q.M = (int)M; q.Nb = N; q.cvec = N % 8 == 0 && x.ldc % 8 == 0 && (uintptr_t)x.c % 16 == 0;
  if (o.part) { q.c = o.part; q.ldc = o.N8; q.N = o.N8; p.split_stride = M * o.N8; }
  else { q.c = x.c; q.ldc = x.ldc; q.N = N; }
  finish_prob(q, small, small ? 128 : 256, small ? 64 : 192, x.k[0] + (x.segs > 1 ? x.k[1] : 0), 0);
  p.ntiles = q.tiles_m * q.tiles_n;
  set_k(p, o.plan, x.k[0], x.segs > 1 ? x.k[1] : 0);
  p.bias = x.bias; p.bias_f32 = x.bias_f32;
  return p;
}
void add_out_reduce(ReduceParams& r, const OutPlan& o, const OpGemmParams& p, int64_t M, int N, const OutProduct& x) {
  if (o.part) r.r[r.nr++] = SplitReduce{o.part, (h16*)x.c, x.ldc, o.N8, M, p.split_stride, p.splits, N, p.prob[0].cvec, x.bias};
}
template <bool F16, bool BKS> void launch_out(const OutPlan& o, const OpGemmParams& p, hipStream_t s) {
  if (o.part) launch_og<F16, false, BKS, OG_PART, 192>(p, true, s);
  else launch_og<F16, false, BKS, OG_PLAIN, 192>(p, o.plan.small, s);
}

// Layout of what the forward call keeps: h, then the upper 16 bits of s and of a, then their next 8 bits
struct FfnSaved { h16* h; Saved24 s, a; };
FfnSaved ffn_saved(void* base, int64_t rows, int inner) {
  if (!base) return FfnSaved{};
  const size_t n = (size_t)rows * up8(inner), two = align256(2 * n), one = align256(n);
  char* b = (char*)base;
  return FfnSaved{(h16*)b, {(unsigned short*)(b + two), (unsigned char*)(b + 3 * two)}, {(unsigned short*)(b + 2 * two), (unsigned char*)(b + 3 * two + one)}};
}

size_t ffn_forward(const FfnArgs& a, const vtc_mat* y, void* saved, char* ws, bool launch, hipStream_t s) {
  Arena ar{ws};
  const int F8 = up8(a.F);
  Operands in{ar};
  const OpMat x = in.get(a.x, a.M, a.K);
  // gate and up share one pitch in the kernel
  const bool copy_w = a.wg->row != a.wu->row || !pieces_ok(a.wg, a.K) || !pieces_ok(a.wu, a.K);
  const OpMat wg = in.get(a.wg, a.F, a.K, copy_w), wu = in.get(a.wu, a.F, a.K, copy_w);
  const OpMat wd = in.get(a.wd, a.N, a.F);
  const FfnSaved sv = ffn_saved(saved, a.M, a.F);
  h16* h = saved ? sv.h : ar.take<h16>((size_t)a.M * F8);
  const bool skinny = a.M <= kSkinnyRows;
  OutPlan out{};
  if (!skinny) out = plan_out(ar, a.M, a.N, div_up(a.F, 64));
  if (!launch) return ar.used;
  in.copy(s);
  by_f16(a.dtype, [&](auto f) {
    constexpr bool F16 = decltype(f)::value;
    gate_up<F16>(a.M, a.K, a.F, x, wg, wu, a.bg, a.bu, a.bias_f32, a.act, GateOut{h, sv.s, sv.a}, skinny, s);
    if (skinny) {
      SkinnyParams p{};
      p.x = h; p.ldx = F8; p.w0 = p.w1 = wd.p; p.ldw = wd.ld;
      p.M = (int)a.M; p.K = a.F; p.N = p.Nb = a.N; p.b0 = a.bd; p.bias_f32 = a.bias_f32; p.out = (h16*)y->p; p.ldo = y->row;
      launch_skinny<F16, false>(p, s);
    } else {
      const OpMat hm{h, F8};
      const OutProduct x{&hm, &wd, &a.F, 1, a.bd, a.bias_f32, (void*)y->p, y->row};
      const OpGemmParams p = out_params(out, a.M, a.N, x);
      launch_out<F16, false>(out, p, s);
      ReduceParams r{};
      r.bias_f32 = a.bias_f32;
      add_out_reduce(r, out, p, a.M, a.N, x);
      launch_reduce<F16>(r, s);
    }
  });
  return ar.used;
}

size_t ffn_backward(const FfnArgs& a, const vtc_mat* dy, const void* saved, const vtc_ffn_grads* o, char* ws, bool launch, hipStream_t s) {
  Arena ar{ws};
  const int K8 = up8(a.K), F8 = up8(a.F), N8 = up8(a.N);
  const int M = (int)a.M;
  Operands in{ar};
  const OpMat x = in.get(a.x, a.M, a.K), y = in.get(dy, a.M, a.N);
  const bool copy_w = a.wg->row != a.wu->row || !pieces_ok(a.wg, a.K) || !pieces_ok(a.wu, a.K);
  const OpMat wg = in.get(a.wg, a.F, a.K, copy_w), wu = in.get(a.wu, a.F, a.K, copy_w);
  const OpMat wd = in.get(a.wd, a.N, a.F);
  h16 *dg = ar.take<h16>((size_t)a.M * F8), *du = ar.take<h16>((size_t)a.M * F8);
  // dh and what it turns into
  const OgPlan dplan = plan_dgate(M, a.N, F8);
  const long long parts = dplan.small ? 4ll * div_up(M, 128) : 2ll * div_up(M, 256);
  const int row_blocks = div_up(M, kColRows);
  float* cs_f = (o->db_gate || o->db_up) || !launch ? ar.take<float>((size_t)2 * parts * F8) : nullptr;
  float* cs_n = o->db_down || !launch ? ar.take<float>((size_t)row_blocks * N8) : nullptr;
  const OutPlan xplan = plan_out(ar, M, a.K, 2 * div_up(a.F, 64));
  // weights' gradients: few output tiles, a long contraction over the rows, so in K splits
  OpGemmParams w{};
  w.nprob = 3;
  const h16* as[3] = {dg, du, y.p};
  const long long lda[3] = {F8, F8, y.ld};
  const h16* bs[3] = {x.p, x.p, launch ? ffn_saved((void*)saved, a.M, a.F).h : nullptr};
  const long long ldb[3] = {x.ld, x.ld, F8};
  const int rows[3] = {a.F, a.F, a.N}, cols[3] = {a.K, a.K, a.F}, pitch[3] = {K8, K8, F8};
  const long long one = (long long)a.F * K8;
  w.split_stride = 2 * one + (long long)a.N * F8;
  const OgPlan wplan = plan_weights(M, a.K, a.F, a.N);
  int tiles = 0;
  for (int i = 0; i < 3; ++i) {
    OpProb& q = w.prob[i];
    q.a[0] = OpMat{as[i], lda[i]}; q.b[0] = OpMat{bs[i], ldb[i]};
    q.M = rows[i]; q.N = pitch[i]; q.Nb = cols[i]; q.ldc = pitch[i];
    finish_prob(q, wplan.small, wplan.small ? 128 : 256, wplan.small ? 64 : 256, M, tiles);
    tiles += q.tiles_m * q.tiles_n;
  }
  w.ntiles = tiles;
  set_k(w, wplan, M);
  float* part = o->dw_gate || !launch ? ar.take<float>((size_t)w.splits * w.split_stride) : nullptr;
  if (!launch) return ar.used;
  in.copy(s);
  for (int i = 0; i < 3; ++i) w.prob[i].c = part + i * one;

  const FfnSaved sv = ffn_saved((void*)saved, a.M, a.F);
  by_f16(a.dtype, [&](auto f) {
    constexpr bool F16 = decltype(f)::value;
    OpGemmParams d{};
    d.nprob = 1;
    OpProb& e = d.prob[0];
    e.a[0] = y; e.b[0] = wd; e.M = M; e.N = F8; e.Nb = a.F; e.ldc = F8;
    finish_prob(e, dplan.small, dplan.small ? 128 : 256, dplan.small ? 64 : 192, a.N, 0);
    d.ntiles = e.tiles_m * e.tiles_n;
    set_k(d, dplan, a.N);
    d.s = sv.s; d.a = sv.a; d.dg = dg; d.du = du; d.ldg = F8; d.colsum = cs_f;
    launch_og<F16, false, true, OG_DGATE, 192>(d, dplan.small, s);
    ReduceParams r{};
    r.bias_f32 = a.bias_f32;
    const OpMat xa[2] = {{dg, F8}, {du, F8}}, xb[2] = {wg, wu};
    const int xk[2] = {a.F, a.F};
    const OutProduct xp{xa, xb, xk, 2, nullptr, 0, o->dx, o->dx_row};
    const OpGemmParams dx = out_params(xplan, M, a.K, xp);
    const int col_blocks = (N8 / 8 + 63) / 64;
    const ColSumParams cs{y.p, y.ld, M, cs_n, N8, a.N, row_blocks, cs_n ? row_blocks * col_blocks : 0};
    const long long joint = (long long)w.ntiles * w.splits + (long long)dx.ntiles * dx.splits + cs.blocks;
    if (o->dx && part && xplan.plan.small && wplan.small && joint <= kMaxBlocks) {
      const SmallGradsParams g{w, dx, cs, (unsigned)(w.ntiles * w.splits), (unsigned)(dx.ntiles * dx.splits)};
      const dim3 grid((unsigned)joint);
      if (xplan.part) hipLaunchKernelGGL((small_grads_kernel<F16, OG_PART>), grid, dim3(256), 0, s, g);
      else hipLaunchKernelGGL((small_grads_kernel<F16, OG_PLAIN>), grid, dim3(256), 0, s, g);
    } else {
      if (o->dx) launch_out<F16, true>(xplan, dx, s);
      if (part) launch_og<F16, true, true, OG_PART, 256>(w, wplan.small, s);
      if (cs_n) hipLaunchKernelGGL((colsum_kernel<F16>), dim3((unsigned)cs.blocks), dim3(256), 0, s, cs);
    }
    if (o->dx) add_out_reduce(r, xplan, dx, M, a.K, xp);
    void* outs[3] = {o->dw_gate, o->dw_up, o->dw_down};
    for (int i = 0; i < 3 && part; ++i)
      r.r[r.nr++] = SplitReduce{part + i * one, (h16*)outs[i], cols[i], pitch[i], rows[i], w.split_stride, w.splits, cols[i],
                                cols[i] % 8 == 0 && (uintptr_t)outs[i] % 16 == 0, nullptr};
    auto add = [&](const float* src, void* out, long long count, int pitch_, int c) {
      if (out) r.c[r.nc++] = ColReduce{src, out, count, pitch_, c};
    };
    add(cs_f, o->db_gate, parts, F8, a.F);
    add(cs_f ? cs_f + (size_t)parts * F8 : nullptr, o->db_up, parts, F8, a.F);
    add(cs_n, o->db_down, row_blocks, N8, a.N);
    launch_reduce<F16>(r, s);
  });
  return ar.used;
}

}  // namespace

void vtc::launch_gated_up(int dtype, int64_t M, int K, int F, const unsigned short* x, const unsigned short* wg, const unsigned short* wu, const float* bg,
                          const float* bu, int act, unsigned short* h, hipStream_t s) {
  by_f16(dtype, [&](auto f) {
    gate_up<decltype(f)::value>(M, K, F, OpMat{x, K}, OpMat{wg, K}, OpMat{wu, K}, bg, bu, 1, act, GateOut{h, {}, {}}, false, s);
  });
}

extern "C" int64_t vtc_gated_ffn_workspace(int64_t rows, int32_t width, int32_t inner, int32_t out_width, int32_t backward) {
  if (rows < 0 || rows > (1ll << 31) - 256 || width < 1 || inner < 1 || out_width < 1 || width > kFfnMaxDim || inner > kFfnMaxDim || out_width > kFfnMaxDim) {
    fail_handleless(VTC_ERR_ARG, "gated ffn: bad sizes");
    return VTC_ERR_ARG;
  }
  if (rows == 0) return 0;
  const vtc_mat odd{(const void*)2, 1};   // operands that all have to be copied: enough for every alignment
  const FfnArgs a{OP_F16, 0, 0, rows, width, inner, out_width, &odd, &odd, &odd, &odd, nullptr, nullptr, nullptr};
  vtc_ffn_grads o{};
  return (int64_t)(backward ? ffn_backward(a, &odd, nullptr, &o, nullptr, false, nullptr) : ffn_forward(a, nullptr, nullptr, nullptr, false, nullptr));
}

extern "C" int64_t vtc_gated_ffn_saved(int64_t rows, int32_t inner) {
  if (rows < 0 || inner < 1 || inner > kFfnMaxDim || rows > (1ll << 31) - 256) { fail_handleless(VTC_ERR_ARG, "gated ffn: bad sizes"); return VTC_ERR_ARG; }
  const size_t n = (size_t)rows * up8(inner);
  return (int64_t)(3 * align256(2 * n) + 2 * align256(n));
}

extern "C" int vtc_gated_ffn(int device, int dtype, int64_t rows, int32_t width, int32_t inner, int32_t out_width, const vtc_mat* x,
                             const vtc_mat* w_gate, const vtc_mat* w_up, const vtc_mat* w_down, const void* b_gate, const void* b_up,
                             const void* b_down, int32_t bias_f32, int32_t act, const vtc_mat* y, void* saved, int64_t saved_bytes,
                             void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "gated ffn";
  OneRow one[5];
  one[0].narrow(x, rows, width); one[1].narrow(w_gate, inner, width); one[2].narrow(w_up, inner, width); one[3].narrow(w_down, out_width, inner);
  one[4].narrow(y, rows, out_width);
  FfnArgs a{dtype, act, bias_f32, rows, width, inner, out_width, x, w_gate, w_up, w_down, b_gate, b_up, b_down};
  if (int rc = ffn_check(what, a)) return rc;
  if (int rc = ffn_check_mat(what, "y", y, rows, out_width)) return rc;
  if (rows == 0) return VTC_OK;
  const int bs = bias_f32 ? 4 : 2;
  if (int rc = ffn_apart(what, {span("y", y, rows, out_width)}, {span("x", x, rows, width), span("w_gate", w_gate, inner, width), span("w_up", w_up, inner, width),
                                span("w_down", w_down, out_width, inner), span("b_gate", b_gate, 1, 0, inner, bs), span("b_up", b_up, 1, 0, inner, bs),
                                span("b_down", b_down, 1, 0, out_width, bs)})) return rc;
  const int64_t need_s = vtc_gated_ffn_saved(rows, inner);
  if (saved && saved_bytes < need_s) return fail_handleless(VTC_ERR_CAPACITY, "%s: the saved buffer holds %lld bytes, %lld needed", what, (long long)saved_bytes, (long long)need_s);
  const size_t need = ffn_forward(a, nullptr, saved, nullptr, false, nullptr);
  if (need && (!workspace || workspace_bytes < (int64_t)need)) return fail_handleless(VTC_ERR_CAPACITY, "%s: the workspace holds %lld bytes, %lld needed", what, (long long)workspace_bytes, (long long)need);
  if ((uintptr_t)workspace % 256 || (uintptr_t)saved % 256) return fail_handleless(VTC_ERR_ARG, "%s: workspace and saved buffer must be aligned to 256 bytes", what);
  DeviceGuard guard(device);
  if (guard.rc) return guard.rc;
  ffn_forward(a, y, saved, (char*)workspace, true, (hipStream_t)stream);
  return launched(what);
}

extern "C" int vtc_gated_ffn_backward(int device, int dtype, int64_t rows, int32_t width, int32_t inner, int32_t out_width, const vtc_mat* dy,
                                      const vtc_mat* x, const vtc_mat* w_gate, const vtc_mat* w_up, const vtc_mat* w_down, const void* saved,
                                      int64_t saved_bytes, int32_t bias_f32, const vtc_ffn_grads* grads, void* workspace,
                                      int64_t workspace_bytes, void* stream) {
  const char* what = "gated ffn backward";
  OneRow one[5];
  one[0].narrow(x, rows, width); one[1].narrow(w_gate, inner, width); one[2].narrow(w_up, inner, width); one[3].narrow(w_down, out_width, inner);
  one[4].narrow(dy, rows, out_width);
  FfnArgs a{dtype, ACT_NONE, bias_f32, rows, width, inner, out_width, x, w_gate, w_up, w_down, nullptr, nullptr, nullptr};
  if (int rc = ffn_check(what, a)) return rc;
  if (int rc = ffn_check_mat(what, "dy", dy, rows, out_width)) return rc;
  if (grads && grads->db_down && (rows / kColRows + 1) * (out_width / 512 + 1) > kMaxBlocks)
    return fail_handleless(VTC_ERR_ARG, "%s: %lld rows of width %d are too many", what, (long long)rows, out_width);
  if (!grads) return fail_handleless(VTC_ERR_ARG, "%s: null argument", what);
  vtc_ffn_grads flat = *grads;
  if (rows == 1) flat.dx_row = width;
  grads = &flat;
  if (rows == 0) return fail_handleless(VTC_ERR_ARG, "%s: no rows (the gradients of nothing are zeros, which the caller has)", what);
  if ((grads->dw_gate || grads->dw_up || grads->dw_down) && !(grads->dw_gate && grads->dw_up && grads->dw_down))
    return fail_handleless(VTC_ERR_ARG, "%s: the three weight gradients go together", what);
  for (const void* p : {grads->dx, grads->dw_gate, grads->dw_up, grads->dw_down})
    if ((uintptr_t)p % 2) return fail_handleless(VTC_ERR_ARG, "%s: a gradient is not aligned to its type", what);
  if (grads->dx) {
    if (grads->dx_row < width || grads->dx_row > kMaxPitch) return fail_handleless(VTC_ERR_ARG, "%s: dx has a row pitch of %lld for %d columns", what, (long long)grads->dx_row, width);
  }
  const int bs = bias_f32 ? 4 : 2;
  for (const void* p : {grads->db_gate, grads->db_up, grads->db_down})
    if ((uintptr_t)p % bs) return fail_handleless(VTC_ERR_ARG, "%s: a gradient is not aligned to its type", what);
  if (int rc = ffn_apart(what, {span("dx", grads->dx, rows, grads->dx_row, width, 2), span("dw_gate", grads->dw_gate, inner, width, width, 2),
                                span("dw_up", grads->dw_up, inner, width, width, 2), span("dw_down", grads->dw_down, out_width, inner, inner, 2),
                                span("db_gate", grads->db_gate, 1, 0, inner, bs), span("db_up", grads->db_up, 1, 0, inner, bs), span("db_down", grads->db_down, 1, 0, out_width, bs)},
                         {span("x", x, rows, width), span("dy", dy, rows, out_width), span("w_gate", w_gate, inner, width), span("w_up", w_up, inner, width),
                          span("w_down", w_down, out_width, inner)})) return rc;
  const int64_t need_s = vtc_gated_ffn_saved(rows, inner);
  if (!saved || saved_bytes < need_s) return fail_handleless(VTC_ERR_CAPACITY, "%s: the saved buffer of the forward call holds %lld bytes, %lld needed", what, (long long)saved_bytes, (long long)need_s);
  const size_t need = ffn_backward(a, dy, nullptr, grads, nullptr, false, nullptr);
  if (!workspace || workspace_bytes < (int64_t)need) return fail_handleless(VTC_ERR_CAPACITY, "%s: the workspace holds %lld bytes, %lld needed", what, (long long)workspace_bytes, (long long)need);
  if ((uintptr_t)workspace % 256 || (uintptr_t)saved % 256) return fail_handleless(VTC_ERR_ARG, "%s: workspace and saved buffer must be aligned to 256 bytes", what);
  DeviceGuard guard(device);
  if (guard.rc) return guard.rc;
  ffn_backward(a, dy, saved, grads, (char*)workspace, true, (hipStream_t)stream);
  return launched(what);
}
