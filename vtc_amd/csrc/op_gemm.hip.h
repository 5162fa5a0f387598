// Matrix products of the gated feed-forward block, any sizes: 256 x BN x 64 tiles, 8 waves, persistent, the schedule of
// gemm256.hip.h (two K-tile buffers in LDS, four half-tiles, one half-tile prefetched per phase, counted vmcnt, staggered wave
// rows) with three differences:
//   * operands are fetched through buffer descriptors of the half-tile: rows and K beyond the matrix read as zero, so no size has to
//     divide anything but 8 (16-byte pieces), and the 32-bit offsets are relative to the tile (matrices beyond 4 GiB work).  Only
//     the descriptor's base moves along K;
//   * an operand may be stored with the contraction index along its ROWS ("KS": dy^T h, dg^T x, dy W_down).  Its half-tile is 64
//     k-rows x 128 columns (256 B each); ds_read_b64_tr_b16 hands every lane 4 k of one column, so two of them make the fragment
//     that one ds_read_b128 reads from the other layout and nothing is transposed in memory.  32-byte pieces of a k-row are
//     XOR-swizzled by (k & 3) | (k >> 3 & 1) << 2: the 8 k-rows a half-wave reads fall into 8 different pieces;
//   * the contraction may run over two operand pairs (dx = dg W_gate + du W_up) or be split over K into fp32 partials.
//
// Bound: the matrix pipes in the K loop, memory in the epilogues that keep or read slopes.  Measured, 16384 x 768 x 2048: gate and up
// 109 us (945 TFLOP/s), down 59 (873), dx over two pairs 109 (945), weights' gradients 165 (937); a library product of such a shape
// reaches 1100 - 1170, one of 8192^3 1473.  With slopes kept gate and up take 147 us (201 MB more), dg and du 149 us (51 GFLOP and
// 335 MB of slopes and gradients; two blocks per CU, half the CUs started late and slopes loaded ahead of the K loop change nothing).
//
// Accumulators hold C^T: lane (fr, fq) has row i * 16 + fr and, of each 32-column group, columns 8 fq .. + 8.
#pragma once
#include "common.hip.h"
#include "gemm256.hip.h"
#include "op_act.hip.h"
#include "op_extent.h"

namespace vtc {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

// What the backward pass multiplies dh by, kept in 24 bits (the upper ones of fp32: 16 in one array, 8 in another).  Rounded to
// the operands' type, dx and the weights' gradients would carry that rounding on top of dg's own and the result's
// (bf16: 3.1e-3 of the norm instead of 2.4e-3, the result's own being 1.7e-3); a byte more per value removes it.
struct Saved24 { unsigned short* hi; unsigned char* lo; };

struct OpMat {
  const h16* p;
  long long ld;   // elements between rows of the stored matrix (a multiple of 8)
};
// One product C[M, N] (+)= A B^T.  Stored shapes: A is [M][K] (or [K][M] when KS), B is [N][K] (or [K][N]).
struct OpProb {
  OpMat a[2], b[2];
  void* c;
  long long ldc;
  int M, N, Nb;    // N: columns of C that are written; Nb: rows (KS: columns) of B that exist (C's padding columns come out as zero)
  int tiles_m, tiles_n, group_n, tile0;   // tile0: index of the problem's first tile in the launch
  int cvec;        // columns of a row of c start 16-byte aligned: whole-vector stores
};
enum : int { OG_PLAIN = 0,   // 16-bit C (+ bias)
             OG_PART = 1,    // fp32 partial of a K split
             OG_GATE = 2,    // b[0] = W_gate, b[1] = W_up: h = act(g) u
             OG_GATE_SAVE = 3,   // the same, and what the backward pass needs: s = u act'(g) and a = act(g)
             OG_DGATE = 4 }; // C = dh: dg = dh s, du = dh a, and their column sums
constexpr bool og_gate(int epi) { return epi == OG_GATE || epi == OG_GATE_SAVE; }
struct OpGemmParams {
  OpProb prob[3];
  int nprob, ntiles;          // ntiles: tiles of all problems
  int K[2], nk0, nk;          // contraction lengths of the two segments; K-tiles of the first, of both (even)
  int splits, kps;            // K splits, K-tiles of a split (even); split s covers [s kps, min(nk, (s + 1) kps))
  long long split_stride;     // elements between partials
  const void *bias, *bias2;   // OG_PLAIN: bias; OG_GATE: b_gate, b_up (type: bias_f32 ? fp32 : the operands')
  int bias_f32, act;
  Saved24 s, a;               // OG_GATE_SAVE: written, OG_DGATE: read
  h16 *dg, *du;               // OG_DGATE
  long long ldg;              // pitch of h, s, a, dg, du
  float* colsum;              // OG_DGATE: [2][parts][ldg] sums of dg, du over the rows of a tile that one wave row holds (two parts per
                              // 256-row tile, four per 128-row tile), or null
};

__device__ __forceinline__ float op_bias(const void* b, int i, int f32, bool f16) {
  if (!b) return 0.f;
  if (f32) {
    const unsigned v = ((const unsigned*)b)[i];
    return __uint_as_float((v & 0x7fffffffu) > 0x7f800000u ? 0x7fc00000u : v);   // a NaN whose low bits survive store24's rounding
  }
  const h16 v = ((const h16*)b)[i];
  return f16 ? from_h16<true>(v) : from_h16<false>(v);
}

typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
constexpr unsigned kOob = 0x80000000u;   // a buffer offset that is out of range of every descriptor used here

// The output side of a tile: descriptors of [rows x cols left] windows, stores that drop what lies outside.
template <bool F16> struct OpTile {
  long long m0;
  int n0, rows, cols, bcols;   // rows of the tile that exist; columns left from n0, and those of them that have a bias
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const void* base, long long ld, int es) const {
    return __builtin_amdgcn_make_buffer_rsrc((void*)((const char*)base + (m0 * ld + n0) * es), 0, ((rows - 1) * (int)ld + cols) * es, 0x00020000);
  }
  __device__ __forceinline__ unsigned off(long long ld, int r, int c, int es) const {
    return (r < rows && c < cols) ? (unsigned)((r * (int)ld + c) * es) : kOob;
  }
  // N (4 or 8) consecutive values: one store where rows start aligned, else one by one
  template <int N> __device__ __forceinline__ void store(__amdgpu_buffer_rsrc_t rs, long long ld, int vec, int r, int c, const float* v) const {
    if (vec) {
      const unsigned o = off(ld, r, c, 2);
      if constexpr (N == 8)
        __builtin_amdgcn_raw_buffer_store_b128(u32x4{pack2<F16>(v[0], v[1]), pack2<F16>(v[2], v[3]), pack2<F16>(v[4], v[5]), pack2<F16>(v[6], v[7])}, rs, o, 0, 0);
      else
        __builtin_amdgcn_raw_buffer_store_b64(u32x2{pack2<F16>(v[0], v[1]), pack2<F16>(v[2], v[3])}, rs, o, 0, 0);
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k) __builtin_amdgcn_raw_buffer_store_b16(to_h16<F16>(v[k]), rs, off(ld, r, c + k, 2), 0, 0);
    }
  }
  template <int N> __device__ __forceinline__ void store32(__amdgpu_buffer_rsrc_t rs, long long ld, int r, int c, const float* v) const {
#pragma unroll
    for (int h = 0; h < N / 4; ++h)
      __builtin_amdgcn_raw_buffer_store_b128(u32x4{__float_as_uint(v[4 * h]), __float_as_uint(v[4 * h + 1]), __float_as_uint(v[4 * h + 2]), __float_as_uint(v[4 * h + 3])},
                                             rs, off(ld, r, c + 4 * h, 4), 0, 0);
  }
  // 8 values in 24 bits (round half away; inf stays, and so does a NaN whose low bits are clear: those of 16-bit values, of the matrix
  // instructions and of op_bias)
  __device__ __forceinline__ void store24(__amdgpu_buffer_rsrc_t hi, __amdgpu_buffer_rsrc_t lo, long long ld, int r, int c, const float* v) const {
    unsigned b[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) b[k] = __float_as_uint(v[k]) + 0x80u;
    u32x4 h;
    u32x2 l;
#pragma unroll
    for (int k = 0; k < 4; ++k) h[k] = (b[2 * k] >> 16) | (b[2 * k + 1] & 0xffff0000u);
#pragma unroll
    for (int k = 0; k < 2; ++k)
      l[k] = (b[4 * k] >> 8 & 0xffu) | (b[4 * k + 1] & 0xff00u) | (b[4 * k + 2] << 8 & 0xff0000u) | (b[4 * k + 3] << 16 & 0xff000000u);
    __builtin_amdgcn_raw_buffer_store_b128(h, hi, off(ld, r, c, 2), 0, 0);
    __builtin_amdgcn_raw_buffer_store_b64(l, lo, off(ld, r, c, 1), 0, 0);
  }
  static __device__ __forceinline__ float value24(const u32x4& h, const u32x2& l, int k) {
    const unsigned top = k & 1 ? h[k >> 1] & 0xffff0000u : h[k >> 1] << 16;
    return __uint_as_float(top | ((l[k >> 2] >> (8 * (k & 3)) & 0xffu) << 8));
  }
};
// run(integral_constant<ACT>) for the run-time activation
template <typename F> __device__ __forceinline__ void og_by_act(int act, F&& run) {
  if (act == ACT_GELU) run(std::integral_constant<int, ACT_GELU>{});
  else if (act == ACT_SILU) run(std::integral_constant<int, ACT_SILU>{});
  else if (act == ACT_SIGMOID) run(std::integral_constant<int, ACT_SIGMOID>{});
  else run(std::integral_constant<int, ACT_NONE>{});
}
// One row group of the gate / up epilogue: 8 columns of g and u (without bias) -> h, and s, a where they are kept
template <bool F16, bool SAVE> struct OgGate {
  const OpGemmParams& p;
  const OpTile<F16>& t;
  float bg[8], bu[8];
  __amdgpu_buffer_rsrc_t rh, rsh, rsl, rah, ral;
  __device__ __forceinline__ OgGate(const OpGemmParams& p_, const OpTile<F16>& t_, void* h, int c) : p(p_), t(t_) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      bg[k] = c + k < t.bcols ? op_bias(p.bias, t.n0 + c + k, p.bias_f32, F16) : 0.f;
      bu[k] = c + k < t.bcols ? op_bias(p.bias2, t.n0 + c + k, p.bias_f32, F16) : 0.f;
    }
    rh = t.rsrc(h, p.ldg, 2);
    if constexpr (SAVE) { rsh = t.rsrc(p.s.hi, p.ldg, 2); rsl = t.rsrc(p.s.lo, p.ldg, 1); rah = t.rsrc(p.a.hi, p.ldg, 2); ral = t.rsrc(p.a.lo, p.ldg, 1); }
  }
  template <int ACT> __device__ __forceinline__ void row(int r, int c, const float* g_, const float* u_) const {
    float h[8], a[8], s[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float g = g_[k] + bg[k], u = u_[k] + bu[k];
      if constexpr (SAVE) {
        float d;
        op_act_grad<ACT, false>(g, a[k], d);
        s[k] = u * d;
        h[k] = a[k] * u;
      } else {
        h[k] = op_act<ACT, false>(g) * u;
      }
    }
    if constexpr (SAVE) { t.store24(rsh, rsl, p.ldg, r, c, s); t.store24(rah, ral, p.ldg, r, c, a); }
    t.template store<8>(rh, p.ldg, 1, r, c, h);
  }
};
// Gradient epilogue of 8 columns, G row groups at a time (row(g) is a group's row, dh(g, k) its value): dg, du and their column sums
template <bool F16> struct OgDgate {
  const OpGemmParams& p;
  const OpTile<F16>& t;
  __amdgpu_buffer_rsrc_t rsh, rsl, rah, ral, rdg, rdu;
  float sg[8], su[8];
  __device__ __forceinline__ OgDgate(const OpGemmParams& p_, const OpTile<F16>& t_) : p(p_), t(t_) {
    rsh = t.rsrc(p.s.hi, p.ldg, 2); rsl = t.rsrc(p.s.lo, p.ldg, 1); rah = t.rsrc(p.a.hi, p.ldg, 2); ral = t.rsrc(p.a.lo, p.ldg, 1);
    rdg = t.rsrc(p.dg, p.ldg, 2); rdu = t.rsrc(p.du, p.ldg, 2);
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int k = 0; k < 8; ++k) sg[k] = su[k] = 0.f;
  }
  template <int G, int N, typename R, typename D> __device__ __forceinline__ void groups(int c, R&& row, D&& dh) {
    u32x4 sh[G], ah[G];
    u32x2 sl[G], al[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const unsigned o2 = t.off(p.ldg, row(g), c, 2), o1 = o2 == kOob ? kOob : o2 >> 1;
      if constexpr (N == 8) {
        sh[g] = __builtin_amdgcn_raw_buffer_load_b128(rsh, o2, 0, 0);
        ah[g] = __builtin_amdgcn_raw_buffer_load_b128(rah, o2, 0, 0);
        sl[g] = __builtin_amdgcn_raw_buffer_load_b64(rsl, o1, 0, 0);
        al[g] = __builtin_amdgcn_raw_buffer_load_b64(ral, o1, 0, 0);
      } else {
        const u32x2 x = __builtin_amdgcn_raw_buffer_load_b64(rsh, o2, 0, 0), y = __builtin_amdgcn_raw_buffer_load_b64(rah, o2, 0, 0);
        sh[g] = u32x4{x[0], x[1], 0u, 0u};
        ah[g] = u32x4{y[0], y[1], 0u, 0u};
        sl[g] = u32x2{__builtin_amdgcn_raw_buffer_load_b32(rsl, o1, 0, 0), 0u};
        al[g] = u32x2{__builtin_amdgcn_raw_buffer_load_b32(ral, o1, 0, 0), 0u};
      }
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float dg[N], du[N];
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const float d = dh(g, k);
        dg[k] = d * OpTile<F16>::value24(sh[g], sl[g], k);
        du[k] = d * OpTile<F16>::value24(ah[g], al[g], k);
        sg[k] += dg[k];
        su[k] += du[k];
      }
      t.template store<N>(rdg, p.ldg, 1, row(g), c, dg);
      t.template store<N>(rdu, p.ldg, 1, row(g), c, du);
    }
  }
  // sums over the 16 rows that lanes hold, into row `part` of the partial sums (rows outside contributed 0: dh is 0 there)
  template <int N> __device__ __forceinline__ void finish(int c, int fr, long long part, long long parts) {
    if (!p.colsum) return;
#pragma unroll
    for (int k = 0; k < N; ++k) { sg[k] = row16_sum(sg[k]); su[k] = row16_sum(su[k]); }
    if (fr == 0 && c < t.cols) {
      float* dst = p.colsum + part * p.ldg + t.n0 + c;
#pragma unroll
      for (int k = 0; k < N; ++k) { dst[k] = sg[k]; dst[parts * p.ldg + k] = su[k]; }
    }
  }
};

// Two transposed LDS reads: 4 + 4 contraction indices of the lane's column.  The restrict parameters give the reads alias
// information; without any, the compiler drains every copy to LDS in flight (vmcnt(0)) in front of each of them.
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
__device__ __forceinline__ u16x8 tr_frag(const lds_s16x4* __restrict__ a, const lds_s16x4* __restrict__ b) {
  const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)a);
  const s16x4 v2 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)b);
  return __builtin_bit_cast(u16x8, __builtin_shufflevector(v1, v2, 0, 1, 2, 3, 4, 5, 6, 7));
}

template <bool F16, bool AKS, bool BKS, int EPI, int BN>
__global__ __launch_bounds__(512, 2) void op_gemm_kernel(const OpGemmParams p) {
  using TC = Tile256<BN>;
  constexpr int NJ1 = TC::NJ1;
  static_assert(!og_gate(EPI) || BN == 256, "gate and up columns sit in the two halves of a tile");
  __shared__ __attribute__((aligned(16))) char smem[TC::SMEM];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 2, wn = wave & 3;
  const int fr = lane & 15, fq = lane >> 4;
  // ---- staging.  Lane offsets are bytes from a half-tile's origin and the same for every tile; what changes per tile and K-tile is
  // scalar: the origin, the bytes that exist behind it and the contraction that is left.
  const int lr = lane >> 3, lc = lane & 7;
  unsigned va[2], vb[2], vb1[1];     // of the two instructions of a half-tile (vb1: B1's one instruction where BN = 192)
  int pca[2], pcb[2], pcb1[1];       // KC: k of the lane's 16-byte piece inside the K-tile
  constexpr int NSEG = (EPI == OG_PLAIN && BKS) ? 2 : 1;   // dx sums over two operand pairs
  constexpr bool MULTI = AKS;                              // several problems in one launch: the weights' gradients
  struct Stream {     // what a half-tile's copies need, all scalar; a step is a 64-bit add and a subtraction
    const char* p;    // origin of the next K-tile's half
    int end;          // KC: descriptor size, up to the end of the last row's pieces (rows beyond read as zero, k beyond K is masked per
                      // lane).  KS: bytes of the last k-row less a pitch; k-rows beyond K read as zero, columns beyond the matrix run
                      // into the next k-row and end in rows or columns of C that are not stored.
    int left;         // KC: k left, in whole pieces; KS: k-rows left
    int seg;
  };
  Stream sa0, sa1, sb0, sb1;
  int lda2 = 0, ldb2 = 0;   // pitches in bytes

  auto unit = [&](unsigned t, int& pi, int& tm, int& tn, int& k0, int& k1) {   // work unit -> problem, tile, K-tiles
    const unsigned ti = t / (unsigned)p.splits;
    const int s = (int)(t - ti * (unsigned)p.splits);
    pi = 0;
    if constexpr (MULTI) {
      if (p.nprob > 1 && (int)ti >= p.prob[1].tile0) pi = 1;
      if (p.nprob > 2 && (int)ti >= p.prob[2].tile0) pi = 2;
    }
    const OpProb& q = p.prob[pi];
    const unsigned r0 = ti - (unsigned)q.tile0, per = (unsigned)(q.tiles_m * q.group_n);
    const unsigned g = r0 / per, r = r0 - g * per;
    tm = (int)(r / (unsigned)q.group_n);
    tn = (int)(g * (unsigned)q.group_n + r % (unsigned)q.group_n);
    k0 = s * p.kps;
    k1 = min(p.nk, k0 + p.kps);
  };
  auto half_kc = [&](Stream& d, const h16* base, long long ld, int row0, int rows, int k0, int K) {   // rows: left from row0
    const int K8 = (K + 7) & ~7;
    d.p = (const char*)(base + (long long)row0 * ld + k0);
    d.end = rows > 0 ? (min(rows, 128) - 1) * (int)ld * 2 + K8 * 2 : 0;
    d.left = K8 - k0;
  };
  auto half_ks = [&](Stream& d, const h16* base, long long ld, int col0, int cols, int k0, int K) {   // cols: left from col0
    d.p = (const char*)(base + (long long)k0 * ld + col0);
    d.end = __builtin_amdgcn_readfirstlane(ks_end(cols, 128, (int)ld));   // (clamps are vector instructions)
    d.left = ks_left(cols, K, k0);
  };
  int cur_tm = 0, cur_tn = 0;   // tile being staged
  // operand A (half h) / B (half h) of segment s from contraction index k0 on
  auto set_a = [&](Stream& d, const OpProb& q, int h, int s, int k0) {
    const int r0 = cur_tm * 256 + h * 128;
    if constexpr (AKS) half_ks(d, q.a[s].p, q.a[s].ld, r0, q.M - r0, k0, p.K[s]);
    else half_kc(d, q.a[s].p, q.a[s].ld, r0, q.M - r0, k0, p.K[s]);
    d.seg = s;
  };
  auto set_b = [&](Stream& d, const OpProb& q, int h, int s, int k0) {
    const OpMat B = og_gate(EPI) ? q.b[h] : q.b[s];
    const int c0 = og_gate(EPI) ? cur_tn * 128 : cur_tn * BN + h * 128;
    if constexpr (BKS) half_ks(d, B.p, B.ld, c0, q.Nb - c0, k0, p.K[s]);
    else half_kc(d, B.p, B.ld, c0, q.Nb - c0, k0, p.K[s]);
    d.seg = s;
  };
  auto lane_offsets = [&](int pi) {
    const OpProb& q = p.prob[MULTI ? pi : 0];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = (wave * 2 + i) * 8 + lr;                 // KC: row of the half-tile, place lc holds piece lc ^ swz(r)
      const int ch = lc ^ lds_swz(r);
      const int kr = (wave * 2 + i) * 4 + (lane >> 4);       // KS: k-row of the half-tile
      const int sw = (kr & 3) | ((kr >> 3 & 1) << 2);
      const int cc = ((((lane & 15) >> 1) ^ sw) << 1) | (lane & 1);
      pca[i] = AKS ? cc * 8 : ch * 8;
      va[i] = AKS ? (unsigned)(kr * (int)q.a[0].ld * 2 + cc * 16) : (unsigned)(r * (int)q.a[0].ld * 2 + ch * 16);
      const int wr = (r & ~31) + perm32(r & 31);
      pcb[i] = BKS ? cc * 8 : ch * 8;
      vb[i] = BKS ? (unsigned)(kr * (int)q.b[0].ld * 2 + cc * 16) : (unsigned)(wr * (int)q.b[0].ld * 2 + ch * 16);
    }
    if constexpr (NJ1 == 1) {                                // B1 of 64 columns: 16-column groups need no permutation
      const int r = wave * 8 + lr, ch = lc ^ lds_swz(r);
      const int sw = (r >> 1 & 1) | ((r >> 3 & 1) << 1);     // KS: k-rows of 128 bytes, four 32-byte pieces
      const int cc = (((lc >> 1) ^ sw) << 1) | (lc & 1);
      pcb1[0] = (BKS ? cc : ch) * 8;
      vb1[0] = (unsigned)(r * (int)q.b[0].ld * 2 + (BKS ? cc : ch) * 16);
    }
  };
  lane_offsets(0);
  auto set_tile = [&](int pi, int tm, int tn, int k0) {   // (only products of one segment are split)
    const OpProb& q = p.prob[MULTI ? pi : 0];
    cur_tm = tm; cur_tn = tn;
    lda2 = (int)q.a[0].ld * 2; ldb2 = (int)q.b[0].ld * 2;
    set_a(sa0, q, 0, 0, k0 * 64); set_a(sa1, q, 1, 0, k0 * 64);
    set_b(sb0, q, 0, 0, k0 * 64); set_b(sb1, q, 1, 0, k0 * 64);
    if constexpr (MULTI) lane_offsets(pi);
  };

  // N copies of 16 bytes per lane to LDS (everything that does not exist arrives as zero), then one K-tile on
  auto copies = [&](auto ks, auto count, Stream& d, int ld2, const unsigned* vo, const int* piece, char* lds) {
    constexpr bool KS = decltype(ks)::value;
    const int end = KS ? __builtin_amdgcn_readfirstlane(ks_bytes(d.left, ld2, d.end)) : d.end;
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)d.p, 0, end, 0x00020000);
#pragma unroll
    for (int i = 0; i < decltype(count)::value; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, LPTR(lds + i * 1024), 16, (int)(KS || piece[i] < d.left ? vo[i] : kOob), 0, 0, 0);
    d.p += KS ? (long long)64 * ld2 : 128ll;
    d.left -= 64;
  };
  using AK = std::integral_constant<bool, AKS>;
  using BK = std::integral_constant<bool, BKS>;
  using Two = std::integral_constant<int, 2>;
  auto issue_a = [&](int h, int buf, int) {
    Stream& d = h ? sa1 : sa0;
    if constexpr (NSEG == 2) { if (d.left <= 0 && d.seg == 0) set_a(d, p.prob[0], h, 1, 0); }
    copies(AK{}, Two{}, d, lda2, va, pca, smem + buf * TC::BUF + (h ? TC::OFF_A1 : TC::OFF_A0) + wave * 2048);
  };
  auto issue_b0 = [&](int buf, int) {
    if constexpr (NSEG == 2) { if (sb0.left <= 0 && sb0.seg == 0) set_b(sb0, p.prob[0], 0, 1, 0); }
    copies(BK{}, Two{}, sb0, ldb2, vb, pcb, smem + buf * TC::BUF + TC::OFF_B0 + wave * 2048);
  };
  auto issue_b1 = [&](int buf, int) {
    if constexpr (NSEG == 2) { if (sb1.left <= 0 && sb1.seg == 0) set_b(sb1, p.prob[0], 1, 1, 0); }
    copies(BK{}, std::integral_constant<int, NJ1>{}, sb1, ldb2, NJ1 == 2 ? vb : vb1, NJ1 == 2 ? pcb : pcb1,
           smem + buf * TC::BUF + TC::OFF_B1 + wave * (NJ1 * 1024));
  };

  // ---- fragments
  const int tq = (lane & 15) >> 2, tp = lane & 3;                // KS: k inside a block of 4, piece of 4 columns
  const int ksw = tq | ((fq & 1) << 2);
  int a_off[4], b0_off[2], b1_off[NJ1], a_sw[4], b0_sw[2], b1_sw[NJ1];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = wm * 64 + i * 16 + fr;
    if constexpr (AKS) { a_off[i] = (fq * 8 + tq) * 256 + (((wm * 4 + i) ^ ksw) << 5) + 8 * tp; a_sw[i] = 0; }
    else { a_off[i] = r * 128; a_sw[i] = lds_swz(r); }
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int r = wn * 32 + j * 16 + fr;
    if constexpr (BKS) { b0_off[j] = (fq * 8 + tq) * 256 + (((wn * 2 + (tp >> 1)) ^ ksw) << 5) + (tp & 1) * 16 + 8 * j; b0_sw[j] = 0; }
    else { b0_off[j] = r * 128; b0_sw[j] = lds_swz(r); }
  }
#pragma unroll
  for (int j = 0; j < NJ1; ++j) {
    const int r = wn * (16 * NJ1) + j * 16 + fr;
    if constexpr (BKS && NJ1 == 2) { b1_off[j] = b0_off[j]; b1_sw[j] = 0; }
    else if constexpr (BKS) { b1_off[j] = (fq * 8 + tq) * 128 + ((wn ^ ((tq >> 1) | ((fq & 1) << 1))) << 5) + 8 * tp; b1_sw[j] = 0; }
    else { b1_off[j] = r * 128; b1_sw[j] = lds_swz(r); }
  }
  auto frag_kc = [&](const char* base, int off, int sw, int ks) { return *(const u16x8*)(base + off + (((ks * 4 + fq) ^ sw) << 4)); };
  auto frag_ks = [&](const char* base, int off, int ks) { return tr_frag((const lds_s16x4*)(base + off + ks * 8192), (const lds_s16x4*)(base + off + ks * 8192 + 1024)); };

  f32x4 acc0[2][4][2], acc1[2][4][NJ1];
  u16x8 fa[2][4], fb0[2][2], fb1[2][NJ1];
  auto read_a = [&](int buf, int off) {
    const char* base = smem + buf * TC::BUF + off;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int i = 0; i < 4; ++i) { if constexpr (AKS) fa[ks][i] = frag_ks(base, a_off[i], ks); else fa[ks][i] = frag_kc(base, a_off[i], a_sw[i], ks); }
  };
  auto read_b0 = [&](int buf) {
    const char* base = smem + buf * TC::BUF + TC::OFF_B0;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int j = 0; j < 2; ++j) { if constexpr (BKS) fb0[ks][j] = frag_ks(base, b0_off[j], ks); else fb0[ks][j] = frag_kc(base, b0_off[j], b0_sw[j], ks); }
  };
  auto read_b1 = [&](int buf) {
    const char* base = smem + buf * TC::BUF + TC::OFF_B1;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int j = 0; j < NJ1; ++j) {
        if constexpr (BKS && NJ1 == 2) fb1[ks][j] = frag_ks(base, b1_off[j], ks);
        else if constexpr (BKS) fb1[ks][j] = tr_frag((const lds_s16x4*)(base + b1_off[j] + ks * 4096), (const lds_s16x4*)(base + b1_off[j] + ks * 4096 + 512));
        else fb1[ks][j] = frag_kc(base, b1_off[j], b1_sw[j], ks);
      }
  };
  auto mma0 = [&](int mq) {
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc0[mq][i][j] = mfma16<F16>(fb0[ks][j], fa[ks][i], acc0[mq][i][j]);
    __builtin_amdgcn_s_setprio(0);
  };
  auto mma1 = [&](int mq) {
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < NJ1; ++j) acc1[mq][i][j] = mfma16<F16>(fb1[ks][j], fa[ks][i], acc1[mq][i][j]);
    __builtin_amdgcn_s_setprio(0);
  };
  auto sync_reads = [&]() {
    __builtin_amdgcn_s_barrier();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  auto end_phase = [&]() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
  };

  // K-tile T: quadrants (0,B0) (0,B1) (1,B1) (1,B0).  Staging order B1(T+1), A1(T+1), A0(T+2), B0(T+2), across tiles: in the last
  // two K-tiles "T+1" / "T+2" are K-tiles 0 and 1 of the block's next tile (HOOK switches the sources between phases 2 and 3).
  // Every slot is restaged at least two phases after its last read; at the K-tile boundary A0 and B0 (4 copies) stay in flight.
#define VTC_OG_KTILE(BUF, C1, K1, C2, K2, HOOK)                                     \
  {                                                                                 \
    read_b0(BUF);                                                                   \
    __builtin_amdgcn_sched_barrier(0);                                              \
    read_a(BUF, TC::OFF_A0);                                                        \
    if (C1) issue_b1((BUF) ^ 1, (K1));                                              \
    sync_reads();                                                                   \
    mma0(0);                                                                        \
    end_phase();                                                                    \
    read_b1(BUF);                                                                   \
    if (C1) issue_a(1, (BUF) ^ 1, (K1));                                            \
    sync_reads();                                                                   \
    mma1(0);                                                                        \
    end_phase();                                                                    \
    HOOK;                                                                           \
    read_a(BUF, TC::OFF_A1);                                                        \
    if (C2) issue_a(0, BUF, (K2));                                                  \
    sync_reads();                                                                   \
    mma1(1);                                                                        \
    end_phase();                                                                    \
    if (C2) {                                                                       \
      issue_b0(BUF, (K2));                                                          \
      asm volatile("s_waitcnt vmcnt(4)" ::: "memory");                              \
    } else {                                                                        \
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                              \
    }                                                                               \
    __builtin_amdgcn_s_barrier();                                                   \
    __builtin_amdgcn_sched_barrier(0);                                              \
    mma0(1);                                                                        \
    end_phase();                                                                    \
  }

  const unsigned G = gridDim.x, nunits = (unsigned)p.ntiles * (unsigned)p.splits;
  unsigned tl = blockIdx.x;
  {
    int pi, tm, tn, k0, k1;
    unit(xcd_remap(tl, nunits), pi, tm, tn, k0, k1);
    set_tile(pi, tm, tn, k0);
    issue_a(0, 0, 0); issue_b0(0, 0); issue_b1(0, 0); issue_a(1, 0, 0);
    issue_a(0, 1, 1); issue_b0(1, 1);
  }
  bool first_tile = true;
  while (tl < nunits) {
    int pi, tile_m, tile_n, k0, k1;
    const unsigned ucur = xcd_remap(tl, nunits);
    unit(ucur, pi, tile_m, tile_n, k0, k1);
    const int nk_cur = k1 - k0;
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int j = 0; j < 2; ++j) acc0[a][i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < NJ1; ++j) acc1[a][i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
    if (first_tile) {
      asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      first_tile = false;
    }
    const unsigned tl_next = tl + G;
    const bool has_next = tl_next < nunits;
    if (wm == 1) __builtin_amdgcn_s_barrier();   // wave row 1 runs one barrier behind: one row computes while the other reads
    for (int t = 0; t + 2 < nk_cur; t += 2) {
      VTC_OG_KTILE(0, true, t + 1, true, t + 2, )
      VTC_OG_KTILE(1, true, t + 2, true, t + 3, )
    }
    VTC_OG_KTILE(0, true, nk_cur - 1, has_next, 0, if (has_next) {
      int pn; int tmn; int tnn; int kn; int kn1;
      unit(xcd_remap(tl_next, nunits), pn, tmn, tnn, kn, kn1);
      set_tile(pn, tmn, tnn, kn);
    })
    VTC_OG_KTILE(1, has_next, 0, has_next, 1, )
    if (wm == 0) __builtin_amdgcn_s_barrier();
    tl = tl_next;

    // ---- epilogue.  Global accesses through descriptors of the tile: rows outside are dropped by the hardware, columns per lane.
    // The lane id comes from an opaque source: what is derived from it must not be kept in registers across the K loop.
    int el;
    asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(el));
    const int fr = el & 15, fq = el >> 4;
    const OpProb& q = p.prob[MULTI ? pi : 0];
    OpTile<F16> t;
    t.m0 = (long long)tile_m * 256;
    t.n0 = og_gate(EPI) ? tile_n * 128 : tile_n * BN;
    t.rows = min(256, q.M - tile_m * 256);
    t.cols = q.N - t.n0;
    t.bcols = q.Nb - t.n0;
    constexpr int W1 = 4 * NJ1;
    const int c0 = wn * 32 + 8 * fq;                             // columns of the tile: B0 group, B1 group
    const int c1 = og_gate(EPI) ? c0 : 128 + wn * (16 * NJ1) + W1 * fq;
    auto row_of = [&](int g) { return (g >> 2) * 128 + wm * 64 + (g & 3) * 16 + fr; };
    float v0[8], v1[W1];
    auto take = [&](int g) {
      const int mq = g >> 2, i = g & 3;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) v0[4 * j + r] = acc0[mq][i][j][r];
#pragma unroll
      for (int j = 0; j < NJ1; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) v1[4 * j + r] = acc1[mq][i][j][r];
    };
    if constexpr (EPI == OG_PLAIN) {
      float b0[8], b1[W1];
#pragma unroll
      for (int k = 0; k < 8; ++k) b0[k] = c0 + k < t.bcols ? op_bias(p.bias, t.n0 + c0 + k, p.bias_f32, F16) : 0.f;
#pragma unroll
      for (int k = 0; k < W1; ++k) b1[k] = c1 + k < t.bcols ? op_bias(p.bias, t.n0 + c1 + k, p.bias_f32, F16) : 0.f;
      const __amdgpu_buffer_rsrc_t rc = t.rsrc(q.c, q.ldc, 2);
#pragma unroll
      for (int g = 0; g < 8; ++g) {
        take(g);
#pragma unroll
        for (int k = 0; k < 8; ++k) v0[k] += b0[k];
#pragma unroll
        for (int k = 0; k < W1; ++k) v1[k] += b1[k];
        t.template store<8>(rc, q.ldc, q.cvec, row_of(g), c0, v0);
        t.template store<W1>(rc, q.ldc, q.cvec, row_of(g), c1, v1);
      }
    } else if constexpr (EPI == OG_PART) {
      // partial of this split: [M][N] fp32 with the pitch ldc (a multiple of 8)
      const __amdgpu_buffer_rsrc_t rc = t.rsrc((const float*)q.c + (long long)(ucur % (unsigned)p.splits) * p.split_stride, q.ldc, 4);
#pragma unroll
      for (int g = 0; g < 8; ++g) {
        take(g);
        t.template store32<8>(rc, q.ldc, row_of(g), c0, v0);
        t.template store32<W1>(rc, q.ldc, row_of(g), c1, v1);
      }
    } else if constexpr (og_gate(EPI)) {
      if constexpr (NJ1 == 2) {
        const OgGate<F16, EPI == OG_GATE_SAVE> gate(p, t, q.c, c0);
        og_by_act(p.act, [&](auto act) {
#pragma unroll
          for (int g = 0; g < 8; ++g) { take(g); gate.template row<decltype(act)::value>(row_of(g), c0, v0, v1); }
        });
      }
    } else {   // OG_DGATE
      OgDgate<F16> grad(p, t);
      auto half = [&](auto which, auto width) {
        constexpr bool SECOND = decltype(which)::value;
        constexpr int N = decltype(width)::value;
        grad.clear();
#pragma unroll
        for (int g0 = 0; g0 < 8; g0 += 4) {
          __builtin_amdgcn_sched_barrier(0);   // the loads of four row groups at a time: all of them would not fit the registers
          grad.template groups<4, N>(SECOND ? c1 : c0, [&](int g) { return row_of(g0 + g); }, [&](int g, int k) {
            if constexpr (SECOND) return acc1[(g0 + g) >> 2][(g0 + g) & 3][k >> 2][k & 3];
            else return acc0[(g0 + g) >> 2][(g0 + g) & 3][k >> 2][k & 3];
          });
        }
        grad.template finish<N>(SECOND ? c1 : c0, fr, tile_m * 2 + wm, q.tiles_m * 2ll);
      };
      half(std::false_type{}, std::integral_constant<int, 8>{});
      half(std::true_type{}, std::integral_constant<int, W1>{});
    }
  }
#undef VTC_OG_KTILE
}

// ---- small products: 128 x 64 tiles, 4 waves of 32 x 64, one tile per block, two blocks per CU.  A product with few 256-wide tiles
// leaves most CUs idle there; with an eighth of the tile (and K splits) the same work spreads over all of them.  Three K-tile
// buffers (A 16 KB, B 8 KB each), two in flight, one barrier per K-tile.  The contraction runs in the same order as in the kernel
// above, so an unsplit product has the same bits in either.  Measured against the 256-wide tiles: the table at og_plan.
constexpr int kOsA = 16384, kOsStage = 24576;
template <bool F16, bool AKS, bool BKS, int EPI>   // smem: 3 kOsStage bytes
__device__ __forceinline__ void op_small_tile(const OpGemmParams& p, unsigned block, unsigned blocks, char* smem) {
  constexpr bool MULTI = AKS;
  constexpr int NSEG = (EPI == OG_PLAIN || EPI == OG_PART) && BKS && !AKS ? 2 : 1;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int fr = lane & 15, fq = lane >> 4, lr = lane >> 3, lc = lane & 7;
  const unsigned u = xcd_remap(block, blocks);
  const unsigned ti = u / (unsigned)p.splits;
  const int split = (int)(u - ti * (unsigned)p.splits);
  int pi = 0;
  if constexpr (MULTI) {
    if (p.nprob > 1 && (int)ti >= p.prob[1].tile0) pi = 1;
    if (p.nprob > 2 && (int)ti >= p.prob[2].tile0) pi = 2;
  }
  const OpProb& q = p.prob[pi];
  const int tile_m = (int)((ti - (unsigned)q.tile0) / (unsigned)q.tiles_n), tile_n = (int)((ti - (unsigned)q.tile0) % (unsigned)q.tiles_n);
  const int m0 = tile_m * 128, n0 = og_gate(EPI) ? tile_n * 32 : tile_n * 64;
  const int k0 = split * p.kps, nk = min(p.nk, k0 + p.kps) - k0;

  // ---- staging (see op_gemm_kernel): wave w fetches A pieces 4 w .. + 4 and B pieces 2 w, 2 w + 1 of 1 KiB; with gate and up
  // columns side by side, waves 0 and 1 fetch W_gate rows, 2 and 3 W_up's
  unsigned va[4], vb[2];
  int pca[4], pcb[2];
  const int lda2 = (int)q.a[0].ld * 2, ldb2 = (int)q.b[0].ld * 2;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (AKS) {
      const int kr = (wave * 4 + i) * 4 + (lane >> 4), sw = (kr & 3) | ((kr >> 3 & 1) << 2);
      const int cc = ((((lane & 15) >> 1) ^ sw) << 1) | (lane & 1);
      pca[i] = cc * 8; va[i] = (unsigned)(kr * lda2 + cc * 16);
    } else {
      const int r = (wave * 4 + i) * 8 + lr, ch = lc ^ lds_swz(r);
      pca[i] = ch * 8; va[i] = (unsigned)(r * lda2 + ch * 16);
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = (wave * 2 + i) * 8 + lr;
    if constexpr (BKS) {   // 64 k-rows x 64 columns: 128-byte rows, four 32-byte pieces each
      const int sw = (r >> 1 & 1) | ((r >> 3 & 1) << 1);
      const int cc = (((lc >> 1) ^ sw) << 1) | (lc & 1);
      pcb[i] = cc * 8; vb[i] = (unsigned)(r * ldb2 + cc * 16);
    } else {
      const int ch = lc ^ lds_swz(r), wr = (og_gate(EPI) ? 0 : (r & ~31)) + perm32(r & 31);
      pcb[i] = ch * 8; vb[i] = (unsigned)(wr * ldb2 + ch * 16);
    }
  }
  struct Stream { const char* p; int end, left; };   // as in op_gemm_kernel
  Stream sa, sb;
  [[maybe_unused]] int seg = 0;
  const int a_left = q.M - m0, b_left = q.Nb - n0;
  auto stream = [&](auto ks, const OpMat& A, int at, int exist, int most, int kk, int K) {
    const int ld2 = (int)A.ld * 2, K8 = (K + 7) & ~7;
    if constexpr (decltype(ks)::value)
      return Stream{(const char*)(A.p + (long long)kk * A.ld + at), ks_end(exist, most, (int)A.ld), ks_left(exist, K, kk)};
    else
      return Stream{(const char*)(A.p + (long long)at * A.ld + kk), exist > 0 ? (min(exist, most) - 1) * ld2 + K8 * 2 : 0, K8 - kk};
  };
  using AK = std::integral_constant<bool, AKS>;
  using BK = std::integral_constant<bool, BKS>;
  auto set_seg = [&](int s, int kk) {
    sa = stream(AK{}, q.a[s], m0, a_left, 128, kk, p.K[s]);
    sb = stream(BK{}, og_gate(EPI) ? (wave >= 2 ? q.b[1] : q.b[0]) : q.b[s], n0, b_left, og_gate(EPI) ? 32 : 64, kk, p.K[s]);
    seg = s;
  };
  {
    const int nk0 = (p.K[0] + 63) / 64;
    if (NSEG == 2 && k0 >= nk0) set_seg(1, (k0 - nk0) * 64);
    else set_seg(0, k0 * 64);
  }
  auto issue = [&](int stage) {
    if constexpr (NSEG == 2) {
      if (sa.left <= 0 && seg == 0) set_seg(1, 0);
    }
    char* l = smem + stage * kOsStage;
    auto end = [](bool ks, const Stream& d, int ld2) { return ks ? __builtin_amdgcn_readfirstlane(ks_bytes(d.left, ld2, d.end)) : d.end; };
    const __amdgpu_buffer_rsrc_t ra = __builtin_amdgcn_make_buffer_rsrc((void*)sa.p, 0, end(AKS, sa, lda2), 0x00020000);
    const __amdgpu_buffer_rsrc_t rb = __builtin_amdgcn_make_buffer_rsrc((void*)sb.p, 0, end(BKS, sb, ldb2), 0x00020000);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, LPTR(l + (wave * 4 + i) * 1024), 16, (int)(AKS || pca[i] < sa.left ? va[i] : kOob), 0, 0, 0);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, LPTR(l + kOsA + (wave * 2 + i) * 1024), 16, (int)(BKS || pcb[i] < sb.left ? vb[i] : kOob), 0, 0, 0);
    sa.p += AKS ? (long long)64 * lda2 : 128ll; sa.left -= 64;
    sb.p += BKS ? (long long)64 * ldb2 : 128ll; sb.left -= 64;
  };

  // ---- fragments
  const int tq = (lane & 15) >> 2, tp = lane & 3;
  int a_off[2], a_sw[2], b_off[4], b_sw[4];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = wave * 32 + i * 16 + fr;
    if constexpr (AKS) { a_off[i] = (fq * 8 + tq) * 256 + (((wave * 2 + i) ^ (tq | ((fq & 1) << 2))) << 5) + 8 * tp; a_sw[i] = 0; }
    else { a_off[i] = r * 128; a_sw[i] = lds_swz(r); }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {   // tiles 2 g, 2 g + 1 of the 32-column group g
    const int r = j * 16 + fr;
    if constexpr (BKS) {
      const int sw = (tq >> 1) | ((fq & 1) << 1);
      b_off[j] = kOsA + (fq * 8 + tq) * 128 + ((((j >> 1) * 2 + (tp >> 1)) ^ sw) << 5) + (tp & 1) * 16 + 8 * (j & 1);
      b_sw[j] = 0;
    } else { b_off[j] = kOsA + r * 128; b_sw[j] = lds_swz(r); }
  }
  f32x4 acc[2][4];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  issue(0);
  if (nk > 1) issue(1);
  int cur = 0;
  for (int kt = 0; kt < nk; ++kt) {
    if (kt + 1 < nk) asm volatile("s_waitcnt vmcnt(6)" ::: "memory");   // the 6 copies of the next K-tile may stay in flight
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();   // this K-tile is in LDS for everybody; everybody has read the one before last's buffer
    __builtin_amdgcn_sched_barrier(0);
    const int nxt = cur == 0 ? 2 : cur - 1;   // (cur + 2) % 3
    if (kt + 2 < nk) issue(nxt);
    const char* base = smem + cur * kOsStage;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      u16x8 fa[2], fb[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (BKS) fb[j] = tr_frag((const lds_s16x4*)(base + b_off[j] + ks * 4096), (const lds_s16x4*)(base + b_off[j] + ks * 4096 + 512));
        else fb[j] = *(const u16x8*)(base + b_off[j] + (((ks * 4 + fq) ^ b_sw[j]) << 4));
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if constexpr (AKS) fa[i] = tr_frag((const lds_s16x4*)(base + a_off[i] + ks * 8192), (const lds_s16x4*)(base + a_off[i] + ks * 8192 + 1024));
        else fa[i] = *(const u16x8*)(base + a_off[i] + (((ks * 4 + fq) ^ a_sw[i]) << 4));
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = mfma16<F16>(fb[j], fa[i], acc[i][j]);
    }
    __builtin_amdgcn_sched_barrier(0);
    cur = cur == 2 ? 0 : cur + 1;
  }

  // ---- epilogue
  OpTile<F16> t;
  t.m0 = m0; t.n0 = n0;
  t.rows = min(128, q.M - m0);
  t.cols = q.N - n0;
  t.bcols = q.Nb - n0;
  const int c0 = 8 * fq, c1 = og_gate(EPI) ? c0 : 32 + 8 * fq;
  auto row_of = [&](int i) { return wave * 32 + i * 16 + fr; };
  float v0[8], v1[8];
  auto take = [&](int i) {
#pragma unroll
    for (int k = 0; k < 8; ++k) { v0[k] = acc[i][k >> 2][k & 3]; v1[k] = acc[i][2 + (k >> 2)][k & 3]; }
  };
  if constexpr (EPI == OG_PLAIN) {
    const __amdgpu_buffer_rsrc_t rc = t.rsrc(q.c, q.ldc, 2);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      take(i);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        v0[k] += c0 + k < t.bcols ? op_bias(p.bias, n0 + c0 + k, p.bias_f32, F16) : 0.f;
        v1[k] += c1 + k < t.bcols ? op_bias(p.bias, n0 + c1 + k, p.bias_f32, F16) : 0.f;
      }
      t.template store<8>(rc, q.ldc, q.cvec, row_of(i), c0, v0);
      t.template store<8>(rc, q.ldc, q.cvec, row_of(i), c1, v1);
    }
  } else if constexpr (EPI == OG_PART) {
    const __amdgpu_buffer_rsrc_t rc = t.rsrc((const float*)q.c + (long long)split * p.split_stride, q.ldc, 4);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      take(i);
      t.template store32<8>(rc, q.ldc, row_of(i), c0, v0);
      t.template store32<8>(rc, q.ldc, row_of(i), c1, v1);
    }
  } else if constexpr (og_gate(EPI)) {
    const OgGate<F16, EPI == OG_GATE_SAVE> gate(p, t, q.c, c0);
    og_by_act(p.act, [&](auto act) {
#pragma unroll
      for (int i = 0; i < 2; ++i) { take(i); gate.template row<decltype(act)::value>(row_of(i), c0, v0, v1); }
    });
  } else {
    OgDgate<F16> grad(p, t);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      grad.clear();
      grad.template groups<2, 8>(half ? c1 : c0, row_of, [&](int i, int k) { return acc[i][half * 2 + (k >> 2)][k & 3]; });
      grad.template finish<8>(half ? c1 : c0, fr, (long long)tile_m * 4 + wave, q.tiles_m * 4ll);
    }
  }
}

template <bool F16, bool AKS, bool BKS, int EPI>
__global__ __launch_bounds__(256, 2) void op_small_kernel(const OpGemmParams p) {
  __shared__ __attribute__((aligned(16))) char smem[3 * kOsStage];
  op_small_tile<F16, AKS, BKS, EPI>(p, blockIdx.x, gridDim.x, smem);
}

}  // namespace vtc
