// Tree attention and the scores of cached tokens for few rows, and for half
// precision: one warp, up to 16 rows and 16 keys at a time, all in registers.
//
// Single-token decoding and small trees have R to 16 rows per KV head; a
// 128-row tensor-memory tile is mostly padding there and its operands have to
// pass through shared memory.  Here (mma.m16n8k16, f16 operands, fp32 sums)
//
//   S = Q K^T   rows are M, keys N (up to 8 rows: the other way round, see
//               tree_mma8): a thread's packed words are its B operand
//               as they are loaded: four codes' worth of shifts, the code bias
//               taken off, no scale.  Scales multiply the fp32 sums of their
//               group of columns, so scores are exact to fp32 rounding for any
//               scale type.
//   O += P V    the weights are the A operand in the registers where the scores
//               were; V's B operand pairs the same column of two keys, so two
//               keys' words are interleaved before they are taken apart, and
//               values are codes times scale in f16 (f16 scales: and its rest).
//
// Which columns a thread takes is free, as long as Q (or the output) follows:
// thread t of four takes words t, 4 + t, ... of a row of K, thread g of eight
// the g-th eighth of a row of V.
//
// A block of warps takes a range of one unit's keys, 16 keys per warp in turn;
// its warps meet in shared memory, up to eight ranges of one unit in a cluster,
// more in the workspace (tree_merge of branch.cu).  Every warp has a ring of steps of its own, filled
// by asynchronous copies three ahead; nothing waits for another warp on the way.
// Bound: instructions, about 450 per warp and 16 keys of 128 columns, a third of
// which take codes apart; memory next.  Measured, 8 KV heads of 128 columns: single
// tokens of 4 rows, 16 sequences x 4096, 29.5 us (84 MB: 2.8 TB/s, a step in 60 % of
// the issue slots); 8 nodes x 512 9.1 us with the join, most of it loads that wait
// for one another; 32 rows x 4096, batch 4, 23 us.
#include <algorithm>

#include "branch.cuh"
#include "tc_rows.cuh"

namespace kv4 {

// device error word of this file (folded into kv4_device_error)
__device__ int g_branch_error_mma = 0;

namespace {

struct MmaPlan {
  int64_t units;
  int rows, row_tiles, parts;
  bool cluster;  // the parts of a row tile are a cluster and join there
};

constexpr int NW = 4;             // warps per block
constexpr int kClusterParts = 8;  // most blocks that join as a cluster
constexpr float kShift = 7.0f;  // weights are written times 2^7 (see branch_tc.cu)

// The power of two 2^e in a warp's V operands and output sums: it moves when a
// step's scales are not exact at the present one (see tc.cuh; f16 scales: v_scales).
struct VShift {
  int e = 0, least = tc::kMaxShift;  // least: smallest so far; sums move up by 2^48 at most, which they can
  float up = 1.0f;                   // 2^e
};
__device__ __forceinline__ float max3nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Whether the step's scales, four of them times 2^e, are not all exact in f16 (a
// zero counts as too small: seldom, and looked at again in shift_for).
__device__ __forceinline__ bool not_exact(const float (&f)[4]) {
  const float top = max3nan(max3nan(fabsf(f[0]), fabsf(f[1]), fabsf(f[2])), fabsf(f[3]), 0.0f);
  const float low = fminf(fminf(fabsf(f[0]), fabsf(f[1])), fminf(fabsf(f[2]), fabsf(f[3])));
  return !(top < 4096.0f) || low < 0x1p-17f;
}
// The step's power of two; returns what the sums so far have to be multiplied with.
// The whole warp takes part; vs: its 16-bit scales.
__device__ __forceinline__ float shift_for(VShift &V, const uint32_t (&vs)[4]) {
  uint32_t top = 0;
  bool exact = true;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t u = tc::scale_bits(vs[j]);
    exact = exact && tc::scale_exact(u);
    if (tc::scale_usable(u)) top = max(top, u);
  }
  exact = __all_sync(0xffffffffu, exact);
  top = __reduce_max_sync(0xffffffffu, top);
  int e = V.e;
  if (top != 0u) e = min(exact ? 0 : tc::scale_shift(top), V.least + 48);
  const float factor = tc::pow2(e - V.e);
  V.e = e;
  V.least = min(V.least, e);
  V.up = tc::pow2(e);
  return factor;
}

// Code times an f16 scale has up to 14 bits: what f16 cuts off goes through the
// product on its own, so that an f16 output has no error of V's: 2.3e-4 from the
// 64-bit result instead of 3.1e-4 at 17 nodes x 1000 (a plain fp32 form: 2.1e-4), for
// 33 us instead of 29 for 16 single tokens x 4K.  Bf16 scales' products fit.
template <typename ST>
constexpr bool kRest = DT<ST>::code == KV4_F16;

// scale i of a packed row of 16-bit scales
template <typename ST>
__device__ __forceinline__ float scale_at(const uint32_t *w, int i) {
  if (DT<ST>::code == KV4_BF16) return i & 1 ? bf16hi_to_f32(w[i >> 1]) : bf16lo_to_f32(w[i >> 1]);
  return i & 1 ? f16hi_to_f32(w[i >> 1]) : f16lo_to_f32(w[i >> 1]);
}

// whether a V scale can be an operand; one that cannot is reported
template <typename ST>
__device__ __forceinline__ bool usable(uint32_t s) {
  return kRest<ST> ? (s & 0x7FFFu) < 0x7C00u : tc::scale_usable(tc::scale_bits(s));
}

// V's scales of a step, keys in pairs, as f16; `rescale(f)` multiplies the sums so
// far.  The whole warp takes part.
template <typename ST, class F>
__device__ __forceinline__ void v_scales(uint32_t (&sp)[2], const uint32_t (&vs)[4], VShift &V, bool draft,
                                         bool &big, F rescale) {
  if (kRest<ST>) {
    // f16 scales are operands as they are; those from 2^13 on, whose products with
    // codes f16 does not hold, times 2^-4, and then all others too
    const uint32_t end = V.e == 0 ? 0x7000u : 0x7C00u;
    sp[0] = prmt(vs[0], vs[1], 0x5410);
    sp[1] = prmt(vs[2], vs[3], 0x5410);
    const uint32_t most = __vmaxu2(sp[0] & 0x7FFF7FFFu, sp[1] & 0x7FFF7FFFu);
    if (__any_sync(0xffffffffu, max(most & 0xFFFFu, most >> 16) >= end)) {
      bool large = false;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (usable<ST>(vs[j])) {
          large = large || (vs[j] & 0x7FFFu) >= 0x7000u;
        } else {
          big = true;
          if (draft) sp[j >> 1] &= j & 1 ? 0xffffu : 0xffff0000u;  // rows that see it are marked
        }
      }
      if (V.e == 0 && __any_sync(0xffffffffu, large)) {
        V.e = -4;
        rescale(0.0625f);
      }
    }
    if (V.e != 0) {
      sp[0] = tc::hmul2(sp[0], 0x2C002C00u);
      sp[1] = tc::hmul2(sp[1], 0x2C002C00u);
    }
    return;
  }
  float f[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) f[j] = scale_at<ST>(&vs[j], 0);
#pragma unroll
  for (int j = 0; j < 4; ++j) f[j] *= V.up;
  if (__any_sync(0xffffffffu, not_exact(f))) {
    const float factor = shift_for(V, vs);
    if (factor != 1.0f) rescale(factor);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[j] = scale_at<ST>(&vs[j], 0) * V.up;
      if (!usable<ST>(vs[j])) {
        big = true;
        if (draft) f[j] = 0.0f;  // rows that see it are marked
      }
    }
  }
  sp[0] = pack_f16x2(f[0], f[1]);
  sp[1] = pack_f16x2(f[2], f[3]);
}

// A warp's ring of steps in shared memory.  One step is 16 keys: rows of K (and
// V) codes, padded so that the reads below meet no bank twice, then their
// scales.  Copied asynchronously, 16 bytes of codes and 4 of scales at a time;
// what lies past the last key becomes zeros.
template <int D, int G, bool WITH_V>
struct Ring {
  static constexpr int NG = D / G, SB = 2 * NG;           // scales of a key: number, bytes
  static constexpr int ROW = D == 128 ? 80 : 48;          // bytes from key to key
  static constexpr int K = 0, V = 16 * ROW, KS = WITH_V ? 32 * ROW : 16 * ROW, VS = KS + 16 * SB;
  static constexpr int STEP = (WITH_V ? VS + 16 * SB : VS) + 15 & ~15;
  static constexpr int DEPTH = WITH_V ? 4 : 6;
  static constexpr int BYTES = DEPTH * STEP;
};

template <int N>
__device__ __forceinline__ void cp_async(uint32_t dst, const void *src, uint32_t n) {
  if (N == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// One (sequence, KV head) plane of a source
struct Plane {
  const uint8_t *k, *v, *ks, *vs;
};
__device__ __forceinline__ Plane plane_of(const RowSource &S, int64_t b, int h) {
  Plane p;
  p.k = S.kp + b * S.kps[0] + h * S.kps[1];
  p.v = S.vp + b * S.vps[0] + h * S.vps[1];
  p.ks = static_cast<const uint8_t *>(S.ks) + 2 * (b * S.kss[0] + h * S.kss[1]);
  p.vs = static_cast<const uint8_t *>(S.vs) + 2 * (b * S.vss[0] + h * S.vss[1]);
  return p;
}

// Start the copy of keys [k0, k0 + 16) to `to`; those from `left` on do not exist.
template <int D, int G, bool WITH_V>
__device__ __forceinline__ void fetch_step(const Plane &P, int64_t k0, int left, uint32_t to, int lane) {
  using R = Ring<D, G, WITH_V>;
  constexpr int CPR = D / 32;  // 16-byte chunks per row
  const uint8_t *k = P.k + k0 * (D / 2), *v = P.v + k0 * (D / 2);
#pragma unroll
  for (int i = 0; i < CPR / 2; ++i) {
    const int row = lane / CPR + 32 / CPR * i, c = lane % CPR;
    const uint32_t n = row < left ? 16u : 0u;
    const int from = n ? row * (D / 2) + 16 * c : 0;
    cp_async<16>(to + R::K + row * R::ROW + 16 * c, k + from, n);
    if (WITH_V) cp_async<16>(to + R::V + row * R::ROW + 16 * c, v + from, n);
  }
  if (lane < 4 * R::SB) {  // 16 SB bytes of scales, four a lane
    const int have = left * R::SB - 4 * lane;
    const uint32_t n = have >= 4 ? 4u : have > 0 ? static_cast<uint32_t>(have) : 0u;
    const int from = n ? 4 * lane : 0;
    cp_async<4>(to + R::KS + 4 * lane, P.ks + k0 * R::SB + from, n);
    if (WITH_V) cp_async<4>(to + R::VS + 4 * lane, P.vs + k0 * R::SB + from, n);
  }
}

// scales of one key from shared memory
template <int NG>
__device__ __forceinline__ void lds_scales(uint32_t (&w)[(NG + 1) / 2], uint32_t at) {
  if (NG == 4) {
    const uint2 v = lds64(at);
    w[0] = v.x;
    w[(NG + 1) / 2 - 1] = v.y;
  } else if (NG == 2) {
    w[0] = lds32(at);
  } else {
    w[0] = lds16(at);
  }
}

// A operand of 16 (or 8) rows of q, in the column order of the K words, and the
// factor of rows g and g + 8 from sums to base-2 exponents.  bf16 rows are
// scaled by a power of two so that their largest element lies in
// [2^13, 2^14): exact down to 2^-26 of it, and off by at most 2^-34 of it below
// that.  f16 rows are exact below 2^11; with larger elements, down to 2^-10, and off
// by at most 2^-21 below that.
template <int D, bool HALF>
struct Query {
  uint32_t a[D / 16][HALF ? 2 : 4];
  float c[HALF ? 1 : 2];
};
template <int D, bool HALF>
__device__ __forceinline__ void load_query(Query<D, HALF> &Q, const TreeParams &T, int64_t b, int kvh,
                                           int row0, int rows, int lane) {
  const int g = lane >> 2, t = lane & 3;
  constexpr int NR = HALF ? 1 : 2;
  uint4 rows_w[NR][D / 32];  // both rows are on their way before the first is looked at
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const int row = row0 + g + 8 * r, node = row / T.R, head = kvh * T.R + row - node * T.R;
    const uint16_t *q = static_cast<const uint16_t *>(T.q) + b * T.qs[0] + head * T.qs[1] + node * T.qs[2] + 8 * t;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
      rows_w[r][i] = row < rows ? __ldg(reinterpret_cast<const uint4 *>(q + 32 * i)) : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const uint4(&w)[D / 32] = rows_w[r];
    Q.c[r] = T.scale_log2;
    const bool bf = T.q_dtype == KV4_BF16;
    uint32_t top = 0;  // largest |q| as bits: magnitudes of either type order like integers
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      const uint32_t u[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) top = __vmaxu2(top, u[e] & 0x7FFF7FFFu);
    }
    top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 2));
    top = max(top & 0xFFFFu, top >> 16);
    // pairs 1 and 3 meet codes times 16 (see code_pair)
    float up = 1.0f;
    uint32_t even = 0x3C003C00u, odd = 0x2C002C00u;  // 1, 1/16
    if (bf) {
      int ex = 13 - (static_cast<int>(top >> 7) - 127);
      ex = top == 0 ? 0 : min(max(ex, -126), 126);
      up = tc::pow2(ex);
      Q.c[r] *= tc::pow2(-ex);
    } else if (top < 0x6800u) {  // below 2^11: pairs 0 and 2 times 16 instead
      even = 0x4C004C00u;
      odd = 0x3C003C00u;
      Q.c[r] *= 0.0625f;
    }
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      const uint32_t u[4] = {w[i].x, w[i].y, w[i].z, w[i].w};  // columns 8t .. 8t + 7 of the block
      uint32_t p[4];                                          // pairs (0,4) (1,5) (2,6) (3,7)
      if (bf) {
        p[0] = pack_f16x2(bf16lo_to_f32(u[0]) * up, bf16lo_to_f32(u[2]) * up);
        p[1] = pack_f16x2(bf16hi_to_f32(u[0]) * up, bf16hi_to_f32(u[2]) * up);
        p[2] = pack_f16x2(bf16lo_to_f32(u[1]) * up, bf16lo_to_f32(u[3]) * up);
        p[3] = pack_f16x2(bf16hi_to_f32(u[1]) * up, bf16hi_to_f32(u[3]) * up);
      } else {
        p[0] = tc::hmul2(prmt(u[0], u[2], 0x5410), even);
        p[1] = prmt(u[0], u[2], 0x7632);
        p[2] = tc::hmul2(prmt(u[1], u[3], 0x5410), even);
        p[3] = prmt(u[1], u[3], 0x7632);
      }
      p[1] = tc::hmul2(p[1], odd);
      p[3] = tc::hmul2(p[3], odd);
      // k-step 2i: pairs 0 and 1; k-step 2i + 1: pairs 2 and 3
      if (HALF) {
        Q.a[2 * i][0] = p[0];
        Q.a[2 * i][1] = p[1];
        Q.a[2 * i + 1][0] = p[2];
        Q.a[2 * i + 1][1] = p[3];
      } else {
        Q.a[2 * i][r] = p[0];
        Q.a[2 * i][(HALF ? 0 : 2) + r] = p[1];
        Q.a[2 * i + 1][r] = p[2];
        Q.a[2 * i + 1][(HALF ? 0 : 2) + r] = p[3];
      }
    }
  }
}

// f16 pairs of a word's nibbles e and e + 4: code - 8 for even e, 16 times that
// for odd e, whose bits then need no shift of their own (both exact)
__device__ __forceinline__ uint32_t code_pair(uint32_t w, int e) {
  const uint32_t x = e < 2 ? w : w >> 8;
  if (!(e & 1)) return tc::hsub2(tc::nib_pair(x), 0x64086408u);
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(x), "r"(0x00F000F0u), "r"(0x64006400u));
  return tc::hsub2(r, 0x64806480u);
}
__device__ __forceinline__ uint32_t code_pair1(uint32_t w, int e) {  // code - 8 for every e
  return tc::hsub2(tc::nib_pair(w >> (4 * e)), 0x64086408u);
}

// Sums of rows g (s[0], s[1]) and g + 8 (s[2], s[3]) with keys 2t, 2t + 1 of
// key tile n of the step at `at`, scaled group by group.
template <int D, int G, typename ST, bool WITH_V>
__device__ __forceinline__ void scores(float (&s)[4], const Query<D, false> &Q, uint32_t at, int n, int lane) {
  using R = Ring<D, G, WITH_V>;
  const int g = lane >> 2, t = lane & 3;
  uint32_t w[D / 32], k0[(R::NG + 1) / 2], k1[(R::NG + 1) / 2];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) w[i] = lds32(at + R::K + (8 * n + g) * R::ROW + 16 * i + 4 * t);
  lds_scales<R::NG>(k0, at + R::KS + (8 * n + 2 * t) * R::SB);
  lds_scales<R::NG>(k1, at + R::KS + (8 * n + 2 * t + 1) * R::SB);
  s[0] = s[1] = s[2] = s[3] = 0.0f;
#pragma unroll
  for (int gr = 0; gr < R::NG; ++gr) {
    float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < G / 32; ++i) {
      const int blk = gr * (G / 32) + i;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t *a = Q.a[2 * blk + j];
        mma_f16_16816(c, a[0], a[1], a[2], a[3], code_pair(w[blk], 2 * j), code_pair(w[blk], 2 * j + 1));
      }
    }
    const float f0 = scale_at<ST>(k0, gr), f1 = scale_at<ST>(k1, gr);
    s[0] = fmaf(c[0], f0, s[0]);
    s[1] = fmaf(c[1], f1, s[1]);
    s[2] = fmaf(c[2], f0, s[2]);
    s[3] = fmaf(c[3], f1, s[3]);
  }
}

// which of a thread's four keys row `node` sees, as bits j (order of Keys)
__device__ __forceinline__ uint32_t seen_keys(const TreeParams &T, int64_t b, bool draft, int node,
                                              bool row_ok, int64_t k0, int64_t end, int t) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t key = k0 + 2 * t + (j & 1) + 8 * (j >> 1);
    bool on = row_ok && key < end;
    if (on && draft) on = draft_visible(T, b, node, static_cast<int>(key));
    m |= on ? 1u << j : 0u;
  }
  return m;
}

// The block's warps' outputs [NW][NR][D + 4] and (maximum, sum) [NW][NR] become
// the call's output, or the block's partial rows.
template <int D, int NR>
__device__ __forceinline__ void meet(const TreeParams &T, const MmaPlan &L, const float *msm, const float2 *sml,
                                     int64_t unit, int64_t b, int kvh, int part, int row0) {
  constexpr int LD = D + 4;
  const int nr = min(NR, L.rows - row0);
  for (int idx = threadIdx.x; idx < nr * (D / 2); idx += NW * 32) {
    const int r = idx / (D / 2), c = (idx - r * (D / 2)) * 2, row = row0 + r;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, sml[w * NR + r].x);
    const float base = M == -INFINITY ? 0.0f : M;
    float sum = 0.0f, v0 = 0.0f, v1 = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float2 ml = sml[w * NR + r];
      const float f = exp2f(ml.x - base);
      sum = fmaf(ml.y, f, sum);
      const float2 v = *reinterpret_cast<const float2 *>(msm + (w * NR + r) * LD + c);
      v0 = fmaf(v.x, f, v0);
      v1 = fmaf(v.y, f, v1);
    }
    const int64_t at = unit * L.rows + row;
    if (L.parts > 1) {
      const int64_t slot = static_cast<int64_t>(part) * L.units * L.rows + at;
      *reinterpret_cast<float2 *>(T.ws_o + slot * D + c) = make_float2(v0, v1);
      if (c == 0) T.ws_ml[slot] = make_float2(M, sum);
      continue;
    }
    const int nd = row / T.R, head = kvh * T.R + row - nd * T.R;
    const float inv = sum > 0.0f ? 1.0f / sum : (sum == sum ? 0.0f : sum);
    const int64_t off = b * T.os[0] + head * T.os[1] + nd * T.os[2] + c;
    *reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(T.out) + off) =
        T.q_dtype == KV4_BF16 ? pack_bf16x2(v0 * inv, v1 * inv) : pack_f16x2(v0 * inv, v1 * inv);
    if (c == 0) {
      if (T.stats) T.stats[at] = make_float2(M, inv);
      if (T.lse)
        T.lse[b * T.ls[0] + head * T.ls[1] + nd * T.ls[2]] =
            sum == 0.0f ? -INFINITY : (M + log2f(sum)) * kBrLn2;
    }
  }
}

// The same where the parts of a row tile are a cluster: each block joins its warps
// in place, then takes a share of the row tile's output from all of them.  Against
// tree_merge, a launch of its own: 8 nodes x 512 x 8 heads of 128 columns 9.8 us ->
// 8.6, 17 x 1000 x 12 heads of 64, batch 4, 11.4 -> 10.4, 32 rows x 4K, batch 8, 41.6
// -> 40.7.
template <int D, int NR>
__device__ __forceinline__ void meet_cluster(const TreeParams &T, const MmaPlan &L, float *msm, float2 *sml,
                                             int64_t unit, int64_t b, int kvh, int part, int row0) {
  constexpr int LD = D + 4, Q = D / 4;
  float2 *const own = sml + NW * NR;  // this block's (maximum, sum) per row
  const int nr = min(NR, L.rows - row0);
#pragma unroll 1
  for (int idx = threadIdx.x; idx < nr * Q; idx += NW * 32) {
    const int r = idx / Q, c = (idx - r * Q) * 4;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, sml[w * NR + r].x);
    const float base = M == -INFINITY ? 0.0f : M;
    float sum = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float2 ml = sml[w * NR + r];
      const float f = exp2f(ml.x - base);
      sum = fmaf(ml.y, f, sum);
      const float4 v = *reinterpret_cast<const float4 *>(msm + (w * NR + r) * LD + c);
      o = make_float4(fmaf(v.x, f, o.x), fmaf(v.y, f, o.y), fmaf(v.z, f, o.z), fmaf(v.w, f, o.w));
    }
    *reinterpret_cast<float4 *>(msm + r * LD + c) = o;  // read by this thread alone so far
    if (c == 0) own[r] = make_float2(M, sum);
  }
  cluster_sync();
#pragma unroll 1
  for (int idx = part * NW * 32 + threadIdx.x; idx < nr * Q; idx += L.parts * NW * 32) {
    const int r = idx / Q, c = (idx - r * Q) * 4, row = row0 + r;
    const uint32_t at_o = smem_u32(msm + r * LD + c), at_m = smem_u32(own + r);
    float m[kClusterParts], l[kClusterParts], M = -INFINITY;
    float4 v[kClusterParts];
#pragma unroll
    for (int p = 0; p < kClusterParts; ++p) {
      m[p] = -INFINITY;
      if (p < L.parts) {
        m[p] = ld_dsmem_f32(dsmem_addr(at_m, p));
        l[p] = ld_dsmem_f32(dsmem_addr(at_m, p) + 4);
        v[p] = ld_dsmem_f4(dsmem_addr(at_o, p));
      }
    }
#pragma unroll
    for (int p = 0; p < kClusterParts; ++p) M = fmaxf(M, m[p]);
    const float base = M == -INFINITY ? 0.0f : M;
    float sum = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int p = 0; p < kClusterParts; ++p) {
      if (p >= L.parts) break;
      const float f = exp2f(m[p] - base);
      sum = fmaf(l[p], f, sum);
      o = make_float4(fmaf(v[p].x, f, o.x), fmaf(v[p].y, f, o.y), fmaf(v[p].z, f, o.z), fmaf(v[p].w, f, o.w));
    }
    const int nd = row / T.R, head = kvh * T.R + row - nd * T.R;
    const float inv = sum > 0.0f ? 1.0f / sum : (sum == sum ? 0.0f : sum);
    const int64_t off = b * T.os[0] + head * T.os[1] + nd * T.os[2] + c;
    const float x[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
    *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(T.out) + off) =
        T.q_dtype == KV4_BF16 ? make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]))
                              : make_uint2(pack_f16x2(x[0], x[1]), pack_f16x2(x[2], x[3]));
    if (c == 0) {
      if (T.stats) T.stats[unit * L.rows + row] = make_float2(M, inv);
      if (T.lse)
        T.lse[b * T.ls[0] + head * T.ls[1] + nd * T.ls[2]] =
            sum == 0.0f ? -INFINITY : (M + log2f(sum)) * kBrLn2;
    }
  }
  cluster_sync();  // nobody's shared memory goes while it is read
}

template <int D, int G, typename ST>
__global__ void __launch_bounds__(NW * 32, 3)
    tree_mma(const __grid_constant__ TreeParams T, const MmaPlan L) {
  constexpr int NR = 16, RT = 2, DG = D / 8, LD = D + 4;
  extern __shared__ __align__(16) float msm[];  // rings, later [NW][NR][LD] outputs, [NW][NR] float2 (m, l)
  float2 *sml = reinterpret_cast<float2 *>(msm + NW * NR * LD);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int part = static_cast<int>(blockIdx.x % L.parts);
  const int64_t ur = blockIdx.x / L.parts;
  const int rt = static_cast<int>(ur % L.row_tiles), row0 = rt * NR;
  const int64_t unit = ur / L.row_tiles, b = unit / T.Hkv;
  const int kvh = static_cast<int>(unit - b * T.Hkv);
  const int64_t len = context_len(T, b, part == 0 && rt == 0 && kvh == 0 && threadIdx.x == 0 ? &g_branch_error_mma : nullptr);
  const int nctx = static_cast<int>((len + 15) >> 4), steps = nctx + ((T.ndraft + 15) >> 4);
  const int per = (steps + L.parts - 1) / L.parts;
  const int s0 = part * per, s1 = min(steps, s0 + per);

  using R = Ring<D, G, true>;
  const uint32_t ring = smem_u32(msm) + warp * R::BYTES;
  const Plane ctx = plane_of(T.cache, b, kvh);
  auto fetch = [&](int s, uint32_t slot) {
    if (s < nctx) {
      fetch_step<D, G, true>(ctx, static_cast<int64_t>(s) * 16, static_cast<int>(min(len - static_cast<int64_t>(s) * 16, int64_t(16))),
                             ring + slot * R::STEP, lane);
    } else if (s < s1) {
      const Plane dft = plane_of(T.draft, b, kvh);
      fetch_step<D, G, true>(dft, static_cast<int64_t>(s - nctx) * 16, min(T.ndraft - (s - nctx) * 16, 16),
                             ring + slot * R::STEP, lane);
    }
    cp_async_commit();
  };
  // steps s0 + warp, + NW, ...: DEPTH - 1 of them on their way
  int s = s0 + warp;
#pragma unroll 1
  for (int i = 0; i < R::DEPTH - 1; ++i)
    if (s + i * NW < s1) fetch(s + i * NW, i);
    else cp_async_commit();
  Query<D, false> Q;
  load_query(Q, T, b, kvh, row0, L.rows, lane);
  int node[RT];
  bool ok[RT];
  float m[RT], l[RT];
  bool broken[RT];
  float o[DG][4];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int row = row0 + g + 8 * r;
    ok[r] = row < L.rows;
    node[r] = row / T.R;
    m[r] = -INFINITY;
    l[r] = 0.0f;
    broken[r] = false;
  }
#pragma unroll
  for (int j = 0; j < DG; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[j][e] = 0.0f;
  bool big = false;
  VShift V;
  // kept scores of rows g and g + 8 (one row tile holds them all)
  float *const kept = T.kept ? T.kept + kept_at(unit, steps, 2 * t, g, L.rows) : nullptr;
  if (T.kept && part == 0 && warp == 0 && t == 0) {
#pragma unroll
    for (int r = 0; r < RT; ++r)
      if (ok[r]) T.kept_c[unit * L.rows + g + 8 * r] = Q.c[r];
  }

  uint32_t slot = 0;
#pragma unroll 1
  for (; s < s1; s += NW) {
    const bool draft = s >= nctx;
    const int64_t k0 = static_cast<int64_t>(draft ? s - nctx : s) * 16, end = draft ? T.ndraft : len;
    cp_async_wait<R::DEPTH - 2>();
    __syncwarp();  // this step is there for all lanes, and all are done with the one before
    {
      const int ahead = s + (R::DEPTH - 1) * NW;
      if (ahead < s1) fetch(ahead, slot == 0 ? R::DEPTH - 1 : slot - 1);
      else cp_async_commit();
    }
    const uint32_t at = ring + slot * R::STEP;
    slot = slot + 1 == R::DEPTH ? 0 : slot + 1;
    float x[2][4];
    scores<D, G, ST, true>(x[0], Q, at, 0, lane);
    scores<D, G, ST, true>(x[1], Q, at, 1, lane);
    uint32_t vs[4];  // V's scales of this thread's columns, keys 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
    for (int j = 0; j < 4; ++j)
      vs[j] = lds16(at + R::VS + (2 * t + (j & 1) + 8 * (j >> 1)) * R::SB + 2 * (g * DG / G));

    // scores -> weights, in place
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      float y[4] = {x[0][2 * r], x[0][2 * r + 1], x[1][2 * r], x[1][2 * r + 1]};
      if (draft || k0 + 16 > end) {
        const uint32_t on = seen_keys(T, b, draft, node[r], ok[r], k0, end, t);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (!(on >> j & 1u)) y[j] = -INFINITY;
        if (draft) {  // a visible key without a usable V scale: the row has no value
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const bool bad = !usable<ST>(vs[j]);
            const uint32_t any = __ballot_sync(0xffffffffu, bad) & (0x11111111u << t);
            if (any && (on >> j & 1u)) broken[r] = true;
          }
        }
      }
      if (kept && ok[r]) {
        float *p = kept + (static_cast<int64_t>(s) * L.rows + 8 * r) * 16;
        *reinterpret_cast<float2 *>(p) = make_float2(y[0], y[1]);
        *reinterpret_cast<float2 *>(p + 8) = make_float2(y[2], y[3]);
      }
      float mx = fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])) * Q.c[r];
      // the maximum moves only when a score passes it by more than 8: seldom
      if (__any_sync(0xffffffffu, mx > m[r] + 8.0f)) {
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float to = mx > m[r] + 8.0f ? mx : m[r];
        const float alpha = to == m[r] ? 1.0f : m[r] == -INFINITY ? 0.0f : fast_exp2(m[r] - to);
        m[r] = to;
        l[r] *= alpha;
#pragma unroll
        for (int j = 0; j < DG; ++j) {
          o[j][2 * r] *= alpha;
          o[j][2 * r + 1] *= alpha;
        }
      }
      const float base = m[r] == -INFINITY ? 0.0f : m[r] - kShift;
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = fast_exp2(fmaf(y[j], Q.c[r], -base));
      l[r] += (y[0] + y[1]) + (y[2] + y[3]);
      x[0][2 * r] = y[0];
      x[0][2 * r + 1] = y[1];
      x[1][2 * r] = y[2];
      x[1][2 * r + 1] = y[3];
    }
    const uint32_t a0 = pack_f16x2(x[0][0], x[0][1]), a2 = pack_f16x2(x[1][0], x[1][1]);
    const uint32_t a1 = pack_f16x2(x[0][2], x[0][3]);
    const uint32_t a3 = pack_f16x2(x[1][2], x[1][3]);

    // O += P V: column j of this thread's eighth, keys in pairs
    uint32_t sp[2];
    v_scales<ST>(sp, vs, V, draft, big, [&](float f) {
#pragma unroll
      for (int j = 0; j < DG; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][e] *= f;
    });
    uint32_t vw[4][D / 64];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t p = at + R::V + (2 * t + (j & 1) + 8 * (j >> 1)) * R::ROW + g * (D / 16);
      if (D == 128) {
        const uint2 w = lds64(p);
        vw[j][0] = w.x;
        vw[j][D / 64 - 1] = w.y;
      } else {
        vw[j][0] = lds32(p);
      }
    }
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      uint32_t y[2][2];  // [key pair][half word]: the pair's words side by side
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        y[p][0] = prmt(vw[2 * p][i], vw[2 * p + 1][i], 0x5410);
        y[p][1] = prmt(vw[2 * p][i], vw[2 * p + 1][i], 0x7632);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t c0 = code_pair1(y[0][e >> 2], e & 3), c1 = code_pair1(y[1][e >> 2], e & 3);
        const uint32_t b0 = tc::hmul2(c0, sp[0]), b1 = tc::hmul2(c1, sp[1]);
        mma_f16_16816(o[8 * i + e], a0, a1, a2, a3, b0, b1);
        if (kRest<ST>)
          mma_f16_16816(o[8 * i + e], a0, a1, a2, a3, tc::hrest2(c0, sp[0], b0), tc::hrest2(c1, sp[1], b1));
      }
    }
  }
  if (big) atomicOr(&g_branch_error_mma, DEV_ERR_F16_RANGE);

  // ---- the block's warps meet, where the rings were ----
  const float down = tc::pow2(-V.e);
  cp_async_wait<0>();
  __syncthreads();
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    const uint32_t bad = __ballot_sync(0xffffffffu, broken[r]);
    if (bad & (0xFu << (4 * g))) l[r] = __uint_as_float(0x7fc00000u);
    const int at = warp * NR + g + 8 * r;
    if (t == 0) sml[at] = make_float2(m[r] - kShift, l[r]);
    // columns 2t and 2t + 1 of output tile j are dims 2t * DG + j and (2t + 1) * DG + j
#pragma unroll
    for (int j = 0; j < DG; ++j) {
      msm[at * LD + 2 * t * DG + j] = o[j][2 * r] * down;
      msm[at * LD + (2 * t + 1) * DG + j] = o[j][2 * r + 1] * down;
    }
  }
  __syncthreads();
  if (L.cluster) meet_cluster<D, NR>(T, L, msm, sml, unit, b, kvh, part, row0);
  else meet<D, NR>(T, L, msm, sml, unit, b, kvh, part, row0);
}

// Up to 8 rows: keys are M (or, for V, columns), rows N, so that no half of a
// product is padding.  Weights become the B operand of the second product by a
// transpose within the warp.  Against rows as M: half the products, no spills
// (16 sequences x 4096 x 4 rows: 40 us -> 29.5).
template <int D, int G, typename ST>
__global__ void __launch_bounds__(NW * 32, 4) tree_mma8(const __grid_constant__ TreeParams T, const MmaPlan L) {
  constexpr int NR = 8, DG = D / 8, LD = D + 4;
  extern __shared__ __align__(16) float msm[];  // rings, later [NW][NR][LD] outputs, [NW][NR] float2 (m, l)
  float2 *sml = reinterpret_cast<float2 *>(msm + NW * NR * LD);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int part = static_cast<int>(blockIdx.x % L.parts);
  const int64_t unit = blockIdx.x / L.parts, b = unit / T.Hkv;
  const int kvh = static_cast<int>(unit - b * T.Hkv);
  const int64_t len = context_len(T, b, part == 0 && kvh == 0 && threadIdx.x == 0 ? &g_branch_error_mma : nullptr);
  const int nctx = static_cast<int>((len + 15) >> 4), steps = nctx + ((T.ndraft + 15) >> 4);
  const int per = (steps + L.parts - 1) / L.parts;
  const int s0 = part * per, s1 = min(steps, s0 + per);

  using R = Ring<D, G, true>;
  const uint32_t ring = smem_u32(msm) + warp * R::BYTES;
  const Plane ctx = plane_of(T.cache, b, kvh);
  auto fetch = [&](int s, uint32_t slot) {
    if (s < nctx) {
      fetch_step<D, G, true>(ctx, static_cast<int64_t>(s) * 16, static_cast<int>(min(len - static_cast<int64_t>(s) * 16, int64_t(16))),
                             ring + slot * R::STEP, lane);
    } else if (s < s1) {
      const Plane dft = plane_of(T.draft, b, kvh);
      fetch_step<D, G, true>(dft, static_cast<int64_t>(s - nctx) * 16, min(T.ndraft - (s - nctx) * 16, 16),
                             ring + slot * R::STEP, lane);
    }
    cp_async_commit();
  };
  int s = s0 + warp;
#pragma unroll 1
  for (int i = 0; i < R::DEPTH - 1; ++i)
    if (s + i * NW < s1) fetch(s + i * NW, i);
    else cp_async_commit();
  Query<D, true> Q;  // of row g
  load_query(Q, T, b, kvh, 0, L.rows, lane);
  if (T.kept_c && part == 0 && warp == 0 && t == 0 && g < L.rows) T.kept_c[unit * L.rows + g] = Q.c[0];
  // this thread's scores are those of rows 2t, 2t + 1 with keys g, g + 8
  const float c[2] = {__shfl_sync(0xffffffffu, Q.c[0], 8 * t), __shfl_sync(0xffffffffu, Q.c[0], 8 * t + 4)};
  const bool ok[2] = {2 * t < L.rows, 2 * t + 1 < L.rows};
  float *const kept = T.kept ? T.kept + kept_at(unit, steps, g, 2 * t, L.rows) : nullptr;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
  bool broken[2] = {false, false};
  float o[D / 16][4];  // columns 2j, 2j + 1 of eighth g, rows 2t, 2t + 1
#pragma unroll
  for (int j = 0; j < D / 16; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[j][e] = 0.0f;
  bool big = false;
  VShift V;

  uint32_t slot = 0;
#pragma unroll 1
  for (; s < s1; s += NW) {
    const bool draft = s >= nctx;
    const int64_t k0 = static_cast<int64_t>(draft ? s - nctx : s) * 16, end = draft ? T.ndraft : len;
    cp_async_wait<R::DEPTH - 2>();
    __syncwarp();  // this step is there for all lanes, and all are done with the one before
    {
      const int ahead = s + (R::DEPTH - 1) * NW;
      if (ahead < s1) fetch(ahead, slot == 0 ? R::DEPTH - 1 : slot - 1);
      else cp_async_commit();
    }
    const uint32_t at = ring + slot * R::STEP;
    slot = slot + 1 == R::DEPTH ? 0 : slot + 1;

    // S = K Q^T, scaled group by group
    float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // (key g, rows 2t, 2t + 1), (key g + 8, the same)
    {
      uint32_t w0[D / 32], w1[D / 32], f0[(R::NG + 1) / 2], f1[(R::NG + 1) / 2];
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        w0[i] = lds32(at + R::K + g * R::ROW + 16 * i + 4 * t);
        w1[i] = lds32(at + R::K + (g + 8) * R::ROW + 16 * i + 4 * t);
      }
      lds_scales<R::NG>(f0, at + R::KS + g * R::SB);
      lds_scales<R::NG>(f1, at + R::KS + (g + 8) * R::SB);
#pragma unroll
      for (int gr = 0; gr < R::NG; ++gr) {
        float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < G / 32; ++i) {
          const int blk = gr * (G / 32) + i;
#pragma unroll
          for (int j = 0; j < 2; ++j)
            mma_f16_16816(y, code_pair(w0[blk], 2 * j), code_pair(w1[blk], 2 * j), code_pair(w0[blk], 2 * j + 1),
                          code_pair(w1[blk], 2 * j + 1), Q.a[2 * blk + j][0], Q.a[2 * blk + j][1]);
        }
        const float k0f = scale_at<ST>(f0, gr), k1f = scale_at<ST>(f1, gr);
        x[0] = fmaf(y[0], k0f, x[0]);
        x[1] = fmaf(y[1], k0f, x[1]);
        x[2] = fmaf(y[2], k1f, x[2]);
        x[3] = fmaf(y[3], k1f, x[3]);
      }
    }
    uint32_t vs[4];  // V's scales of eighth g, keys 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
    for (int j = 0; j < 4; ++j)
      vs[j] = lds16(at + R::VS + (2 * t + (j & 1) + 8 * (j >> 1)) * R::SB + 2 * (g * DG / G));

    if (draft || k0 + 16 > end) {
      uint32_t bad = 0;  // keys of this step without a usable V scale
      if (draft) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (!usable<ST>(vs[j])) bad |= 1u << (2 * t + (j & 1) + 8 * (j >> 1));
        bad = __reduce_or_sync(0xffffffffu, bad);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = e & 1, k = g + 8 * (e >> 1);
        bool on = ok[r] && k0 + k < end;
        if (on && draft) on = draft_visible(T, b, (2 * t + r) / T.R, static_cast<int>(k0) + k);
        if (!on) x[e] = -INFINITY;
        else if (bad >> k & 1u) broken[r] = true;  // the row has no value
      }
    }
    if (kept) {
      float *p = kept + static_cast<int64_t>(s) * L.rows * 16;
      if (ok[0]) {
        p[0] = x[0];
        p[8] = x[2];
      }
      if (ok[1]) {
        p[16] = x[1];
        p[24] = x[3];
      }
    }
    // scores -> weights, in place; the maximum moves only when a score passes it
    // by more than 8: seldom
    float mx[2] = {fmaxf(x[0], x[2]) * c[0], fmaxf(x[1], x[3]) * c[1]};
    if (__any_sync(0xffffffffu, mx[0] > m[0] + 8.0f || mx[1] > m[1] + 8.0f)) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], d));
        const float to = mx[r] > m[r] + 8.0f ? mx[r] : m[r];
        const float alpha = to == m[r] ? 1.0f : m[r] == -INFINITY ? 0.0f : fast_exp2(m[r] - to);
        m[r] = to;
        l[r] *= alpha;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
          o[j][r] *= alpha;
          o[j][2 + r] *= alpha;
        }
      }
    }
    const float base[2] = {m[0] == -INFINITY ? 0.0f : m[0] - kShift, m[1] == -INFINITY ? 0.0f : m[1] - kShift};
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = fast_exp2(fmaf(x[e], c[e & 1], -base[e & 1]));
    l[0] += x[0] + x[2];
    l[1] += x[1] + x[3];
    const uint32_t p0 = movmatrix_trans(pack_f16x2(x[0], x[1]));  // row g, keys 2t, 2t + 1
    const uint32_t p1 = movmatrix_trans(pack_f16x2(x[2], x[3]));  // keys 2t + 8, 2t + 9

    // O^T += V^T P^T: two columns of this thread's eighth, keys in pairs
    uint32_t sp[2];
    v_scales<ST>(sp, vs, V, draft, big, [&](float f) {
#pragma unroll
      for (int j = 0; j < D / 16; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][e] *= f;
    });
    uint32_t vw[4][D / 64];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t p = at + R::V + (2 * t + (j & 1) + 8 * (j >> 1)) * R::ROW + g * (D / 16);
      if (D == 128) {
        const uint2 w = lds64(p);
        vw[j][0] = w.x;
        vw[j][D / 64 - 1] = w.y;
      } else {
        vw[j][0] = lds32(p);
      }
    }
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      uint32_t y[2][2];  // [key pair][half word]: the pair's words side by side
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        y[p][0] = prmt(vw[2 * p][i], vw[2 * p + 1][i], 0x5410);
        y[p][1] = prmt(vw[2 * p][i], vw[2 * p + 1][i], 0x7632);
      }
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        uint32_t a[4], rest[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t code = code_pair1(y[k >> 1][e >> 2], (e & 3) + (k & 1));
          a[k] = tc::hmul2(code, sp[k >> 1]);
          rest[k] = kRest<ST> ? tc::hrest2(code, sp[k >> 1], a[k]) : 0u;
        }
        mma_f16_16816(o[4 * i + e / 2], a[0], a[1], a[2], a[3], p0, p1);
        if (kRest<ST>) mma_f16_16816(o[4 * i + e / 2], rest[0], rest[1], rest[2], rest[3], p0, p1);
      }
    }
  }
  if (big) atomicOr(&g_branch_error_mma, DEV_ERR_F16_RANGE);

  // ---- the block's warps meet, where the rings were ----
  const float down = tc::pow2(-V.e);
  cp_async_wait<0>();
  __syncthreads();
#pragma unroll
  for (int r = 0; r < 2; ++r) {
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], d);
    const uint32_t bad = __ballot_sync(0xffffffffu, broken[r]);
    if (bad & (0x11111111u << t)) l[r] = __uint_as_float(0x7fc00000u);
    const int row = warp * NR + 2 * t + r;
    if (g == 0) sml[row] = make_float2(m[r] - kShift, l[r]);
#pragma unroll
    for (int j = 0; j < D / 16; ++j)
      *reinterpret_cast<float2 *>(msm + row * LD + g * DG + 2 * j) = make_float2(o[j][r] * down, o[j][2 + r] * down);
  }
  __syncthreads();
  if (L.cluster) meet_cluster<D, NR>(T, L, msm, sml, unit, b, kvh, part, 0);
  else meet<D, NR>(T, L, msm, sml, unit, b, kvh, part, 0);
}

// Scores of the cached tokens for more rows than score_kept takes: weights formed
// again from K, the rows' maxima and sums, summed over the rows of each key (rows
// are lanes: three shuffles).  Instructions bound it: 32 rows x 4096 keys x 8
// heads of 128 columns, batch 4, 18.4 us.
template <int D, int G, typename ST>
__global__ void __launch_bounds__(NW * 32, 3)
    score_mma(const __grid_constant__ ScoreParams P, int rows, uint32_t steps_per_unit, uint32_t total) {
  constexpr int RT = 2, NR = 16;
  const TreeParams &T = P.t;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t warps = gridDim.x * NW, w = blockIdx.x * NW + (threadIdx.x >> 5);
  // warps take runs of one unit's 16-key steps
  const uint32_t each = total / warps, rest = total - each * warps;
  uint32_t at = w * each + min(w, rest);
  const uint32_t stop = at + each + (w < rest ? 1u : 0u);
  const int nctx = static_cast<int>((T.S + 15) >> 4);
  using R = Ring<D, G, false>;
  __shared__ __align__(16) uint8_t rings[NW * R::BYTES];
  const uint32_t ring = smem_u32(rings) + (threadIdx.x >> 5) * R::BYTES;
  griddep_wait();  // the rows' maxima and sums come from the kernel before
#pragma unroll 1
  while (at < stop) {
    const uint32_t unit = at / steps_per_unit, b = unit / T.Hkv;
    const int kvh = static_cast<int>(unit - b * T.Hkv);
    const int first = static_cast<int>(at - unit * steps_per_unit);
    const int last = static_cast<int>(min(steps_per_unit, first + stop - at));
    at += last - first;
    const float *in = P.in + b * P.is[0] + kvh * P.is[1];
    float *out = P.out + b * P.os[0] + kvh * P.os[1];
#pragma unroll 1
    for (int row0 = 0; row0 < rows; row0 += NR) {
      Query<D, false> Q;
      load_query(Q, T, b, kvh, row0, rows, lane);
      float sm[RT], sl[RT];  // maximum and 1 / sum of rows g, g + 8
      int node[RT];
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const int row = row0 + g + 8 * r;
        const float2 st = row < rows ? T.stats[static_cast<int64_t>(unit) * rows + row] : make_float2(0.0f, 0.0f);
        sm[r] = st.x;
        sl[r] = st.y;  // 0: a row that saw nothing, or none at all
        node[r] = row / T.R;
      }
      auto fetch = [&](int s, uint32_t slot) {
        const bool d = s >= nctx;
        const Plane p = plane_of(d ? T.draft : T.cache, b, kvh);
        const int64_t k0 = static_cast<int64_t>(d ? s - nctx : s) * 16, end = d ? T.ndraft : T.S;
        fetch_step<D, G, false>(p, k0, static_cast<int>(min(end - k0, int64_t(16))), ring + slot * R::STEP, lane);
        cp_async_commit();
      };
#pragma unroll 1
      for (int i = 0; i < R::DEPTH - 1; ++i)
        if (first + i < last) fetch(first + i, i);
        else cp_async_commit();
      uint32_t slot = 0;
#pragma unroll 1
      for (int s = first; s < last; ++s) {
        const bool draft = s >= nctx;
        const int64_t k0 = static_cast<int64_t>(draft ? s - nctx : s) * 16, end = draft ? T.ndraft : T.S;
        // lanes 0-15 end up with a key each
        const int64_t mine = k0 + lane, tok = draft ? T.S + mine : mine;
        float old = 0.0f;
        if (lane < 16 && mine < end) old = row0 == 0 ? in[tok * P.is[2]] * P.decay : out[tok * P.os[2]];
        cp_async_wait<R::DEPTH - 2>();
        __syncwarp();  // this step is there for all lanes, and all are done with the one before
        if (s + R::DEPTH - 1 < last) fetch(s + R::DEPTH - 1, slot == 0 ? R::DEPTH - 1 : slot - 1);
        else cp_async_commit();
        const uint32_t step = ring + slot * R::STEP;
        slot = slot + 1 == R::DEPTH ? 0 : slot + 1;
        float x[2][4];
        scores<D, G, ST, false>(x[0], Q, step, 0, lane);
        scores<D, G, ST, false>(x[1], Q, step, 1, lane);
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const float y[4] = {x[0][2 * r], x[0][2 * r + 1], x[1][2 * r], x[1][2 * r + 1]};
          const uint32_t on = draft ? seen_keys(T, b, true, node[r], true, k0, end, t) : 0xFu;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float v = fast_exp2(fmaf(y[j], Q.c[r], -sm[r])) * sl[r];
            if ((on >> j & 1u) && sl[r] != 0.0f) sum[j] += v;
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], d);
        }
        // key 8n + 2t + i of this step is sum[2n + i] of lanes with that t
        const int src = (lane & 7) >> 1;
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = __shfl_sync(0xffffffffu, sum[j], src);
        const float add = lane < 8 ? (lane & 1 ? v[1] : v[0]) : (lane & 1 ? v[3] : v[2]);
        if (lane < 16 && mine < end) out[tok * P.os[2]] = old + add;
      }
      cp_async_wait<0>();
      __syncwarp();  // the ring is free for the next pass
    }
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
bool half_rows(int rows) { return rows <= 8; }

MmaPlan mma_plan(const TreeParams &T) {
  MmaPlan L{};
  L.rows = T.R * T.nodes;
  const int nr = half_rows(L.rows) ? 8 : 16;
  L.row_tiles = (L.rows + nr - 1) / nr;
  L.units = T.B * T.Hkv;
  // one wave of blocks, each warp at least two steps of 16 keys; four where a
  // cluster does not hold the parts (32 rows x 4096 of 8 heads: 15.0 us with 16
  // parts, 16.9 with 27; 4 rows x 2048 7.4 with 8, 8.2 with 16)
  const int64_t steps = (T.S + 15) / 16 + (T.ndraft + 15) / 16, have = L.units * L.row_tiles;
  const int64_t room = static_cast<int64_t>(sm_count()) * (half_rows(L.rows) ? 4 : 3);
  const int64_t most = std::max({int64_t(1), std::min<int64_t>(kClusterParts, steps / (2 * NW)), steps / (4 * NW)});
  L.parts = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({room / have, most, 64})));
  L.cluster = L.parts > 1 && L.parts <= kClusterParts && !T.kept;  // score_kept joins the parts itself
  return L;
}

template <int D, int G, typename ST, bool HALF>
int launch_tree(const TreeParams &T, const MmaPlan &L, cudaStream_t st) {
  constexpr int NR = HALF ? 8 : 16;
  constexpr int meeting = NW * NR * ((D + 4) * 4 + 8) + NR * 8, rings = NW * Ring<D, G, true>::BYTES;
  constexpr int smem = meeting > rings ? meeting : rings;
  const auto kernel = HALF ? tree_mma8<D, G, ST> : tree_mma<D, G, ST>;
  static bool configured[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = 0;
  if (!configured[dev]) {
    const int rc = cuda_status(
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    if (rc) return rc;
    configured[dev] = true;
  }
  const int64_t blocks = L.units * L.row_tiles * L.parts;
  if (blocks > 0x7fffffff) return KV4_ERR_UNSUPPORTED;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(NW * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = static_cast<unsigned>(L.parts);
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = L.cluster ? 1 : 0;
  return cuda_status(cudaLaunchKernelEx(&cfg, kernel, T, L));
}

template <int D, int G, typename ST>
int launch_score(const ScoreParams &P, int rows, cudaStream_t st) {
  const int64_t steps = (P.t.S + 15) / 16 + (P.t.ndraft + 15) / 16, total = P.t.B * P.t.Hkv * steps;
  if (total >= (int64_t(1) << 31)) return KV4_ERR_UNSUPPORTED;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(
      std::min<int64_t>(static_cast<int64_t>(sm_count()) * 3, (total + NW - 1) / NW)));
  cfg.blockDim = dim3(NW * 32);
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, score_mma<D, G, ST>, P, rows, static_cast<uint32_t>(steps),
                                        static_cast<uint32_t>(total)));
}

// f(integral D, integral G, ST{})
template <class F>
int by_shape(const TreeParams &T, F f) {
  auto type = [&](auto d, auto g) {
    return T.s_dtype == KV4_BF16 ? f(d, g, __nv_bfloat16{}) : f(d, g, __half{});
  };
  if (T.d == 64) {
    if (T.G == 32) return type(std::integral_constant<int, 64>{}, std::integral_constant<int, 32>{});
    return type(std::integral_constant<int, 64>{}, std::integral_constant<int, 64>{});
  }
  if (T.G == 32) return type(std::integral_constant<int, 128>{}, std::integral_constant<int, 32>{});
  if (T.G == 64) return type(std::integral_constant<int, 128>{}, std::integral_constant<int, 64>{});
  return type(std::integral_constant<int, 128>{}, std::integral_constant<int, 128>{});
}

// rows of `pw` code bytes and `bytes` scale bytes without gaps between tokens
bool close_rows(const RowSource &S, int64_t B, int Hkv, int64_t T, int pw, int bytes) {
  if (T == 0) return true;
  const int e = bytes / 2;  // scales of a row
  if (T > 1 && (S.kps[2] != pw || S.vps[2] != pw || S.kss[2] != e || S.vss[2] != e)) return false;
  // scales are copied four bytes at a time
  if ((reinterpret_cast<uintptr_t>(S.ks) | reinterpret_cast<uintptr_t>(S.vs)) & 3u) return false;
  for (const int64_t *st : {S.kss, S.vss})
    if (st[3] != 1 || (Hkv > 1 && st[1] % 2) || (B > 1 && st[0] % 2)) return false;
  return true;
}

}  // namespace

// Whether warps in registers beat tensor-memory tiles (branch_tc.cu, trim_tc.cu).
// They take 1.3 us per SM for every 16 rows of a 128-key tile, whatever the
// total; the tiles 1.5 to 1.9 us for up to 128 rows, and about 18 us to begin and
// to join.  Measured (us, warps / tiles; 8 KV heads of 128 columns): 16 rows x
// 4K keys, batch 16 42 / 62; 32 rows x 4K, batch 1 17 / 37, batch 8 42 / 43, batch
// 16 79 / 62; 48 rows x 4K, batch 4 33 / 37, batch 8 56 / 44; 64 rows x 4K, batch 1
// 18 / 40, batch 4 41 / 37; 128 rows x 4K 26 / 44, x 1K, batch 4 28 / 34.
bool few_rows(const TreeParams &T) {
  const int64_t row_tiles = (static_cast<int64_t>(T.R) * T.nodes + 15) / 16;
  const int64_t tiles = T.B * T.Hkv * ((T.S + T.ndraft + 127) / 128);
  return tiles * (2 * row_tiles - 3) <= 26 * static_cast<int64_t>(sm_count());
}

// Whether the kernels of this file take the call: 16-bit queries and scales, the
// sizes they are built for, rows without gaps that aligned loads can read; and
// either little to do, or half precision somewhere, which branch_tc.cu leaves
// alone (a product of a code and an f16 scale does not fit an f16).
bool tree_mma_takes(const TreeParams &T) {
  if ((T.q_dtype != KV4_BF16 && T.q_dtype != KV4_F16) || (T.s_dtype != KV4_BF16 && T.s_dtype != KV4_F16))
    return false;
  if (T.d != 64 && T.d != 128) return false;
  if ((T.G != 32 && T.G != 64 && T.G != 128) || T.G > T.d) return false;
  if (!rows_ok(T.cache, T.B, T.Hkv, T.S) || !rows_ok(T.draft, T.B, T.Hkv, T.ndraft)) return false;
  const int bytes = 2 * T.d / T.G;
  if (!close_rows(T.cache, T.B, T.Hkv, T.S, T.d / 2, bytes) ||
      !close_rows(T.draft, T.B, T.Hkv, T.ndraft, T.d / 2, bytes))
    return false;
  if (!al16(T.q) || !al16(T.out) || T.qs[3] != 1 || T.os[3] != 1) return false;
  const int64_t n[3] = {T.B, static_cast<int64_t>(T.Hkv) * T.R, T.nodes};
  for (int i = 0; i < 3; ++i)
    if (n[i] > 1 && (T.qs[i] % 8 || T.os[i] % 8)) return false;
  return !tree_tc_takes(T) || few_rows(T);
}

int tree_mma_parts(const TreeParams &T) { return mma_plan(T).parts; }
bool tree_mma_joins(const TreeParams &T) { return mma_plan(T).cluster; }

int tree_mma_run(const TreeParams &T, cudaStream_t st) {
  const MmaPlan L = mma_plan(T);
  return by_shape(T, [&](auto d, auto g, auto s) {
    constexpr int D = decltype(d)::value, G = decltype(g)::value;
    if (half_rows(L.rows)) return launch_tree<D, G, decltype(s), true>(T, L, st);
    return launch_tree<D, G, decltype(s), false>(T, L, st);
  });
}

int score_mma_run(const ScoreParams &P, cudaStream_t st) {
  return by_shape(P.t, [&](auto d, auto g, auto s) {
    return launch_score<decltype(d)::value, decltype(g)::value, decltype(s)>(P, P.t.R * P.t.nodes, st);
  });
}

int branch_mma_take_device_error(int *v) {
  int zero = 0;
  int rc = cuda_status(cudaMemcpyFromSymbol(v, g_branch_error_mma, sizeof(int)));
  if (rc) return rc;
  return cuda_status(cudaMemcpyToSymbol(g_branch_error_mma, &zero, sizeof(int)));
}

}  // namespace kv4
