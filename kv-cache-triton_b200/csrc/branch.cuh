// Shared declarations of the operators that branch and trim the INT4 cache
// (branch.cu: tree attention and the commit of an accepted path; trim.cu:
// attention that scores the cached tokens, and eviction).
#pragma once

#include "common.cuh"

namespace kv4 {

constexpr float kBrLog2e = 1.4426950408889634f;
constexpr float kBrLn2 = 0.6931471805599453f;

// Packed K and V rows and their scales: [B, Hkv, T, ...], strides in bytes
// for the codes and in elements for the scales (batch, head, token, column).
struct RowSource {
  const uint8_t *kp, *vp;
  const void *ks, *vs;
  int64_t kps[4], vps[4], kss[4], vss[4];
};

// Attention of `nodes` query rows per sequence over the cache's context rows
// [0, len_b) followed by `ndraft` rows of `draft`.  Node i sees every context
// row and draft row j iff mask[b, i, j] (when given), or j <= i + shift (when
// causal), or always.
struct TreeParams {
  const void *q;
  void *out;
  float *lse;  // natural log, or null
  int q_dtype, s_dtype;
  int64_t qs[4], os[4], ls[3];
  RowSource cache, draft;
  const uint8_t *mask;
  int64_t ms[3];  // batch, node, draft strides (bytes)
  const int32_t *lens;  // context rows of each sequence, or null: all of them
  int64_t B;
  int Hkv, R, nodes, ndraft, d, G, causal, shift;
  int words;           // bytes that rows of codes can be read in (16, 4: eight codes of a group a word; 0: one)
  int64_t S;           // context rows in the cache views
  float scale_log2;    // sm_scale * log2(e)
  float2 *stats;       // per (unit, row): base-2 maximum and 1 / sum; or null
  float *ws_o;         // split partials, see the kernels
  float2 *ws_ml;
  float *kept;         // raw scores of every row, see kept_at; or null
  float *kept_c;       // per (unit, row): factor from those to base-2 exponents
};

// Kept scores lie in blocks of 16 keys, [unit][block][row][16]; context rows
// fill whole blocks, drafted rows begin a new one.
__host__ __device__ __forceinline__ int64_t kept_blocks(const TreeParams &P) {
  return ((P.S + 15) >> 4) + ((P.ndraft + 15) >> 4);
}
__device__ __forceinline__ int64_t kept_at(int64_t unit, int64_t blocks, int64_t slot, int row, int rows) {
  return ((unit * blocks + (slot >> 4)) * rows + row) * 16 + (slot & 15);
}

// context rows of sequence b; an entry outside [0, S] is reported and read as 0
__device__ __forceinline__ int64_t context_len(const TreeParams &P, int64_t b, int *err) {
  if (!P.lens) return P.S;
  const int n = __ldg(P.lens + b);
  if (n < 0 || n > P.S) {
    if (err) atomicOr(err, DEV_ERR_BAD_LENGTH);
    return 0;
  }
  return n;
}

__device__ __forceinline__ bool draft_visible(const TreeParams &P, int64_t b, int i, int j) {
  if (P.mask) return P.mask[b * P.ms[0] + i * P.ms[1] + j * P.ms[2]] != 0;
  return !P.causal || j <= i + P.shift;
}

// Fill everything of P that comes from the arguments; KV4_OK or the reason.
// draft tensors null: no drafted rows.
int tree_fill(TreeParams &P, const kv4_tensor *q, const kv4_tensor *const cache[4],
              const kv4_tensor *const draft[4], const kv4_tensor *out, int group_size,
              float sm_scale);
// Workspace bytes of tree_run and the run itself (branch.cu).
int64_t tree_workspace(const TreeParams &P);
int tree_run(TreeParams &P, void *workspace, int64_t bytes, cudaStream_t st);

// Bytes of the widest copy that rows of `bytes` bytes allow, given the
// addresses and strides (batch, head, token) of both sides.
inline int copy_width(const void *dst, const void *src, int bytes, const int64_t (&ds)[3],
                      const int64_t (&ss)[3]) {
  uint64_t a = reinterpret_cast<uintptr_t>(dst) | reinterpret_cast<uintptr_t>(src) |
               static_cast<uint64_t>(bytes);
  for (int i = 0; i < 3; ++i) a |= static_cast<uint64_t>(ds[i] | ss[i]);
  int v = 16;
  while (a & (v - 1)) v >>= 1;
  return v;
}

// 8 elements of a packed row as floats times their scale, element by element:
// columns [8c, 8c + 8), those at or past d are 0
template <typename ST>
__device__ __forceinline__ void dequant8(const uint8_t *row, int64_t cs, const ST *srow, int64_t scs,
                                         int G, int pb, int d, int c, float (&v)[8]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const int e = 8 * c + k;
    v[k] = 0.0f;
    if (e < d) {
      const int g = e / G, nib = g * 2 * pb + (e - g * G);
      const uint32_t byte = row[(nib >> 1) * cs];
      const int code = (nib & 1) ? byte >> 4 : byte & 15;
      v[k] = static_cast<float>(code - 8) * to_f32(srow[g * scs]);
    }
  }
}

// 32 rows (keys t0 .. t0+31 of `len` context rows then draft rows) of K or V
// as floats in shared memory, ld floats apart, by one warp, a row per lane; rows
// at or past `end` are 0.  d is padded with zeros to a multiple of 8.  Where rows
// can be read in words, up to 16 of them (128 columns) are in flight.
template <typename ST>
__device__ __forceinline__ void warp_dequant_rows(const TreeParams &P, bool is_v, int64_t b, int h,
                                                  int64_t len, int64_t t0, int64_t end, float *dst,
                                                  int ld, int lane) {
  const int d8 = (P.d + 7) >> 3, pb = (P.G + 1) >> 1;
  const int64_t t = t0 + lane;
  const bool in = t < end, ctx = t < len;
  const RowSource &S = ctx ? P.cache : P.draft;
  const int64_t row = ctx ? t : t - len;
  const int64_t *ps = is_v ? S.vps : S.kps, *ss = is_v ? S.vss : S.kss;
  const uint8_t *p = (is_v ? S.vp : S.kp) + b * ps[0] + h * ps[1] + row * ps[2];
  const ST *q = static_cast<const ST *>(is_v ? S.vs : S.ks) + b * ss[0] + h * ss[1] + row * ss[2];
  const int64_t cs = ps[3], scs = ss[3];
  float4 *o = reinterpret_cast<float4 *>(dst + lane * ld);
  if (P.words) {
    const int lg = __ffs(P.G) - 1;  // groups of a power of two, at least 8
    const uint32_t *pw = reinterpret_cast<const uint32_t *>(p);
#pragma unroll 1
    for (int c0 = 0; c0 < d8; c0 += 16) {
      uint32_t w[16];
      ST s[16];
#pragma unroll
      for (int u = 0; u < 16; u += 4) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (in && c0 + u < d8) {
          if (P.words == 16) {
            v = __ldg(reinterpret_cast<const uint4 *>(pw + c0 + u));
          } else {
            v.x = __ldg(pw + c0 + u);
            if (c0 + u + 1 < d8) v.y = __ldg(pw + c0 + u + 1);
            if (c0 + u + 2 < d8) v.z = __ldg(pw + c0 + u + 2);
            if (c0 + u + 3 < d8) v.w = __ldg(pw + c0 + u + 3);
          }
        }
        w[u] = v.x;
        w[u + 1] = v.y;
        w[u + 2] = v.z;
        w[u + 3] = v.w;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[u + e] = from_f32<ST>(0.0f);
          if (e > 0 && P.G >= 32) s[u + e] = s[u];
          else if (in && c0 + u + e < d8) s[u + e] = q[((8 * (c0 + u + e)) >> lg) * scs];
        }
      }
#pragma unroll
      for (int u = 0; u < 16; ++u) {
        if (c0 + u >= d8) break;
        const float f = to_f32(s[u]);
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)  // 2^23 + code, then code - 8: exact
          v[k] = (__uint_as_float(0x4B000000u | ((w[u] >> (4 * k)) & 15u)) - 8388616.0f) * f;
        o[2 * (c0 + u)] = make_float4(v[0], v[1], v[2], v[3]);
        o[2 * (c0 + u) + 1] = make_float4(v[4], v[5], v[6], v[7]);
      }
    }
    return;
  }
#pragma unroll 1
  for (int c = 0; c < d8; ++c) {
    float v[8] = {};
    if (in) dequant8<ST>(p, cs, q, scs, P.G, pb, P.d, c, v);
    o[2 * c] = make_float4(v[0], v[1], v[2], v[3]);
    o[2 * c + 1] = make_float4(v[4], v[5], v[6], v[7]);
  }
}
__device__ __forceinline__ void warp_dequant_tile(const TreeParams &P, bool is_v, int64_t b, int h,
                                                  int64_t len, int64_t t0, int64_t end, float *dst,
                                                  int ld, int lane) {
  if (P.s_dtype == KV4_F32) warp_dequant_rows<float>(P, is_v, b, h, len, t0, end, dst, ld, lane);
  else if (P.s_dtype == KV4_F16) warp_dequant_rows<__half>(P, is_v, b, h, len, t0, end, dst, ld, lane);
  else warp_dequant_rows<__nv_bfloat16>(P, is_v, b, h, len, t0, end, dst, ld, lane);
}

// N rows from row0 on of a KV head's queries (row = node * R + head of the
// group) as floats in shared memory, ld apart, by one warp; rows at or past
// `rows` and columns past d are 0.
template <typename QT, int N>
__device__ __forceinline__ void warp_query_rows(const TreeParams &P, int64_t b, int kvh, int row0,
                                                int rows, float *dst, int ld, int lane) {
  const int w = (P.d + 7) & ~7;
  const QT *q[N];
#pragma unroll
  for (int r = 0; r < N; ++r) {
    const int row = row0 + r, i = row / P.R, h = kvh * P.R + row - i * P.R;
    q[r] = row < rows ? static_cast<const QT *>(P.q) + b * P.qs[0] + h * P.qs[1] + i * P.qs[2] : nullptr;
  }
#pragma unroll 1
  for (int c = lane; c < w; c += 32) {
    QT v[N];
#pragma unroll
    for (int r = 0; r < N; ++r) v[r] = q[r] && c < P.d ? q[r][c * P.qs[3]] : from_f32<QT>(0.0f);
#pragma unroll
    for (int r = 0; r < N; ++r) dst[r * ld + c] = to_f32(v[r]);
  }
}
template <int N>
__device__ __forceinline__ void warp_query(const TreeParams &P, int64_t b, int kvh, int row0, int rows,
                                           float *dst, int ld, int lane) {
  if (P.q_dtype == KV4_F32) warp_query_rows<float, N>(P, b, kvh, row0, rows, dst, ld, lane);
  else if (P.q_dtype == KV4_F16) warp_query_rows<__half, N>(P, b, kvh, row0, rows, dst, ld, lane);
  else warp_query_rows<__nv_bfloat16, N>(P, b, kvh, row0, rows, dst, ld, lane);
}

// four sums side by side: a quarter of the roundings in a row (error of an fp32 score
// of 64 columns against 64 bits: half of one sum's)
__device__ __forceinline__ void fma4(float4 &s, const float4 &a, const float4 &b) {
  s.x = fmaf(a.x, b.x, s.x);
  s.y = fmaf(a.y, b.y, s.y);
  s.z = fmaf(a.z, b.z, s.z);
  s.w = fmaf(a.w, b.w, s.w);
}
__device__ __forceinline__ float sum4(const float4 &s) { return (s.x + s.y) + (s.z + s.w); }

// shared-memory row length of a d-wide row: float4 steps, an odd number of
// them, so that 32 rows read in step fall into different banks
__host__ __device__ constexpr int row_ld(int d) { return 4 * (((d + 7) / 8 * 2) | 1); }

// Scores of the cached tokens: the attention in `t` (its rows' maxima and
// sums in t.stats), the running scores in and out.
struct ScoreParams {
  TreeParams t;
  const float *in;
  float *out;
  int64_t is[3], os[3];  // batch, head, token strides of the scores
  float decay;
  int64_t keys;          // tokens in the cache: context plus drafted rows
};

bool tree_tc_takes(const TreeParams &P);                   // branch_tc.cu
int score_tc_run(const ScoreParams &P, cudaStream_t st);   // trim_tc.cu
bool tree_mma_takes(const TreeParams &P);                  // branch_mma.cu
int score_mma_run(const ScoreParams &P, cudaStream_t st);

}  // namespace kv4
