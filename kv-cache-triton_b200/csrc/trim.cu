// Attention that scores the cached tokens, and eviction by that score.
//
// Scored attention: out as ordinary attention over the cache, and
//
//   score'[b, g, t] = decay * score[b, g, t] + sum over the queries i and the
//                     q heads h of KV head g of softmax(x[b, h, i])[t]
//
// The weights are known only when a row's maximum and sum are, so the keys are
// read twice: the attention leaves (maximum, 1 / sum) of each row, and
// score_generic forms the weights again, a key per lane, summed over the rows
// in a fixed order (no atomics: two calls give the same bits).  bf16 queries
// over bf16 scales take trim_tc.cu's kernel where the layout allows.
//
// Eviction cuts each (sequence, KV head) to `keep` tokens: the first `sinks`,
// the last `recent` and, of the rest, those with the highest score (equal
// scores: the earlier token; NaN below everything).  evict_select finds the
// threshold by radix select and writes the kept indices in token order;
// evict_gather moves the rows.
#include <algorithm>

#include "branch.cuh"

namespace kv4 {
namespace {

constexpr int SROWS = 8;  // query rows a warp holds at a time

// A warp per 32 keys of one (sequence, KV head).
__global__ void score_generic(const ScoreParams P, int warps, int ld, int64_t tiles, int64_t tasks) {
  extern __shared__ __align__(16) float ssm[];
  const TreeParams &T = P.t;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t task = static_cast<int64_t>(blockIdx.x) * warps + warp;
  if (task >= tasks) return;
  float *sK = ssm + warp * (32 + SROWS) * ld, *sQ = sK + 32 * ld;
  const int64_t unit = task / tiles, t0 = (task - unit * tiles) * 32, b = unit / T.Hkv;
  const int kvh = static_cast<int>(unit - b * T.Hkv);
  const int rows = T.nodes * T.R, d8 = (T.d + 7) >> 3;
  const int64_t t = t0 + lane;
  warp_dequant_tile(T, false, b, kvh, T.S, t0, P.keys, sK, ld, lane);
  float total = 0.0f;
  for (int r0 = 0; r0 < rows; r0 += SROWS) {
    __syncwarp();
    const int nr = min(SROWS, rows - r0);
    for (int r = 0; r < nr; ++r) {
      const int row = r0 + r, i = row / T.R, h = kvh * T.R + row - i * T.R;
      for (int c = lane; c < 8 * d8; c += 32)
        sQ[r * ld + c] = c < T.d ? load_as_f32(T.q, T.q_dtype,
                                               b * T.qs[0] + h * T.qs[1] + i * T.qs[2] + c * T.qs[3])
                                 : 0.0f;
    }
    __syncwarp();
    float s[SROWS];
#pragma unroll
    for (int r = 0; r < SROWS; ++r) s[r] = 0.0f;
    for (int c = 0; c < 2 * d8; ++c) {
      const float4 k4 = *reinterpret_cast<const float4 *>(sK + lane * ld + 4 * c);
#pragma unroll
      for (int r = 0; r < SROWS; ++r) {
        if (r >= nr) break;
        const float4 q4 = *reinterpret_cast<const float4 *>(sQ + r * ld + 4 * c);
        s[r] = fmaf(q4.x, k4.x, s[r]);
        s[r] = fmaf(q4.y, k4.y, s[r]);
        s[r] = fmaf(q4.z, k4.z, s[r]);
        s[r] = fmaf(q4.w, k4.w, s[r]);
      }
    }
#pragma unroll
    for (int r = 0; r < SROWS; ++r) {
      if (r >= nr) break;
      const int row = r0 + r;
      bool see = t < P.keys;
      if (see && t >= T.S) see = draft_visible(T, b, row / T.R, static_cast<int>(t - T.S));
      const float2 st = T.stats[unit * rows + row];
      if (see && st.y > 0.0f) total = fmaf(exp2f(s[r] * T.scale_log2 - st.x), st.y, total);
    }
  }
  if (t < P.keys) {
    const float old = P.in[b * P.is[0] + kvh * P.is[1] + t * P.is[2]];
    P.out[b * P.os[0] + kvh * P.os[1] + t * P.os[2]] = fmaf(old, P.decay, total);
  }
}

}  // namespace

int score_run(const ScoreParams &P, cudaStream_t st) {
  const TreeParams &T = P.t;
  const int ld = row_ld(T.d);
  const size_t per_warp = sizeof(float) * (32 + SROWS) * ld;
  const int warps = static_cast<int>(std::max<size_t>(1, std::min<size_t>(4, 100 * 1024 / per_warp)));
  const int64_t tiles = (P.keys + 31) / 32, tasks = T.B * T.Hkv * tiles;
  const int64_t blocks = (tasks + warps - 1) / warps;
  if (blocks > 0x7fffffff) return KV4_ERR_UNSUPPORTED;
  if (blocks == 0) return KV4_OK;
  if (per_warp * warps > 48 * 1024) {
    const int rc = cuda_status(cudaFuncSetAttribute(
        score_generic, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024));
    if (rc) return rc;
  }
  score_generic<<<static_cast<unsigned>(blocks), 32 * warps, per_warp * warps, st>>>(P, warps, ld,
                                                                                    tiles, tasks);
  return cuda_status(cudaGetLastError());
}

namespace {

// rows [from, to) of the token dimension
kv4_tensor token_range(const kv4_tensor *t, int64_t from, int64_t to) {
  kv4_tensor r = *t;
  r.data = static_cast<char *>(t->data) + from * t->stride[2] * dtype_size(t->dtype);
  r.shape[2] = to - from;
  return r;
}

// The call's attention as one over context [0, S - n) and drafted rows
// [S - n, S) with n = min(queries, S): bottom-right causal is then a rule
// about the drafted rows alone.
int scored_fill(TreeParams &P, kv4_tensor ctx[4], kv4_tensor tail[4], const kv4_tensor *q,
                const kv4_tensor *const cache[4], const kv4_tensor *out, int G, int is_causal,
                float sm_scale) {
  if (!q) return KV4_ERR_INVALID;
  for (int k = 0; k < 4; ++k)
    if (!cache[k]) return KV4_ERR_INVALID;
  const int64_t S = cache[0]->shape[2];
  for (int k = 1; k < 4; ++k)
    if (cache[k]->shape[2] != S) return KV4_ERR_SHAPE;
  // a single query sees everything either way
  const int64_t n = is_causal && q->shape[2] > 1 ? std::min(q->shape[2], S) : 0;
  const kv4_tensor *pc[4], *pt[4];
  for (int k = 0; k < 4; ++k) {
    ctx[k] = token_range(cache[k], 0, S - n);
    tail[k] = token_range(cache[k], S - n, S);
    pc[k] = &ctx[k];
    pt[k] = n ? &tail[k] : nullptr;
  }
  const int rc = tree_fill(P, q, pc, pt, out, G, sm_scale);
  P.causal = 1;
  P.shift = static_cast<int>(n - q->shape[2]);
  return rc;
}

int64_t stats_bytes(const TreeParams &P) {
  return (P.B * P.Hkv * P.nodes * P.R * static_cast<int64_t>(sizeof(float2)) + 255) / 256 * 256;
}

// ---------------------------------------------------------------------------
// eviction
// ---------------------------------------------------------------------------
struct EvictParams {
  const float *mass;
  int64_t ms[3];  // batch, head, token strides
  int32_t *index;  // [B, Hkv, keep]
  int64_t S;
  int Hkv, keep, recent, sinks;
};

// order-preserving 32-bit key of a score: NaN lowest, -0 as +0
__device__ __forceinline__ uint32_t score_key(float x) {
  if (x != x) return 0u;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

constexpr int SEL = 1024;

// A block per (sequence, KV head): four passes of eight bits find the
// threshold key, a fifth writes the kept indices by block-wide prefix sums.
__global__ void __launch_bounds__(SEL) evict_select(const EvictParams P) {
  __shared__ int hist[256];
  __shared__ uint32_t s_prefix;
  __shared__ int s_left;
  __shared__ int w_gt[32], w_eq[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t b = blockIdx.x / P.Hkv, h = blockIdx.x - b * P.Hkv;
  const float *mass = P.mass + b * P.ms[0] + h * P.ms[1];
  const int64_t lo = P.sinks, hi = P.S - P.recent;
  int left = P.keep - P.sinks - P.recent;  // still to be taken among equals
  uint32_t prefix = 0, known = 0;
  if (left > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int64_t t = lo + tid; t < hi; t += SEL) {
        const uint32_t k = score_key(mass[t * P.ms[2]]);
        if ((k & known) == prefix) atomicAdd(&hist[(k >> shift) & 255u], 1);
      }
      __syncthreads();
      if (tid == 0) {
        int bin = 255, above = 0;
        while (bin > 0 && above + hist[bin] < left) above += hist[bin--];
        s_prefix = prefix | (static_cast<uint32_t>(bin) << shift);
        s_left = left - above;
      }
      __syncthreads();
      prefix = s_prefix;
      left = s_left;
      known |= 255u << shift;
    }
  }
  const bool none = P.keep - P.sinks - P.recent <= 0;
  int32_t *out = P.index + static_cast<int64_t>(blockIdx.x) * P.keep;
  int gt_base = 0, eq_base = 0;  // kept for sure, and equal to the threshold, so far
  for (int64_t c = 0; c < P.S; c += SEL) {
    const int64_t t = c + tid;
    bool gt = false, eq = false;
    if (t < P.S) {
      if (t < lo || t >= hi) gt = true;
      else if (!none) {
        const uint32_t k = score_key(mass[t * P.ms[2]]);
        gt = k > prefix;
        eq = k == prefix;
      }
    }
    const uint32_t mg = __ballot_sync(0xffffffffu, gt), me = __ballot_sync(0xffffffffu, eq);
    __syncthreads();
    if (lane == 0) {
      w_gt[warp] = __popc(mg);
      w_eq[warp] = __popc(me);
    }
    __syncthreads();
    int g = gt_base, e = eq_base;
    for (int w = 0; w < SEL / 32; ++w) {
      if (w < warp) {
        g += w_gt[w];
        e += w_eq[w];
      }
      gt_base += w_gt[w];
      eq_base += w_eq[w];
    }
    const uint32_t before = (1u << lane) - 1u;
    g += __popc(mg & before);
    e += __popc(me & before);
    if (gt || (eq && e < left)) out[g + min(e, left)] = static_cast<int32_t>(t);
  }
}

struct GatherParams {
  const uint8_t *src[5];
  uint8_t *dst[5];
  int64_t ss[5][3], ds[5][3];  // batch, head, token strides (bytes)
  int bytes[5], vec[5];        // of a row; of one copy
  const int32_t *index;
  int Hkv, keep, tiles;
};

constexpr int GROWS = 64;  // kept rows per block

template <typename V>
__device__ __forceinline__ void gather_rows(const GatherParams &P, int k, int64_t b, int64_t h,
                                            int j0, int n, const int32_t *idx) {
  const int per = P.bytes[k] / static_cast<int>(sizeof(V));
  const uint8_t *src = P.src[k] + b * P.ss[k][0] + h * P.ss[k][1];
  uint8_t *dst = P.dst[k] + b * P.ds[k][0] + h * P.ds[k][1];
  for (int e = threadIdx.x; e < n * per; e += blockDim.x) {
    const int j = e / per, c = e - j * per;
    reinterpret_cast<V *>(dst + (j0 + j) * P.ds[k][2])[c] =
        __ldg(reinterpret_cast<const V *>(src + idx[j] * P.ss[k][2]) + c);
  }
}

__global__ void __launch_bounds__(256) evict_gather(const GatherParams P) {
  __shared__ int32_t idx[GROWS];
  const int64_t unit = blockIdx.x / P.tiles, b = unit / P.Hkv, h = unit - b * P.Hkv;
  const int j0 = static_cast<int>(blockIdx.x - unit * P.tiles) * GROWS, n = min(GROWS, P.keep - j0);
  if (static_cast<int>(threadIdx.x) < n) idx[threadIdx.x] = P.index[unit * P.keep + j0 + threadIdx.x];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 5; ++k) {
    switch (P.vec[k]) {
      case 16: gather_rows<uint4>(P, k, b, h, j0, n, idx); break;
      case 8: gather_rows<uint2>(P, k, b, h, j0, n, idx); break;
      case 4: gather_rows<uint32_t>(P, k, b, h, j0, n, idx); break;
      case 2: gather_rows<uint16_t>(P, k, b, h, j0, n, idx); break;
      default: gather_rows<uint8_t>(P, k, b, h, j0, n, idx); break;
    }
  }
}

// the widest copy that the rows of both sides allow
int copy_width(const GatherParams &P, int k) {
  uint64_t a = reinterpret_cast<uintptr_t>(P.src[k]) | reinterpret_cast<uintptr_t>(P.dst[k]) |
               static_cast<uint64_t>(P.bytes[k]);
  for (int i = 0; i < 3; ++i) a |= static_cast<uint64_t>(P.ss[k][i] | P.ds[k][i]);
  int v = 16;
  while (a & (v - 1)) v >>= 1;
  return v;
}

bool is_float(int dt) { return dt == KV4_F32 || dt == KV4_F16 || dt == KV4_BF16; }

}  // namespace
}  // namespace kv4

using namespace kv4;

extern "C" int64_t kv4_scored_workspace(const kv4_tensor *q, const kv4_tensor *k_packed,
                                        const kv4_tensor *k_scales, const kv4_tensor *v_packed,
                                        const kv4_tensor *v_scales, int group_size,
                                        int is_causal) {
  const kv4_tensor *cache[4] = {k_packed, k_scales, v_packed, v_scales};
  kv4_tensor ctx[4], tail[4];
  TreeParams P{};
  const int rc = scored_fill(P, ctx, tail, q, cache, q, group_size, is_causal, 0.0f);
  return rc ? -rc : stats_bytes(P) + tree_workspace(P);
}

extern "C" int kv4_scored_attention(const kv4_tensor *q, const kv4_tensor *k_packed,
                                    const kv4_tensor *k_scales, const kv4_tensor *v_packed,
                                    const kv4_tensor *v_scales, const kv4_tensor *score_in,
                                    const kv4_tensor *score_out, const kv4_tensor *out,
                                    int group_size, int is_causal, float decay, float sm_scale,
                                    void *workspace, size_t workspace_bytes, void *stream) {
  const kv4_tensor *cache[4] = {k_packed, k_scales, v_packed, v_scales};
  if (!score_in || !score_out || !out) return KV4_ERR_INVALID;
  kv4_tensor ctx[4], tail[4];
  ScoreParams P{};
  int rc = scored_fill(P.t, ctx, tail, q, cache, out, group_size, is_causal, sm_scale);
  if (rc) return rc;
  P.keys = cache[0]->shape[2];
  for (const kv4_tensor *s : {score_in, score_out}) {
    if (s->dtype != KV4_F32) return KV4_ERR_DTYPE;
    if (s->shape[0] != 1 || s->shape[1] != P.t.B || s->shape[2] != P.t.Hkv || s->shape[3] != P.keys)
      return KV4_ERR_SHAPE;
  }
  P.in = static_cast<const float *>(score_in->data);
  P.out = static_cast<float *>(score_out->data);
  for (int i = 0; i < 3; ++i) {
    P.is[i] = score_in->stride[i + 1];
    P.os[i] = score_out->stride[i + 1];
  }
  P.decay = decay;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t sb = stats_bytes(P.t);
  if (sb > 0 && (!workspace || static_cast<int64_t>(workspace_bytes) < sb)) return KV4_ERR_WORKSPACE;
  P.t.stats = static_cast<float2 *>(workspace);
  rc = tree_run(P.t, static_cast<char *>(workspace) + sb,
                static_cast<int64_t>(workspace_bytes) - sb, st);
  if (rc) return rc;
  return score_tc_takes(P) ? score_tc_run(P, st) : score_run(P, st);
}

extern "C" int kv4_evict(const kv4_tensor *k_packed, const kv4_tensor *k_scales,
                         const kv4_tensor *v_packed, const kv4_tensor *v_scales,
                         const kv4_tensor *score, const kv4_tensor *out_k_packed,
                         const kv4_tensor *out_k_scales, const kv4_tensor *out_v_packed,
                         const kv4_tensor *out_v_scales, const kv4_tensor *out_score,
                         int32_t *index, int64_t recent, int64_t sinks, void *stream) {
  const kv4_tensor *src[5] = {k_packed, k_scales, v_packed, v_scales, score};
  const kv4_tensor *dst[5] = {out_k_packed, out_k_scales, out_v_packed, out_v_scales, out_score};
  for (int k = 0; k < 5; ++k)
    if (!src[k] || !dst[k]) return KV4_ERR_INVALID;
  if (score->dtype != KV4_F32) return KV4_ERR_DTYPE;
  const int64_t B = k_packed->shape[0], Hkv = k_packed->shape[1], S = k_packed->shape[2];
  const int64_t keep = out_k_packed->shape[2];
  GatherParams G{};
  for (int k = 0; k < 5; ++k) {
    const kv4_tensor *s = src[k], *o = dst[k];
    if (s->dtype != o->dtype) return KV4_ERR_DTYPE;
    if (k < 4 && ((k & 1) ? !is_float(s->dtype) : s->dtype != KV4_U8)) return KV4_ERR_DTYPE;
    // rows [B, Hkv, T, width]; the scores are [1, B, Hkv, T]
    const int at = k < 4 ? 0 : 1;
    if (s->shape[at] != B || s->shape[at + 1] != Hkv || s->shape[at + 2] != S ||
        o->shape[at] != B || o->shape[at + 1] != Hkv || o->shape[at + 2] != keep)
      return KV4_ERR_SHAPE;
    if (k < 4 && s->shape[3] != o->shape[3]) return KV4_ERR_SHAPE;
    if (k < 4 && s->shape[3] > 1 && (s->stride[3] != 1 || o->stride[3] != 1)) return KV4_ERR_LAYOUT;
    const int e = dtype_size(s->dtype);
    G.bytes[k] = static_cast<int>(k < 4 ? s->shape[3] * e : e);
    G.src[k] = static_cast<const uint8_t *>(s->data);
    G.dst[k] = static_cast<uint8_t *>(o->data);
    for (int i = 0; i < 3; ++i) {
      G.ss[k][i] = s->stride[at + i] * e;
      G.ds[k][i] = o->stride[at + i] * e;
    }
    G.vec[k] = copy_width(G, k);
  }
  if (recent < 0 || sinks < 0 || keep < 0 || recent + sinks > keep || keep > S)
    return KV4_ERR_INVALID;
  if (S >= (int64_t(1) << 30)) return KV4_ERR_UNSUPPORTED;
  if (B == 0 || Hkv == 0 || keep == 0) return KV4_OK;
  if (!index) return KV4_ERR_INVALID;
  const int64_t tiles = (keep + GROWS - 1) / GROWS;
  if (B * Hkv * tiles > 0x7fffffff) return KV4_ERR_UNSUPPORTED;
  EvictParams E{};
  E.mass = static_cast<const float *>(score->data);
  for (int i = 0; i < 3; ++i) E.ms[i] = score->stride[i + 1];
  E.index = index;
  E.S = S;
  E.Hkv = static_cast<int>(Hkv);
  E.keep = static_cast<int>(keep);
  E.recent = static_cast<int>(recent);
  E.sinks = static_cast<int>(sinks);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  evict_select<<<static_cast<unsigned>(B * Hkv), SEL, 0, st>>>(E);
  int rc = cuda_status(cudaGetLastError());
  if (rc) return rc;
  G.index = index;
  G.Hkv = static_cast<int>(Hkv);
  G.keep = static_cast<int>(keep);
  G.tiles = static_cast<int>(tiles);
  evict_gather<<<static_cast<unsigned>(B * Hkv * tiles), 256, 0, st>>>(G);
  return cuda_status(cudaGetLastError());
}
