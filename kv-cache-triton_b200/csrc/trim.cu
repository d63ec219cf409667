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
// in a fixed order (no atomics: two calls give the same bits).  16-bit types
// take the kernels of branch_mma.cu and trim_tc.cu where the layout allows.
//
// Eviction cuts each (sequence, KV head) to `keep` tokens: the first `sinks`,
// the last `recent` and, of the rest, those with the highest score (equal
// scores: the earlier token; NaN below everything).  evict_select finds the
// threshold by radix select and writes the kept indices in token order;
// evict_gather moves the rows.  The scores are read once and the kept rows
// once, which is what eviction cannot do without; memory bounds it.
#include <algorithm>

#include "merge.cuh"

namespace kv4 {
namespace {

constexpr int SROWS = 8;  // query rows a warp holds at a time

// A warp per 32 keys of one (sequence, KV head); bound by instructions like
// tree_generic (fp32, 32 rows x 2000 keys x 8 heads of 128, batch 2: 48 us).
__global__ void __launch_bounds__(128, 2) score_generic(const ScoreParams P, int warps, int ld, int64_t tiles, int64_t tasks) {
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
    warp_query<SROWS>(T, b, kvh, r0, rows, sQ, ld, lane);
    __syncwarp();
    float4 s[SROWS];  // four sums per score, as in tree_generic
#pragma unroll
    for (int r = 0; r < SROWS; ++r) s[r] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int c = 0; c < 2 * d8; ++c) {
      const float4 k4 = *reinterpret_cast<const float4 *>(sK + lane * ld + 4 * c);
#pragma unroll
      for (int r = 0; r < SROWS; ++r) {
        if (r >= nr) break;
        fma4(s[r], *reinterpret_cast<const float4 *>(sQ + r * ld + 4 * c), k4);
      }
    }
#pragma unroll
    for (int r = 0; r < SROWS; ++r) {
      if (r >= nr) break;
      const int row = r0 + r;
      bool see = t < P.keys;
      if (see && t >= T.S) see = draft_visible(T, b, row / T.R, static_cast<int>(t - T.S));
      const float2 st = T.stats[unit * rows + row];  // 1 / sum 0: a row that saw nothing; NaN: a row without a value
      if (see && st.y != 0.0f) total = fmaf(exp2f(fmaf(sum4(s[r]), T.scale_log2, -st.x)), st.y, total);
    }
  }
  if (t < P.keys) {
    const float old = P.in[b * P.is[0] + kvh * P.is[1] + t * P.is[2]];
    P.out[b * P.os[0] + kvh * P.os[1] + t * P.os[2]] = fmaf(old, P.decay, total);
  }
}

constexpr int KTHREADS = 256;  // of score_kept
constexpr int KROWS = 16;      // most rows of a KV head whose scores are kept

// Few rows (single tokens above all): the attention keeps its scores, 4 bytes a
// row and key where the keys themselves are d / 2 and their scales, so nothing
// is read or multiplied twice, and its parts are joined here too.  The first
// `joins` blocks join the outputs, a warp per row; the others take 256 keys of a
// (sequence, KV head) each: their warps join the rows' maxima and sums, then a
// thread sums the weights of its keys, PER of them.  Against reading K again, 16
// sequences x 4096 x 4 rows: 24 us -> 7 (8.4 MB of scores, from L2); fp32, 1023
// tokens: 13 -> 3.3, the join included.
template <int DC, int PER>
__global__ void __launch_bounds__(KTHREADS, 4)
    score_kept(const __grid_constant__ ScoreParams P, const GenPlan L, int joins, int blocks) {
  __shared__ float sm[KROWS], sl[KROWS], sc[KROWS];
  const TreeParams &T = P.t;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (static_cast<int>(blockIdx.x) < joins) {
    const int64_t at = static_cast<int64_t>(blockIdx.x) * (KTHREADS / 32) + warp;
    griddep_wait();
    if (at < L.units * L.rows) merge_row<DC>(T, L, at, lane);
    return;
  }
  const int at = static_cast<int>(blockIdx.x) - joins, unit = at / blocks, b = unit / T.Hkv;
  const int kvh = unit - b * T.Hkv;
  const int64_t slot0 = static_cast<int64_t>(at - unit * blocks) * (PER * KTHREADS) + tid;
  const int64_t ctx = (T.S + 15) & ~int64_t(15);
  const float *in = P.in + b * P.is[0] + kvh * P.is[1];
  float *out = P.out + b * P.os[0] + kvh * P.os[1];
  float old[PER], sum[PER];  // the weights are summed before they meet the score, and its rounding
  bool on[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int64_t slot = slot0 + i * KTHREADS, t = slot < ctx ? slot : T.S + slot - ctx;
    on[i] = slot < ctx ? slot < T.S : t < P.keys;
    old[i] = on[i] ? in[t * P.is[2]] : 0.0f;  // was there before the attention began
    sum[i] = 0.0f;
  }
  griddep_wait();
  // The first rows' scores are on their way while maxima and sums are joined: 3.7 us
  // -> 3.2 for one query x 1023, fp32; with four keys a thread their registers
  // cost what they gain.
  constexpr int EARLY = PER == 1 ? 4 : 0;
  const int64_t blks = kept_blocks(T);
  const float *x[PER];
  float early[EARLY + 1][PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) x[i] = T.kept + kept_at(unit, blks, on[i] ? slot0 + i * KTHREADS : 0, 0, L.rows);
#pragma unroll
  for (int r = 0; r < EARLY; ++r)
#pragma unroll
    for (int i = 0; i < PER; ++i) early[r][i] = r < L.rows ? x[i][16 * r] : 0.0f;
  const int64_t n = L.units * L.rows, first = static_cast<int64_t>(unit) * L.rows;
  for (int r = warp; r < L.rows; r += KTHREADS / 32) {
    float m = -INFINITY, l = 0.0f, inv;
    if (L.parts > 1) {
      for (int p = lane; p < L.parts; p += 32) {
        const float2 ml = T.ws_ml[p * n + first + r];
        const float to = fmaxf(m, ml.x), base = to == -INFINITY ? 0.0f : to;
        l = l * exp2f(m - base) + ml.y * exp2f(ml.x - base);
        m = to;
      }
      float top = m;
#pragma unroll
      for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      l *= exp2f(m - (top == -INFINITY ? 0.0f : top));
      m = top;
#pragma unroll
      for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
      inv = l > 0.0f ? 1.0f / l : (l == l ? 0.0f : l);
    } else {
      const float2 st = T.stats[first + r];
      m = st.x;
      inv = st.y;
    }
    if (lane == 0) {
      sm[r] = m;
      sl[r] = inv;  // 0: a row that saw nothing
      sc[r] = T.kept_c[first + r];
    }
  }
  __syncthreads();
  auto add = [&](int r, const float (&y)[PER]) {
    const float m = sm[r], inv = sl[r], c = sc[r];
    if (inv == 0.0f) return;
#pragma unroll
    for (int i = 0; i < PER; ++i) sum[i] += exp2f(fmaf(y[i], c, -m)) * inv;
  };
#pragma unroll
  for (int r = 0; r < EARLY; ++r)
    if (r < L.rows) add(r, early[r]);
#pragma unroll 4
  for (int r = EARLY; r < L.rows; ++r) {
    float y[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) y[i] = x[i][16 * r];
    add(r, y);
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int64_t slot = slot0 + i * KTHREADS, t = slot < ctx ? slot : T.S + slot - ctx;
    if (on[i]) out[t * P.os[2]] = fmaf(old[i], P.decay, sum[i]);
  }
}

template <int DC, int PER>
int launch_kept(const ScoreParams &P, cudaStream_t st) {
  const GenPlan L = tree_plan(P.t);
  const int64_t joins = L.parts > 1 ? (L.units * L.rows + KTHREADS / 32 - 1) / (KTHREADS / 32) : 0;
  const int64_t blocks = (16 * kept_blocks(P.t) + PER * KTHREADS - 1) / (PER * KTHREADS), all = joins + L.units * blocks;
  if (all > 0x7fffffff) return KV4_ERR_UNSUPPORTED;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(all));
  cfg.blockDim = dim3(KTHREADS);
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, score_kept<DC, PER>, P, L, static_cast<int>(joins), static_cast<int>(blocks)));
}

// four keys a thread once that still gives every SM a block
template <int DC>
int launch_kept_per(const ScoreParams &P, cudaStream_t st) {
  const bool many = P.t.B * P.t.Hkv * (16 * kept_blocks(P.t) / (4 * KTHREADS)) >= 148;
  return many ? launch_kept<DC, 4>(P, st) : launch_kept<DC, 1>(P, st);
}

int kept_run(const ScoreParams &P, cudaStream_t st) {
  if (P.t.d <= 64) return launch_kept_per<2>(P, st);
  if (P.t.d <= 128) return launch_kept_per<4>(P, st);
  if (P.t.d <= 256) return launch_kept_per<8>(P, st);
  return launch_kept_per<16>(P, st);
}

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

// kept scores and their factors, where few enough rows read a KV head
int64_t kept_bytes(const TreeParams &P) {
  const int64_t rows = static_cast<int64_t>(P.R) * P.nodes;
  if (rows > KROWS) return 0;
  return (P.B * P.Hkv * rows * (16 * kept_blocks(P) + 1) * 4 + 255) / 256 * 256;
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
  bool vec;        // rows that 16-byte loads can read
};

// order-preserving 32-bit key of a score: NaN lowest, -0 as +0
__device__ __forceinline__ uint32_t score_key(float x) {
  if (x != x) return 0u;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

constexpr int SEL = 1024;   // threads per block
constexpr int BINS = 2048;  // of one radix pass: 11, 11 and 10 bits

// exclusive prefix over the block of a pair of counts (a in the low half);
// `total` is the whole block's
__device__ __forceinline__ uint64_t block_prefix(uint64_t v, uint64_t *warps, uint64_t &total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint64_t inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t y = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += y;
  }
  __syncthreads();
  if (lane == 31) warps[warp] = inc;
  __syncthreads();
  uint64_t w = warps[lane], p = w;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t y = __shfl_up_sync(0xffffffffu, p, o);
    if (lane >= o) p += y;
  }
  total = __shfl_sync(0xffffffffu, p, 31);
  return __shfl_sync(0xffffffffu, p - w, warp) + inc - v;
}

// A cluster of `ranks` blocks per (sequence, KV head); each block takes `per`
// tokens in a row, each thread K of them, held as keys in registers.  Three
// passes find the threshold key (histograms in shared memory, added up over the
// cluster through distributed shared memory), then prefix sums give every kept
// token its place.  Scores are read once: 4 bytes a token, so that passes over
// registers and their barriers bound it (128 rows of 16384: 14.6 us; 8 rows of
// 1537: 6.4 us).
template <int K>
__global__ void __launch_bounds__(SEL, 1) evict_select(const __grid_constant__ EvictParams P, int ranks) {
  __shared__ uint32_t hist[2][BINS];  // by turns: a block may still read the other
  __shared__ uint64_t warps[32], s_count;
  __shared__ uint32_t s_bin, s_above;
  const int tid = threadIdx.x;
  const uint32_t rank = cluster_ctarank();
  const int unit = blockIdx.x / ranks, b = unit / P.Hkv, h = unit - b * P.Hkv;
  const float *mass = P.mass + b * P.ms[0] + h * P.ms[1];
  const int lo = P.sinks, hi = static_cast<int>(P.S) - P.recent;
  const int t0 = (static_cast<int>(rank) * SEL + tid) * K;
  uint32_t left = static_cast<uint32_t>(P.keep - P.sinks - P.recent);  // to be taken by score
  uint32_t key[K];
  bool mid[K];  // takes part in the ranking
  if (P.vec && t0 + K <= P.S) {
#pragma unroll
    for (int k = 0; k < K; k += 4) {
      const float4 v = *reinterpret_cast<const float4 *>(mass + t0 + k);
      key[k] = score_key(v.x);
      key[k + 1] = score_key(v.y);
      key[k + 2] = score_key(v.z);
      key[k + 3] = score_key(v.w);
    }
  } else {
#pragma unroll
    for (int k = 0; k < K; ++k) key[k] = t0 + k < P.S ? score_key(mass[(t0 + k) * P.ms[2]]) : 0u;
  }
#pragma unroll
  for (int k = 0; k < K; ++k) mid[k] = t0 + k >= lo && t0 + k < hi;

  uint32_t prefix = 0, known = 0;
  const bool ranked = left > 0;
  if (ranked) {
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
      const uint32_t mask = pass == 2 ? 1023u : 2047u;
      uint32_t *bins = hist[pass & 1];
      bins[tid] = 0u;
      bins[tid + SEL] = 0u;
      __syncthreads();
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (mid[k] && (key[k] & known) == prefix) atomicAdd(&bins[(key[k] >> shift) & mask], 1u);
      __syncthreads();
      // bins from the highest down: thread t holds two of them
      const int hb = BINS - 1 - 2 * tid;
      uint32_t c0 = bins[hb], c1 = bins[hb - 1];
      if (ranks > 1) {
        cluster_sync();
        const uint32_t at = smem_u32(bins + hb - 1);
#pragma unroll 1
        for (uint32_t r = 0; r < static_cast<uint32_t>(ranks); ++r) {
          if (r == rank) continue;
          const uint32_t a = dsmem_addr(at, r);
          c1 += static_cast<uint32_t>(ld_dsmem_s32(a));
          c0 += static_cast<uint32_t>(ld_dsmem_s32(a + 4));
        }
      }
      uint64_t total;
      const uint32_t above = static_cast<uint32_t>(block_prefix(c0 + c1, warps, total));
      if (above < left && left <= above + c0) {
        s_bin = hb;
        s_above = above;
      } else if (above + c0 < left && left <= above + c0 + c1) {
        s_bin = hb - 1;
        s_above = above + c0;
      }
      __syncthreads();
      prefix |= s_bin << shift;
      left -= s_above;
      known |= mask << shift;
    }
  }
  // now `left` of the keys equal to `prefix` are kept, the first ones
  uint32_t gt = 0, eq = 0;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const bool forced = t0 + k < P.S && !mid[k];
    if (forced || (ranked && mid[k] && key[k] > prefix)) gt |= 1u << k;
    else if (ranked && mid[k] && key[k] == prefix) eq |= 1u << k;
  }
  uint64_t total;
  uint64_t at = block_prefix(__popc(gt) | static_cast<uint64_t>(__popc(eq)) << 32, warps, total);
  if (ranks > 1) {
    if (tid == 0) s_count = total;
    cluster_sync();
    uint32_t g = 0, e = 0;
#pragma unroll 1
    for (uint32_t r = 0; r < rank; ++r) {
      const uint32_t a = dsmem_addr(smem_u32(&s_count), r);
      g += static_cast<uint32_t>(ld_dsmem_s32(a));
      e += static_cast<uint32_t>(ld_dsmem_s32(a + 4));
    }
    at += g | static_cast<uint64_t>(e) << 32;
    cluster_sync();  // nobody's shared memory goes while it is read
  }
  int32_t *out = P.index + static_cast<int64_t>(unit) * P.keep;
  uint32_t g = static_cast<uint32_t>(at), e = static_cast<uint32_t>(at >> 32);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if ((gt >> k & 1u) || ((eq >> k & 1u) && e < left)) out[g + min(e, left)] = t0 + k;
    g += gt >> k & 1u;
    e += eq >> k & 1u;
  }
}

// The same for rows longer than a cluster holds: a block per row reads the
// scores once for each of four eight-bit passes and once more to place them
// (2 rows of 300000: 446 us).
__global__ void __launch_bounds__(SEL) evict_select_long(const __grid_constant__ EvictParams P) {
  __shared__ int hist[256];
  __shared__ uint32_t s_prefix;
  __shared__ int s_left;
  __shared__ uint64_t warps[32];
  const int tid = threadIdx.x;
  const int64_t b = blockIdx.x / P.Hkv, h = blockIdx.x - b * P.Hkv;
  const float *mass = P.mass + b * P.ms[0] + h * P.ms[1];
  const int64_t lo = P.sinks, hi = P.S - P.recent;
  int left = P.keep - P.sinks - P.recent;  // still to be taken among equals
  const bool ranked = left > 0;
  uint32_t prefix = 0, known = 0;
  if (ranked) {
#pragma unroll 1
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
  int32_t *out = P.index + static_cast<int64_t>(blockIdx.x) * P.keep;
  uint64_t base = 0;  // kept for sure (low half) and equal to the threshold, so far
  for (int64_t c = 0; c < P.S; c += SEL) {
    const int64_t t = c + tid;
    bool gt = false, eq = false;
    if (t < P.S) {
      if (t < lo || t >= hi) gt = true;
      else if (ranked) {
        const uint32_t k = score_key(mass[t * P.ms[2]]);
        gt = k > prefix;
        eq = k == prefix;
      }
    }
    uint64_t total;
    const uint64_t at =
        base + block_prefix((gt ? 1u : 0u) | static_cast<uint64_t>(eq ? 1u : 0u) << 32, warps, total);
    const int g = static_cast<int>(at & 0xffffffffu), e = static_cast<int>(at >> 32);
    if (gt || (eq && e < left)) out[g + min(e, left)] = static_cast<int32_t>(t);
    base += total;
  }
}

template <int K>
int launch_select(const EvictParams &E, int64_t units, int ranks, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(units * ranks));
  cfg.blockDim = dim3(SEL);
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = static_cast<unsigned>(ranks);
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, evict_select<K>, E, ranks));
}

// Blocks of 1024 threads, up to 16 tokens a thread and 8 blocks a row.  Few
// rows: more blocks each, while 4 tokens a thread and an SM for each block remain
// (128 rows of 16K: one block a row takes 14.7 us, two 21.3, four 46).
int run_select(const EvictParams &E, int64_t units, cudaStream_t st) {
  int ranks = 1;
  while (ranks < 8 && E.S > static_cast<int64_t>(ranks) * SEL * 16) ranks *= 2;
  while (ranks < 8 && E.S > static_cast<int64_t>(ranks) * SEL * 4 && units * ranks * 2 <= 148)
    ranks *= 2;
  const int64_t per = (E.S + static_cast<int64_t>(ranks) * SEL - 1) / (static_cast<int64_t>(ranks) * SEL);
  if (per <= 4) return launch_select<4>(E, units, ranks, st);
  if (per <= 8) return launch_select<8>(E, units, ranks, st);
  if (per <= 16) return launch_select<16>(E, units, ranks, st);
  evict_select_long<<<static_cast<unsigned>(units), SEL, 0, st>>>(E);
  return cuda_status(cudaGetLastError());
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

// Any row sizes and alignments.
__global__ void __launch_bounds__(256) evict_gather(const __grid_constant__ GatherParams P) {
  __shared__ int32_t idx[GROWS];
  const int64_t unit = blockIdx.x / P.tiles, b = unit / P.Hkv, h = unit - b * P.Hkv;
  const int j0 = static_cast<int>(blockIdx.x - unit * P.tiles) * GROWS, n = min(GROWS, P.keep - j0);
  griddep_wait();  // the indices come from the kernel before
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

// Packed rows of CH 16-byte chunks and scale rows of one V each (the usual
// caches): every thread has all of its loads in flight before its first store.
// Memory bounds it: 128 rows, 4096 of 16384 tokens of 128 columns, 35.7 us; its
// scattered 8-byte scale rows move whole 32-byte sectors, 5.5 TB/s with those.
template <int CH, typename V>
__global__ void __launch_bounds__(256, 4) evict_gather_fast(const __grid_constant__ GatherParams P) {
  constexpr int ROWS = 256 / CH;  // per block
  const int64_t unit = blockIdx.x / P.tiles, b = unit / P.Hkv, h = unit - b * P.Hkv;
  const int j0 = static_cast<int>(blockIdx.x - unit * P.tiles) * ROWS;
  const int t = threadIdx.x, j = j0 + t / CH, c = t % CH;
  const bool in = j < P.keep;
  griddep_wait();
  const int64_t at = in ? P.index[unit * P.keep + j] : 0;
  uint4 w[2];
  V s{};
  uint32_t m = 0;
  const uint8_t *src[5];
#pragma unroll
  for (int k = 0; k < 5; ++k) src[k] = P.src[k] + b * P.ss[k][0] + h * P.ss[k][1] + at * P.ss[k][2];
  if (in) {
    w[0] = __ldg(reinterpret_cast<const uint4 *>(src[0]) + c);
    w[1] = __ldg(reinterpret_cast<const uint4 *>(src[2]) + c);
    if (c < 2) s = __ldg(reinterpret_cast<const V *>(c ? src[3] : src[1]));
    if (c == CH - 1) m = __ldg(reinterpret_cast<const uint32_t *>(src[4]));
  }
  uint8_t *dst[5];
#pragma unroll
  for (int k = 0; k < 5; ++k) dst[k] = P.dst[k] + b * P.ds[k][0] + h * P.ds[k][1] + j * P.ds[k][2];
  if (in) {
    reinterpret_cast<uint4 *>(dst[0])[c] = w[0];
    reinterpret_cast<uint4 *>(dst[2])[c] = w[1];
    if (c < 2) *reinterpret_cast<V *>(c ? dst[3] : dst[1]) = s;
    if (c == CH - 1) *reinterpret_cast<uint32_t *>(dst[4]) = m;
  }
}

template <class F>
int launch_gather(F kernel, GatherParams &G, int rows, int64_t units, cudaStream_t st) {
  const int64_t tiles = (G.keep + rows - 1) / rows;
  if (units * tiles > 0x7fffffff) return KV4_ERR_UNSUPPORTED;
  G.tiles = static_cast<int>(tiles);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(units * tiles));
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, kernel, G));
}

int run_gather(GatherParams &G, int64_t units, cudaStream_t st) {
  const bool packed = G.vec[0] == 16 && G.vec[2] == 16 && G.bytes[0] == G.bytes[2];
  const bool scales = G.bytes[1] == G.bytes[3] && G.vec[1] == G.bytes[1] && G.vec[3] == G.bytes[3];
  if (packed && scales) {
    if (G.bytes[0] == 64 && G.bytes[1] == 16) return launch_gather(evict_gather_fast<4, uint4>, G, 64, units, st);
    if (G.bytes[0] == 64 && G.bytes[1] == 8) return launch_gather(evict_gather_fast<4, uint2>, G, 64, units, st);
    if (G.bytes[0] == 64 && G.bytes[1] == 4) return launch_gather(evict_gather_fast<4, uint32_t>, G, 64, units, st);
    if (G.bytes[0] == 64 && G.bytes[1] == 2) return launch_gather(evict_gather_fast<4, uint16_t>, G, 64, units, st);
    if (G.bytes[0] == 32 && G.bytes[1] == 8) return launch_gather(evict_gather_fast<2, uint2>, G, 128, units, st);
    if (G.bytes[0] == 32 && G.bytes[1] == 4) return launch_gather(evict_gather_fast<2, uint32_t>, G, 128, units, st);
    if (G.bytes[0] == 32 && G.bytes[1] == 2) return launch_gather(evict_gather_fast<2, uint16_t>, G, 128, units, st);
  }
  return launch_gather(evict_gather, G, GROWS, units, st);
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
  return rc ? -rc : stats_bytes(P) + kept_bytes(P) + tree_workspace(P);
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
  if (P.t.B == 0 || P.t.Hkv == 0) return KV4_OK;
  // a call that leaves nothing but scores to scale
  const bool work = P.keys > 0 && P.t.nodes > 0, mma = tree_mma_takes(P.t), tc = !mma && tree_tc_takes(P.t);
  const bool keep = work && !tc && kept_bytes(P.t) > 0;
  const int64_t sb = stats_bytes(P.t), kb = keep ? kept_bytes(P.t) : 0;
  if (sb + kb > 0 && (!workspace || static_cast<int64_t>(workspace_bytes) < sb + kb)) return KV4_ERR_WORKSPACE;
  P.t.stats = static_cast<float2 *>(workspace);
  if (keep) {
    P.t.kept = reinterpret_cast<float *>(static_cast<char *>(workspace) + sb);
    P.t.kept_c = P.t.kept + P.t.B * P.t.Hkv * P.t.R * P.t.nodes * 16 * kept_blocks(P.t);
  }
  rc = tree_run(P.t, static_cast<char *>(workspace) + sb + kb,
                static_cast<int64_t>(workspace_bytes) - sb - kb, st);
  if (rc) return rc;
  if (keep) return kept_run(P, st);
  if (work && mma) return score_mma_run(P, st);
  if (work && tc) return score_tc_run(P, st);
  return score_run(P, st);
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
    G.vec[k] = copy_width(G.dst[k], G.src[k], G.bytes[k], G.ds[k], G.ss[k]);
  }
  if (recent < 0 || sinks < 0 || keep < 0 || recent + sinks > keep || keep > S)
    return KV4_ERR_INVALID;
  if (S >= (int64_t(1) << 30)) return KV4_ERR_UNSUPPORTED;
  if (B == 0 || Hkv == 0 || keep == 0) return KV4_OK;
  if (!index) return KV4_ERR_INVALID;
  if (B * Hkv > (int64_t(1) << 24)) return KV4_ERR_UNSUPPORTED;
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
  E.vec = (reinterpret_cast<uintptr_t>(E.mass) & 15u) == 0 && E.ms[2] == 1 && E.ms[0] % 4 == 0 &&
          E.ms[1] % 4 == 0;
  const int rc = run_select(E, B * Hkv, st);
  if (rc) return rc;
  G.index = index;
  G.Hkv = static_cast<int>(Hkv);
  G.keep = static_cast<int>(keep);
  return run_gather(G, B * Hkv, st);
}
