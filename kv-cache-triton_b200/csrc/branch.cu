// Tree attention over the INT4 cache, and the commit of an accepted path.
//
// Speculative decoding drafts a tree of N nodes per sequence.  Their K/V rows
// are quantized into a draft buffer; verification is one attention call in
// which node i (of every q head) sees the whole committed context and the
// drafted nodes that a boolean mask lets it see (its ancestors and itself):
//
//   x[t]  = q . K[t] * sm_scale        t < len_b, and drafted rows j with mask[b, i, j]
//   out   = sum_t softmax(x)[t] V[t]   (0 where the row sees nothing)
//
// Rows that share a KV head share one read of it: row r of a (sequence, KV
// head) unit is node r / R of q head kvh * R + r % R, R = Hq / Hkv.
//
// tree_generic: any head size up to 512, group size, strides and float types,
// in fp32 FFMA.  A warp owns RW rows and a range of keys: 32 keys at a time it
// dequantizes K into its own shared memory (lane = key for the scores), then V
// over it (lane = column for the output), with the running maximum and sum of
// the softmax per row.  A block's warps meet at the end, blocks of one unit in
// tree_merge through the workspace.  16-bit types take branch_tc.cu's
// and branch_mma.cu's kernels where the layout allows.
// Bound by instructions: 6000 for 8 rows x 32 keys x 128 columns, a third of them
// the products, at two warps a scheduler (shared memory holds no more tiles).
// Measured, fp32: 64 rows x 2016 keys of 128 columns in 16 units 94 us with the join
// (11 TFLOP/s); 12 rows x 789 keys of 64 columns in 24 units 15.6 us and 3 to join,
// where a warp has one tile and its chain counts.
#include <algorithm>

#include "merge.cuh"

namespace kv4 {

// device error word of this file (folded into kv4_device_error)
__device__ int g_branch_error = 0;

namespace {

template <int RW>
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

template <int DC, int RW>
__global__ void __launch_bounds__(128, 1) tree_generic(const TreeParams P, const GenPlan L) {
  extern __shared__ __align__(16) float gsm[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int area = 32 * L.ld + RW * L.ld + 32 * RW;  // floats of a warp
  float *sT = gsm + warp * area;                     // K or V tile
  float *sQ = sT + 32 * L.ld, *sP = sQ + RW * L.ld;  // rows of q; weights [key][RW]
  const int part = static_cast<int>(blockIdx.x % L.parts);
  const int64_t ur = blockIdx.x / L.parts;
  const int rt = static_cast<int>(ur % L.row_tiles);
  const int64_t unit = ur / L.row_tiles, b = unit / P.Hkv;
  const int kvh = static_cast<int>(unit - b * P.Hkv);
  const int64_t len = context_len(P, b, part == 0 && rt == 0 && threadIdx.x == 0 ? &g_branch_error : nullptr);
  const int64_t total = len + P.ndraft, tiles = (total + 31) >> 5;
  const int64_t ranges = static_cast<int64_t>(L.parts) * L.warps, per = (tiles + ranges - 1) / ranges;
  const int64_t k0 = (part * L.warps + warp) * per * 32, k1 = min(total, k0 + per * 32);
  const int r0 = rt * RW, d8 = (P.d + 7) >> 3;

  warp_query<RW>(P, b, kvh, r0, L.rows, sQ, L.ld, lane);
  float m[RW], l[RW], acc[RW][DC];
#pragma unroll
  for (int r = 0; r < RW; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.0f;
#pragma unroll
    for (int k = 0; k < DC; ++k) acc[r][k] = 0.0f;
  }

  // K's tile, then V's over it, by the same code: two copies of it miss the
  // instruction cache
  int64_t t0 = k0;
#pragma unroll 1
  for (bool is_v = false; t0 < k1; is_v = !is_v) {
    __syncwarp();
    warp_dequant_tile(P, is_v, b, kvh, len, t0, k1, sT, L.ld, lane);
    __syncwarp();
    if (is_v) {
      // a drafted row may hold anything where a node does not see it: there a
      // weight of zero leaves it out instead of multiplying it
      const bool guard = t0 + 32 > len;
#pragma unroll 4
      for (int j = 0; j < 32; ++j) {
        float v[DC], p[RW];
#pragma unroll
        for (int k = 0; k < DC; ++k) v[k] = lane + 32 * k < 8 * d8 ? sT[j * L.ld + lane + 32 * k] : 0.0f;
#pragma unroll
        for (int r = 0; r < RW; ++r) p[r] = sP[j * RW + r];
#pragma unroll
        for (int r = 0; r < RW; ++r) {
          if (guard && p[r] == 0.0f) continue;
#pragma unroll
          for (int k = 0; k < DC; ++k) acc[r][k] = fmaf(p[r], v[k], acc[r][k]);
        }
      }
      t0 += 32;
      continue;
    }
    float4 part4[RW];  // four sums per score: a quarter of the roundings in a row
#pragma unroll
    for (int r = 0; r < RW; ++r) part4[r] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 2
    for (int c = 0; c < 2 * d8; ++c) {
      const float4 k4 = *reinterpret_cast<const float4 *>(sT + lane * L.ld + 4 * c);
#pragma unroll
      for (int r = 0; r < RW; ++r) fma4(part4[r], *reinterpret_cast<const float4 *>(sQ + r * L.ld + 4 * c), k4);
    }
    float s[RW];
#pragma unroll
    for (int r = 0; r < RW; ++r) s[r] = sum4(part4[r]);
    const int64_t t = t0 + lane;
#pragma unroll
    for (int r = 0; r < RW; ++r) {
      const int row = r0 + r;
      bool see = t < k1 && row < L.rows;
      if (see && t >= len) see = draft_visible(P, b, row / P.R, static_cast<int>(t - len));
      const float x = see ? s[r] * P.scale_log2 : -INFINITY;
      if (P.kept && t < k1 && row < L.rows) {
        const int64_t slot = t < len ? t : ((len + 15) & ~int64_t(15)) + t - len;
        P.kept[kept_at(unit, kept_blocks(P), slot, row, L.rows)] = see ? s[r] : -INFINITY;
      }
      const float mn = fmaxf(m[r], warp_max<RW>(x));
      const float base = mn == -INFINITY ? 0.0f : mn;
      const float a = exp2f(m[r] - base), p = exp2f(x - base);
      m[r] = mn;
      l[r] = l[r] * a + p;  // this lane's keys; the lanes meet at the end
#pragma unroll
      for (int k = 0; k < DC; ++k) acc[r][k] *= a;
      sP[lane * RW + r] = p;
    }
  }
  // ---- the block's warps meet: outputs where the tiles were, (m, l) for the weights ----
  __syncwarp();
#pragma unroll
  for (int r = 0; r < RW; ++r) {
#pragma unroll
    for (int o = 16; o; o >>= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], o);
#pragma unroll
    for (int k = 0; k < DC; ++k)
      if (lane + 32 * k < P.d) sT[r * L.ld + lane + 32 * k] = acc[r][k];
    if (lane == 0) *reinterpret_cast<float2 *>(sP + 2 * r) = make_float2(m[r], l[r]);
  }
  __syncthreads();
#pragma unroll 1
  for (int r = warp; r < RW && r0 + r < L.rows; r += L.warps) {
    const int row = r0 + r;
    const float *o = gsm + r * L.ld, *ml = gsm + 32 * L.ld + RW * L.ld + 2 * r;
    float M = -INFINITY, sum = 0.0f, v[DC];
#pragma unroll 1
    for (int w = 0; w < L.warps; ++w) M = fmaxf(M, ml[w * area]);
    const float base = M == -INFINITY ? 0.0f : M;
#pragma unroll
    for (int k = 0; k < DC; ++k) v[k] = 0.0f;
#pragma unroll 1
    for (int w = 0; w < L.warps; ++w) {
      const float f = exp2f(ml[w * area] - base);
      sum = fmaf(ml[w * area + 1], f, sum);
#pragma unroll
      for (int k = 0; k < DC; ++k)
        if (lane + 32 * k < P.d) v[k] = fmaf(o[w * area + lane + 32 * k], f, v[k]);
    }
    const int64_t at = unit * L.rows + row;
    if (P.kept && part == 0 && lane == 0) P.kept_c[at] = P.scale_log2;
    if (L.parts == 1) {
      const int i = row / P.R, h = kvh * P.R + row - i * P.R;
      const float inv = sum > 0.0f ? 1.0f / sum : (sum == sum ? 0.0f : sum);
#pragma unroll
      for (int k = 0; k < DC; ++k)
        if (lane + 32 * k < P.d)
          store_from_f32(P.out, P.q_dtype,
                         b * P.os[0] + h * P.os[1] + i * P.os[2] + (lane + 32 * k) * P.os[3],
                         v[k] * inv);
      if (lane == 0) {
        if (P.stats) P.stats[at] = make_float2(M, inv);
        if (P.lse)
          P.lse[b * P.ls[0] + h * P.ls[1] + i * P.ls[2]] =
              sum == 0.0f ? -INFINITY : (M + log2f(sum)) * kBrLn2;
      }
    } else {
      const int64_t slot = static_cast<int64_t>(part) * L.units * L.rows + at;
#pragma unroll
      for (int k = 0; k < DC; ++k)
        if (lane + 32 * k < P.d) P.ws_o[slot * P.d + lane + 32 * k] = v[k];
      if (lane == 0) P.ws_ml[slot] = make_float2(M, sum);
    }
  }
}

template <int DC>
__global__ void __launch_bounds__(128, 4) tree_merge(const __grid_constant__ TreeParams P, const GenPlan L) {
  const int64_t at = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
  griddep_wait();
  if (at < L.units * L.rows) merge_row<DC>(P, L, at, threadIdx.x & 31);
}

constexpr int kSms = 148;

// Rows a warp holds: eight share one dequantized tile, fewer where there are no
// more (measured before the block's warps met: 4 rows x 4000 keys x 8 heads of 128,
// batch 4, fp32, 63 us instead of 76; four for 12 rows x 777 26 instead of 23).
int rows_per_warp(int rows) { return rows <= 2 ? 2 : rows <= 4 ? 4 : 8; }

GenPlan gen_plan(const TreeParams &P) {
  GenPlan L{};
  L.rows = P.R * P.nodes;
  const int rw = rows_per_warp(L.rows);
  L.row_tiles = (L.rows + rw - 1) / rw;
  L.units = P.B * P.Hkv;
  L.ld = row_ld(P.d);
  const size_t per_warp = sizeof(float) * (32 * L.ld + rw * L.ld + 32 * rw);
  L.warps = static_cast<int>(std::max<size_t>(1, std::min<size_t>(4, 100 * 1024 / per_warp)));
  L.smem = per_warp * L.warps;
  // blocks of at least 32 keys a warp, as many as the SMs take at once (a block
  // more on a few of them runs alone at the end: 64 rows x 2000 x 8 heads of 128,
  // batch 2: 153 us with 320 blocks of four warps, 94 with 256)
  const int64_t tiles = (P.S + P.ndraft + 31) / 32, have = L.units * L.row_tiles;
  const int64_t room = kSms * std::min<int64_t>(3, 200 * 1024 / L.smem);
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>(room / have, 64)) * L.warps;
  const int64_t per = std::max<int64_t>(1, (tiles + want - 1) / want) * L.warps;
  L.parts = static_cast<int>(std::max<int64_t>(1, (tiles + per - 1) / per));
  return L;
}

int64_t gen_workspace(const TreeParams &P, const GenPlan &L) {
  if (L.parts == 1) return 0;
  return L.parts * L.units * L.rows * (static_cast<int64_t>(P.d) * 4 + 8);
}

template <int DC>
int launch_merge(const TreeParams &P, const GenPlan &L, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>((L.units * L.rows + 3) / 4));
  cfg.blockDim = dim3(128);
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, tree_merge<DC>, P, L));
}

template <int DC, int RW>
int launch_gen(const TreeParams &P, const GenPlan &L, cudaStream_t st) {
  const int64_t blocks = L.units * L.row_tiles * L.parts;
  if (blocks > 0x7fffffff) return KV4_ERR_UNSUPPORTED;
  if (L.smem > 48 * 1024) {
    const int rc = cuda_status(cudaFuncSetAttribute(
        tree_generic<DC, RW>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024));
    if (rc) return rc;
  }
  tree_generic<DC, RW><<<static_cast<unsigned>(blocks), 32 * L.warps, L.smem, st>>>(P, L);
  const int rc = cuda_status(cudaGetLastError());
  if (rc || L.parts == 1 || P.kept) return rc;  // score_kept joins the parts itself
  return launch_merge<DC>(P, L, st);
}

template <int DC>
int launch_gen_rw(const TreeParams &P, const GenPlan &L, cudaStream_t st) {
  switch (rows_per_warp(L.rows)) {
    case 2: return launch_gen<DC, 2>(P, L, st);
    case 4: return launch_gen<DC, 4>(P, L, st);
    default: return launch_gen<DC, 8>(P, L, st);
  }
}

bool is_float(int dt) { return dt == KV4_F32 || dt == KV4_F16 || dt == KV4_BF16; }

// strides of one K/V source with its shapes checked: rows [B, Hkv, T, ...]
int fill_source(RowSource &S, const kv4_tensor *const t[4], int64_t B, int64_t Hkv, int64_t T,
                int64_t pw, int64_t ng, int s_dtype) {
  for (int k = 0; k < 4; ++k) {
    const kv4_tensor *x = t[k];
    if (!x) return KV4_ERR_INVALID;
    const bool scales = k & 1;
    if (scales ? x->dtype != s_dtype : x->dtype != KV4_U8) return KV4_ERR_DTYPE;
    if (x->shape[0] != B || x->shape[1] != Hkv || x->shape[2] != T ||
        x->shape[3] < (scales ? ng : pw))
      return KV4_ERR_SHAPE;
    if (x->shape[3] != t[k & 1]->shape[3]) return KV4_ERR_SHAPE;
    int64_t *st = k == 0 ? S.kps : k == 1 ? S.kss : k == 2 ? S.vps : S.vss;
    for (int i = 0; i < 4; ++i) st[i] = x->stride[i];
    if (B > 0 && T > 0 && !x->data) return KV4_ERR_INVALID;
  }
  S.kp = static_cast<const uint8_t *>(t[0]->data);
  S.ks = t[1]->data;
  S.vp = static_cast<const uint8_t *>(t[2]->data);
  S.vs = t[3]->data;
  return KV4_OK;
}

}  // namespace

int tree_fill(TreeParams &P, const kv4_tensor *q, const kv4_tensor *const cache[4],
              const kv4_tensor *const draft[4], const kv4_tensor *out, int G, float sm_scale) {
  if (!q || !out || !cache[0] || !cache[1] || G <= 0) return KV4_ERR_INVALID;
  if (!is_float(q->dtype) || out->dtype != q->dtype || !is_float(cache[1]->dtype))
    return KV4_ERR_DTYPE;
  const int64_t B = q->shape[0], Hq = q->shape[1], N = q->shape[2], d = q->shape[3];
  const int64_t Hkv = cache[0]->shape[1], S = cache[0]->shape[2];
  for (int i = 0; i < 4; ++i)
    if (out->shape[i] != q->shape[i]) return KV4_ERR_SHAPE;
  if (Hkv <= 0 || Hq <= 0 || Hq % Hkv) return KV4_ERR_INVALID;
  if (B < 0 || N < 0 || d <= 0) return KV4_ERR_SHAPE;
  if (d > 512 || B * Hkv > (int64_t(1) << 24) || S >= (int64_t(1) << 30) ||
      N * (Hq / Hkv) >= (int64_t(1) << 24))
    return KV4_ERR_UNSUPPORTED;
  const int64_t ng = (d + G - 1) / G, pw = ng * ((G + 1) / 2);
  P.s_dtype = cache[1]->dtype;
  int rc = fill_source(P.cache, cache, B, Hkv, S, pw, ng, P.s_dtype);
  if (rc) return rc;
  P.ndraft = 0;
  if (draft && draft[0]) {
    const int64_t nd = draft[0]->shape[2];
    if (nd >= (int64_t(1) << 24)) return KV4_ERR_UNSUPPORTED;
    rc = fill_source(P.draft, draft, B, Hkv, nd, pw, ng, P.s_dtype);
    if (rc) return rc;
    P.ndraft = static_cast<int>(nd);
  }
  P.q = q->data;
  P.out = out->data;
  P.q_dtype = q->dtype;
  for (int i = 0; i < 4; ++i) {
    P.qs[i] = q->stride[i];
    P.os[i] = out->stride[i];
  }
  P.B = B;
  P.Hkv = static_cast<int>(Hkv);
  P.R = static_cast<int>(Hq / Hkv);
  P.nodes = static_cast<int>(N);
  P.d = static_cast<int>(d);
  P.G = G;
  P.S = S;
  P.words = G < 8 || (G & (G - 1)) || d % 8 ? 0 : d % 32 ? 4 : 16;
  for (const RowSource *src : {&P.cache, &P.draft}) {
    if (src == &P.draft && P.ndraft == 0) continue;
    uint64_t bits = reinterpret_cast<uintptr_t>(src->kp) | reinterpret_cast<uintptr_t>(src->vp);
    for (int i = 0; i < 3; ++i) bits |= static_cast<uint64_t>(src->kps[i] | src->vps[i]);
    if ((bits & 3u) || src->kps[3] != 1 || src->vps[3] != 1) P.words = 0;
    if (bits & 15u) P.words = std::min(P.words, 4);
  }
  P.scale_log2 = (sm_scale > 0.0f ? sm_scale : 1.0f / sqrtf(static_cast<float>(d))) * kBrLog2e;
  return KV4_OK;
}

int tree_mma_parts(const TreeParams &P);   // branch_mma.cu
bool tree_mma_joins(const TreeParams &P);  // within the kernel
int tree_mma_run(const TreeParams &P, cudaStream_t st);
int branch_mma_take_device_error(int *v);
int64_t tree_tc_workspace(const TreeParams &P);  // branch_tc.cu
int tree_tc_run(TreeParams &P, void *workspace, int64_t bytes, cudaStream_t st);
int branch_tc_take_device_error(int *v);
int trim_tc_take_device_error(int *v);  // trim_tc.cu

namespace {
// what tree_merge has to know of a run of branch_mma.cu's kernel
GenPlan mma_merge_plan(const TreeParams &P) {
  GenPlan L{};
  L.units = P.B * P.Hkv;
  L.rows = P.R * P.nodes;
  L.parts = tree_mma_parts(P);
  return L;
}
}  // namespace

GenPlan tree_plan(const TreeParams &P) { return tree_mma_takes(P) ? mma_merge_plan(P) : gen_plan(P); }

// The largest that any output can ask for: where q allows the other kernels, an
// output with other strides or at another address may still leave the call to
// tree_generic.
int64_t tree_workspace(const TreeParams &P) {
  if (P.B == 0 || P.nodes == 0) return 0;  // nothing to cut into parts
  int64_t most = gen_workspace(P, gen_plan(P));
  if (tree_mma_takes(P)) most = std::max(most, gen_workspace(P, mma_merge_plan(P)));
  else if (tree_tc_takes(P)) most = std::max(most, tree_tc_workspace(P));
  return most;
}

int tree_run(TreeParams &P, void *workspace, int64_t bytes, cudaStream_t st) {
  if (P.B == 0 || P.nodes == 0) return KV4_OK;
  const bool mma = tree_mma_takes(P);
  if (!mma && tree_tc_takes(P)) return tree_tc_run(P, workspace, bytes, st);
  const GenPlan L = tree_plan(P);
  if (gen_workspace(P, L) > 0) {
    if (!workspace || bytes < gen_workspace(P, L)) return KV4_ERR_WORKSPACE;
    const int64_t n = L.parts * L.units * L.rows;
    P.ws_ml = static_cast<float2 *>(workspace);
    P.ws_o = static_cast<float *>(workspace) + 2 * n;
  }
  if (mma) {
    const int rc = tree_mma_run(P, st);
    if (rc || L.parts == 1 || P.kept || tree_mma_joins(P)) return rc;
    return P.d == 64 ? launch_merge<2>(P, L, st) : launch_merge<4>(P, L, st);
  }
  if (P.d <= 64) return launch_gen_rw<2>(P, L, st);
  if (P.d <= 128) return launch_gen_rw<4>(P, L, st);
  if (P.d <= 256) return launch_gen_rw<8>(P, L, st);
  return launch_gen_rw<16>(P, L, st);
}

// ---------------------------------------------------------------------------
// commit: the accepted rows of the draft buffer move behind the context
// ---------------------------------------------------------------------------
namespace {

struct CommitParams {
  uint8_t *dst[4];
  const uint8_t *src[4];
  int64_t ds[4][3], ss[4][3];  // batch, head, token strides (bytes)
  int bytes[4], vec[4];        // of a row; of one copy
  const int32_t *path, *accepted, *lens;
  int32_t *lens_out;
  int64_t path_stride;
  int64_t cap;
  int B, Hkv, nodes, width;
};

constexpr int CTHREADS = 64;  // per tensor
constexpr int CPATH = 256;    // path entries held at a time

template <typename V>
__device__ __forceinline__ void move_rows(uint8_t *dst, const uint8_t *src, int64_t ds, int64_t ss,
                                          int bytes, const int32_t *path, int n, int nodes, int t) {
  const int per = bytes / static_cast<int>(sizeof(V));
  for (int e0 = t; e0 < n * per; e0 += 4 * CTHREADS) {
    V v[4];
    bool in[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {  // four in flight
      const int e = e0 + u * CTHREADS, j = e / per, node = e < n * per ? path[j] : -1;
      in[u] = node >= 0 && node < nodes;
      if (in[u]) v[u] = __ldg(reinterpret_cast<const V *>(src + node * ss) + (e - j * per));
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int e = e0 + u * CTHREADS, j = e / per;
      if (in[u]) reinterpret_cast<V *>(dst + j * ds)[e - j * per] = v[u];
    }
  }
}

// A block per (sequence, KV head), 64 threads for each of the four tensors; the
// block of head 0 writes the new length.  Such a call moves little: what it
// costs is two rounds of memory latency (lengths and path, then the rows).
// Measured, 8 heads of 128 columns: 2.5 us for one sequence, 3.0 for 32.
__global__ void __launch_bounds__(4 * CTHREADS, 2) commit_rows(const __grid_constant__ CommitParams P) {
  __shared__ int32_t path[CPATH];
  const int b = blockIdx.x / P.Hkv, h = blockIdx.x - b * P.Hkv;
  const int k = threadIdx.x / CTHREADS, t = threadIdx.x - k * CTHREADS;
  // read once: with one head lens_out may be lens, and is written below
  const int64_t len = P.lens[b], n = P.accepted[b];
  const bool fits = len >= 0 && n >= 0 && n <= P.width && len + n <= P.cap;
  for (int j0 = 0; j0 == 0 || j0 < P.width; j0 += CPATH) {
    const int j = j0 + static_cast<int>(threadIdx.x);
    if (j < P.width) path[threadIdx.x] = P.path[b * P.path_stride + j];
    __syncthreads();
    if (j0 == 0 && h == 0 && threadIdx.x == 0) {
      // a sequence that does not fit is left as it was, and reported
      if (!fits) atomicOr(&g_branch_error, DEV_ERR_BAD_LENGTH);
      P.lens_out[b] = static_cast<int32_t>(fits ? len + n : len);
    }
    if (!fits) return;
    const int m = min(CPATH, static_cast<int>(n) - j0);
    if (static_cast<int>(threadIdx.x) < m &&
        (path[threadIdx.x] < 0 || path[threadIdx.x] >= P.nodes))
      atomicOr(&g_branch_error, DEV_ERR_BAD_LENGTH);
    uint8_t *dst = P.dst[k] + b * P.ds[k][0] + h * P.ds[k][1] + (len + j0) * P.ds[k][2];
    const uint8_t *src = P.src[k] + b * P.ss[k][0] + h * P.ss[k][1];
    switch (P.vec[k]) {
      case 16: move_rows<uint4>(dst, src, P.ds[k][2], P.ss[k][2], P.bytes[k], path, m, P.nodes, t); break;
      case 8: move_rows<uint2>(dst, src, P.ds[k][2], P.ss[k][2], P.bytes[k], path, m, P.nodes, t); break;
      case 4: move_rows<uint32_t>(dst, src, P.ds[k][2], P.ss[k][2], P.bytes[k], path, m, P.nodes, t); break;
      case 2: move_rows<uint16_t>(dst, src, P.ds[k][2], P.ss[k][2], P.bytes[k], path, m, P.nodes, t); break;
      default: move_rows<uint8_t>(dst, src, P.ds[k][2], P.ss[k][2], P.bytes[k], path, m, P.nodes, t); break;
    }
    __syncthreads();
  }
}

}  // namespace

// read-and-clear of this file's device error word
int branch_take_device_error(int *v) {
  int zero = 0, t = 0;
  int rc = cuda_status(cudaMemcpyFromSymbol(v, g_branch_error, sizeof(int)));
  if (rc) return rc;
  rc = cuda_status(cudaMemcpyToSymbol(g_branch_error, &zero, sizeof(int)));
  if (rc) return rc;
  rc = branch_tc_take_device_error(&t);
  *v |= t;
  t = 0;
  if (!rc) rc = trim_tc_take_device_error(&t);
  *v |= t;
  t = 0;
  if (!rc) rc = branch_mma_take_device_error(&t);
  *v |= t;
  return rc;
}

namespace {

int tree_args(TreeParams &P, const kv4_tensor *q, const kv4_tensor *const cache[4],
              const kv4_tensor *const draft[4], const kv4_tensor *mask, const int32_t *lens,
              const kv4_tensor *out, const kv4_tensor *lse, int group_size, float sm_scale) {
  for (int k = 0; k < 4; ++k)
    if (!cache[k] || !draft[k]) return KV4_ERR_INVALID;
  int rc = tree_fill(P, q, cache, draft, out, group_size, sm_scale);
  if (rc) return rc;
  if (!mask) return KV4_ERR_INVALID;
  if (mask->dtype != KV4_U8) return KV4_ERR_DTYPE;
  if (mask->shape[0] != 1 || (mask->shape[1] != 1 && mask->shape[1] != P.B) ||
      mask->shape[2] != P.nodes || mask->shape[3] != P.ndraft)
    return KV4_ERR_SHAPE;
  P.mask = static_cast<const uint8_t *>(mask->data);
  P.ms[0] = mask->shape[1] == 1 ? 0 : mask->stride[1];
  P.ms[1] = mask->stride[2];
  P.ms[2] = mask->stride[3];
  P.lens = lens;
  if (lse) {
    if (lse->dtype != KV4_F32) return KV4_ERR_DTYPE;
    for (int i = 0; i < 3; ++i) {
      if (lse->shape[i] != q->shape[i]) return KV4_ERR_SHAPE;
      P.ls[i] = lse->stride[i];
    }
    P.lse = static_cast<float *>(lse->data);
  }
  return KV4_OK;
}

}  // namespace
}  // namespace kv4

using namespace kv4;

extern "C" int64_t kv4_tree_workspace(const kv4_tensor *q, const kv4_tensor *k_packed,
                                      const kv4_tensor *k_scales, const kv4_tensor *v_packed,
                                      const kv4_tensor *v_scales, const kv4_tensor *dk_packed,
                                      const kv4_tensor *dk_scales, const kv4_tensor *dv_packed,
                                      const kv4_tensor *dv_scales, int group_size) {
  const kv4_tensor *cache[4] = {k_packed, k_scales, v_packed, v_scales};
  const kv4_tensor *draft[4] = {dk_packed, dk_scales, dv_packed, dv_scales};
  TreeParams P{};
  const int rc = tree_fill(P, q, cache, draft, q, group_size, 0.0f);
  return rc ? -rc : tree_workspace(P);
}

extern "C" int kv4_tree_attention(const kv4_tensor *q, const kv4_tensor *k_packed,
                                  const kv4_tensor *k_scales, const kv4_tensor *v_packed,
                                  const kv4_tensor *v_scales, const kv4_tensor *dk_packed,
                                  const kv4_tensor *dk_scales, const kv4_tensor *dv_packed,
                                  const kv4_tensor *dv_scales, const kv4_tensor *mask,
                                  const int32_t *context_lens, const kv4_tensor *out,
                                  const kv4_tensor *lse, int group_size, float sm_scale,
                                  void *workspace, size_t workspace_bytes, void *stream) {
  const kv4_tensor *cache[4] = {k_packed, k_scales, v_packed, v_scales};
  const kv4_tensor *draft[4] = {dk_packed, dk_scales, dv_packed, dv_scales};
  TreeParams P{};
  const int rc = tree_args(P, q, cache, draft, mask, context_lens, out, lse, group_size, sm_scale);
  if (rc) return rc;
  return tree_run(P, workspace, static_cast<int64_t>(workspace_bytes),
                  static_cast<cudaStream_t>(stream));
}

extern "C" int kv4_commit_rows(const kv4_tensor *k_packed, const kv4_tensor *k_scales,
                               const kv4_tensor *v_packed, const kv4_tensor *v_scales,
                               const kv4_tensor *dk_packed, const kv4_tensor *dk_scales,
                               const kv4_tensor *dv_packed, const kv4_tensor *dv_scales,
                               const int32_t *path, int64_t path_stride, int64_t path_width,
                               const int32_t *accepted, const int32_t *context_lens,
                               int32_t *lens_out, void *stream) {
  const kv4_tensor *dst[4] = {k_packed, k_scales, v_packed, v_scales};
  const kv4_tensor *src[4] = {dk_packed, dk_scales, dv_packed, dv_scales};
  CommitParams P{};
  for (int k = 0; k < 4; ++k) {
    const kv4_tensor *c = dst[k], *s = src[k];
    if (!c || !s) return KV4_ERR_INVALID;
    if ((k & 1) ? !is_float(c->dtype) : c->dtype != KV4_U8) return KV4_ERR_DTYPE;
    if (c->dtype != s->dtype) return KV4_ERR_DTYPE;
    if (c->shape[0] != s->shape[0] || c->shape[1] != s->shape[1] || c->shape[3] != s->shape[3] ||
        c->shape[0] != dst[0]->shape[0] || c->shape[1] != dst[0]->shape[1] ||
        c->shape[2] != dst[0]->shape[2] || s->shape[2] != src[0]->shape[2])
      return KV4_ERR_SHAPE;
    if ((c->shape[3] > 1 && c->stride[3] != 1) || (s->shape[3] > 1 && s->stride[3] != 1))
      return KV4_ERR_LAYOUT;
    const int e = dtype_size(c->dtype);
    P.bytes[k] = static_cast<int>(c->shape[3] * e);
    P.dst[k] = static_cast<uint8_t *>(c->data);
    P.src[k] = static_cast<const uint8_t *>(s->data);
    for (int i = 0; i < 3; ++i) {
      P.ds[k][i] = c->stride[i] * e;
      P.ss[k][i] = s->stride[i] * e;
    }
    P.vec[k] = copy_width(P.dst[k], P.src[k], P.bytes[k], P.ds[k], P.ss[k]);
  }
  if (!path || !accepted || !context_lens || !lens_out || path_width < 0) return KV4_ERR_INVALID;
  const int64_t B = dst[0]->shape[0], Hkv = dst[0]->shape[1], n = src[0]->shape[2];
  if (B == 0 || Hkv == 0) return KV4_OK;
  if (B * Hkv > 0x7fffffff || n >= (int64_t(1) << 30) || path_width >= (int64_t(1) << 30))
    return KV4_ERR_UNSUPPORTED;
  P.path = path;
  P.path_stride = path_stride;
  P.accepted = accepted;
  P.lens = context_lens;
  P.lens_out = lens_out;
  P.cap = dst[0]->shape[2];
  P.B = static_cast<int>(B);
  P.Hkv = static_cast<int>(Hkv);
  P.nodes = static_cast<int>(n);
  P.width = static_cast<int>(path_width);
  commit_rows<<<static_cast<unsigned>(B * Hkv), 4 * CTHREADS, 0, static_cast<cudaStream_t>(stream)>>>(P);
  return cuda_status(cudaGetLastError());
}
