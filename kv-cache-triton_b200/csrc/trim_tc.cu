// The second reading of the keys in scored attention, on the tensor cores, for
// what tree_tc takes (bf16 queries and scales, head sizes 64 and 128).
//
//   score'[t] = decay * score[t] + sum over rows r of 2^(c_r s_rt - m_r) / l_r
//
// with s = K q^T: keys are the M dimension here, so a thread owns one key, reads
// its scores of up to 128 rows from tensor memory and sums their weights in a
// register; c_r, m_r and 1 / l_r come from shared memory, the same for all
// threads.  More rows are taken 128 at a time, each pass over the CTA's keys
// adding to what the last one wrote (same CTA, same order every time).
//
// Twelve warps and one that issues, two CTAs per SM: warps 0-3 and 4-7 sum the
// weights of every other tile (one such group alone took 4500 cycles a tile,
// twice what the rest needs), 8-11 dequantize key tiles (loaded two tiles ahead
// into registers) into two buffers.  All (unit, tile) pairs are cut evenly over
// the CTAs.  Measured, 256 rows x 16384 keys x 8 heads, batch 2: 47.3 us, where the
// exponentials take 15.7 (16 a cycle and SM) and the products 5; what is left is
// waiting between the three roles, and a pass of its own for the second 128 rows.
#include <algorithm>

#include "tc_rows.cuh"

namespace kv4 {

// device error word of this file (folded into kv4_device_error)
__device__ int g_trim_error_tc = 0;

namespace {

constexpr int KT = 128;       // keys per tile
constexpr int RT = 128;       // rows per pass
constexpr int THREADS = 416;
constexpr int DQ = 128;       // threads that dequantize
constexpr uint32_t kWaitPolls = 1u << 11;  // of at most 1 ms each

struct STcParams {
  ScoreParams s;
  int rows, passes;      // rows per KV head; passes of 128 of them
  int nctx, tiles;       // tiles of context rows; of all rows
  uint32_t total;        // tiles of all units
};

// one CTA's tiles of one unit
struct Part {
  int b, kvh, tile, ntiles;
};
struct Walk {
  uint32_t at, left;
  __device__ __forceinline__ bool next(const STcParams &P, Part &p) {
    if (left == 0) return false;
    const uint32_t unit = at / P.tiles;
    p.tile = static_cast<int>(at - unit * P.tiles);
    p.ntiles = static_cast<int>(min(static_cast<uint32_t>(P.tiles - p.tile), left));
    p.b = static_cast<int>(unit / P.s.t.Hkv);
    p.kvh = static_cast<int>(unit - p.b * P.s.t.Hkv);
    at += p.ntiles;
    left -= p.ntiles;
    return true;
  }
};

template <int D>
struct Smem {
  static constexpr int TILE = KT * D * 2;
  static constexpr int Q = 0, K = TILE, END = 3 * TILE;
  static constexpr int INFO = END;            // per two rows: float4 (c, c, -m, -m) [64], float2 (1 / l) [64]
  static constexpr int KFAC = INFO + 2048;    // float [4][4]: by tile and warp, what the scores of its rows are multiplied with
  static constexpr int BARS = KFAC + 64;
  static constexpr int MISC = BARS + 128;     // TMEM address, abort flag
  static constexpr int BYTES = MISC + 16;
};
enum Bar { KFULL = 0, KEMPTY = 2, SFULL = 4, SEMPTY = 6, QREADY = 8, NBARS = 9 };

struct Waiter {
  uint32_t bars, flag;
  __device__ __forceinline__ uint32_t at(int i) const { return bars + 8 * i; }
  // phase n of barrier i; after a time-out nobody waits any more: the CTA runs
  // through its loops, reports, and its output is not valid
  __device__ __forceinline__ void wait(int i, uint32_t n) const {
    const uint32_t bar = at(i), parity = n & 1u;
#pragma unroll 1
    for (uint32_t k = 0; k < kWaitPolls; ++k) {
      if (mbar_try_wait(bar, parity)) return;
      uint32_t off;
      asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(off) : "r"(flag) : "memory");
      if (off) return;
    }
    asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(flag), "r"(1u) : "memory");
    atomicOr(&g_trim_error_tc, DEV_ERR_MBAR_TIMEOUT);
  }
};

template <int D, int G>
__device__ __forceinline__ void dequant_role(const STcParams &P, Walk walk, const Waiter &W,
                                             uint32_t smem, int tid) {
  constexpr int RSTEP = DQ / Chunk<D>::CPR, NCH = KT / RSTEP, NS = G < 32 ? 2 : 1;
  using SM = Smem<D>;
  const TreeParams &T = P.s.t;
  struct Regs {
    uint4 w[NCH];
    uint16_t s[NCH * NS];
  };
  const Chunk<D> own(tid);
  const int r0 = own.row, c = own.c;
  Part p;
  bool have = walk.next(P, p);
  int i = 0, pass = 0, rem = 0;
  Source src{};
  auto point = [&]() {
    const int tile = p.tile + i;
    const bool draft = tile >= P.nctx;
    const int t0 = (draft ? tile - P.nctx : tile) * KT + r0;
    rem = static_cast<int>(draft ? T.ndraft : T.S) - t0;
    src = source_of<D, G, DQ>(T, draft, false, p.b, p.kvh, t0, c);
  };
  auto load = [&](Regs &r) {  // and step to the tile after it
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      r.w[k] = make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int e = NS * k; e < NS * k + NS; ++e) r.s[e] = 0;
      if (RSTEP * k < rem) {
        r.w[k] = __ldg(reinterpret_cast<const uint4 *>(src.p + static_cast<int64_t>(k) * src.pst));
#pragma unroll
        for (int e = 0; e < NS; ++e) r.s[NS * k + e] = __ldg(src.s + static_cast<int64_t>(k) * src.sst + e);
      }
    }
    if (++i < p.ntiles && p.tile + i != P.nctx) {
      src.p += static_cast<int64_t>(NCH) * src.pst;
      src.s += static_cast<int64_t>(NCH) * src.sst;
      rem -= KT;
      return;
    }
    if (i == p.ntiles) {  // the next pass over the same tiles, or the next part
      i = 0;
      if (++pass == P.passes) {
        pass = 0;
        have = walk.next(P, p);
      }
    }
    if (have) point();
  };
  bool big = false;
  uint32_t n = 0;
  auto turn_over = [&](Regs &r) {
    const uint32_t st = n & 1u, use = n >> 1, tile = smem + SM::K + st * SM::TILE;
    // the power of two of this warp's rows (see tc.cuh)
    float down = 1.0f;
    if (__any_sync(0xffffffffu, tc::scales_odd(r.s))) {
      const uint32_t top = tc::scales_top(r.s);
      if (top & 0x8000u) {
        const int shift = tc::scale_shift(top & 0x7FFFu);
        const float up = tc::pow2(shift);
        down = tc::pow2(-shift);
#pragma unroll
        for (int k = 0; k < NCH * NS; ++k) {
          r.s[k] = tc::scale_shifted(r.s[k], up);
          big = big || r.s[k] == 0x7F80u;
        }
      }
    }
    W.wait(KEMPTY + st, use + 1u);  // passes at once for the first use of a stage
    if ((tid & 31) == 0)
      asm volatile("st.shared.f32 [%0], %1;" ::"r"(smem + SM::KFAC + 16 * (n & 3u) + 4 * (tid >> 5)), "f"(down)
                   : "memory");
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      uint32_t sp[NS];
#pragma unroll
      for (int e = 0; e < NS; ++e) sp[e] = tc::scale_pair(r.s[NS * k + e]);
      store_chunk<D, NS>(tile, r0 + RSTEP * k, c, r.w[k], sp);
    }
    tc::fence_smem();
    __syncwarp();
    if ((tid & 31) == 0) mbar_arrive(W.at(KFULL + st));
    ++n;
  };
  Regs a, b2;
  bool ha = false, hb = false;
  if (have) point();
#pragma unroll 1
  do {
    if (ha) turn_over(a);
    ha = have;
    if (ha) load(a);
    if (hb) turn_over(b2);
    hb = have;
    if (hb) load(b2);
  } while (ha);
  if (big) atomicOr(&g_trim_error_tc, DEV_ERR_F16_RANGE);
}

// columns of a pass: its rows, to a multiple of 32 (the rest are zero rows)
__device__ __forceinline__ int pass_cols(const STcParams &P, int pass) {
  return min(RT, (P.rows - pass * RT + 31) & ~31);
}

template <int D>
__device__ __forceinline__ void mma_role(const STcParams &P, Walk walk, const Waiter &W,
                                         uint32_t smem, uint32_t tmem) {
  using SM = Smem<D>;
  Part p;
  uint32_t n = 0, np = 0;
  while (walk.next(P, p)) {
#pragma unroll 1
    for (int pass = 0; pass < P.passes; ++pass) {
      const uint32_t id = tc::idesc(static_cast<uint32_t>(pass_cols(P, pass)), false);
      W.wait(QREADY, np++);
#pragma unroll 1
      for (int i = 0; i < p.ntiles; ++i, ++n) {
        const uint32_t st = n & 1u, use = n >> 1;
        const uint64_t dk = tc::desc(smem + SM::K + st * SM::TILE, 16, 1024);
        const uint64_t dq = tc::desc(smem + SM::Q, 16, 1024);
        W.wait(SEMPTY + st, use + 1u);
        W.wait(KFULL + st, use);
        tc::fence_after();
        if (tc::elect()) {
#pragma unroll
          for (int j = 0; j < D / 16; ++j) {
            const uint64_t off = ((j >> 2) * tc::PANEL + (j & 3) * 32) / 16;
            tc::mma_ss(tmem + 128 * st, dk + off, dq + off, id, j > 0 ? 1u : 0u);
          }
          tc::commit(W.at(SFULL + st));
          tc::commit(W.at(KEMPTY + st));
        }
        __syncwarp();
      }
    }
  }
}

// Weights of 32 rows for this thread's key, in row order: even and odd rows
// apart.  FROM: rows below `from` do not see the key.
template <bool FROM>
__device__ __forceinline__ void add32(const uint32_t (&s)[32], uint32_t info, uint32_t inv, int from,
                                      uint64_t &sum) {
#pragma unroll
  for (int e = 0; e < 32; e += 2) {
    const uint4 v = lds128(info + 8 * e);  // c, c, -m, -m
    const uint2 li = lds64(inv + 4 * e);
    float x0, x1;
    unpair(fma2(pair(__uint_as_float(s[e]), __uint_as_float(s[e + 1])),
                pair(__uint_as_float(v.x), __uint_as_float(v.y)),
                pair(__uint_as_float(v.z), __uint_as_float(v.w))),
           x0, x1);
    x0 = fast_exp2(x0);
    x1 = fast_exp2(x1);
    if (FROM) {
      if (e < from) x0 = 0.0f;
      if (e + 1 < from) x1 = 0.0f;
    }
    sum = fma2(pair(x0, x1), pair(__uint_as_float(li.x), __uint_as_float(li.y)), sum);
  }
}

template <int D>
__device__ __forceinline__ void sum_role(const STcParams &P, Walk walk, const Waiter &W,
                                         uint32_t smem, uint32_t tmem, int tid) {
  using SM = Smem<D>;
  const TreeParams &T = P.s.t;
  const int lane = tid & 31, r = tid & 127;
  const uint32_t group = tid >> 7;  // takes the tiles of its parity, in its own buffer
  const uint32_t tS = tmem + 128 * group + (static_cast<uint32_t>((tid >> 5) & 3) << 21);
  Part p;
  uint32_t n = 0;
  while (walk.next(P, p)) {
    const int unit = p.b * T.Hkv + p.kvh;
    const float *in = P.s.in + p.b * P.s.is[0] + p.kvh * P.s.is[1];
    float *out = P.s.out + p.b * P.s.os[0] + p.kvh * P.s.os[1];
#pragma unroll 1
    for (int pass = 0; pass < P.passes; ++pass) {
      const int cols = pass_cols(P, pass);
      // all products with the last queries are complete: their scores have been
      // read, and what the last pass added can be read
      asm volatile("bar.sync 1, 256;" ::: "memory");
      if (group == 0) {
        const int row = pass * RT + r;
        const float c0 = load_query_row<D>(T, P.rows, p.b, p.kvh, row, smem + SM::Q, r);
        float c = 0.0f, nm = 0.0f, li = 0.0f;
        if (row < P.rows) {
          const float2 st = T.stats[static_cast<int64_t>(unit) * P.rows + row];
          // a row that saw nothing weighs nothing: 2^0 * 0
          if (st.y != 0.0f) {
            c = c0;
            nm = -st.x;
            li = st.y;
          }
        }
        float *info = reinterpret_cast<float *>(__cvta_shared_to_generic(smem + SM::INFO));
        info[(r >> 1) * 4 + (r & 1)] = c;
        info[(r >> 1) * 4 + 2 + (r & 1)] = nm;
        info[256 + r] = li;
        tc::fence_smem();
        tc::fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(W.at(QREADY));
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");  // everyone's rows are in INFO
#pragma unroll 1
      for (int i = 0; i < p.ntiles; ++i, ++n) {
        if ((n & 1u) != group) continue;
        const int tile = p.tile + i;
        const bool draft = tile >= P.nctx;
        const int key = (draft ? tile - P.nctx : tile) * KT + r;  // within its source
        const bool ok = key < (draft ? T.ndraft : static_cast<int>(T.S));
        const int64_t t = draft ? T.S + key : key;
        const float *from_where = pass == 0 ? in + t * P.s.is[2] : out + t * P.s.os[2];
        float old = 0.0f;  // not used before the sums are there
        if (ok) old = *from_where;
        W.wait(SFULL + group, n >> 1);
        tc::fence_after();
        // query i sees drafted key j iff j <= i + shift
        const int from = draft && T.causal ? max(0, key - T.shift) * T.R - pass * RT : 0;
        const bool some = __any_sync(0xffffffffu, from > 0);
        // of the warp that dequantized this key; seldom other than 1.  Its place is
        // written again four tiles on, behind SEMPTY below
        const float kf = __uint_as_float(lds32(smem + SM::KFAC + 16 * (n & 3u) + 4 * Chunk<D>::warp_of(r)));
        const bool shifted = __any_sync(0xffffffffu, kf != 1.0f);
        uint64_t sum = 0;
#pragma unroll 1
        for (int c = 0; c < cols; c += 32) {
          uint32_t s[32];
          tc::ld32(tS + c, s);
          tc::wait_ld(s);
          if (shifted) {
#pragma unroll
            for (int e = 0; e < 32; ++e) s[e] = __float_as_uint(__uint_as_float(s[e]) * kf);
          }
          const uint32_t info = smem + SM::INFO + 8 * c;
          if (some) add32<true>(s, info, info + 1024 - 4 * c, from - c, sum);
          else add32<false>(s, info, info + 1024 - 4 * c, 0, sum);
        }
        tc::fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(W.at(SEMPTY + group));
        float t0, t1;
        unpair(sum, t0, t1);
        if (ok) out[t * P.s.os[2]] = fmaf(old, pass == 0 ? P.s.decay : 1.0f, t0 + t1);
      }
    }
  }
}

template <int D, int G>
__global__ void __launch_bounds__(THREADS, 2) score_tc(const __grid_constant__ STcParams P) {
  using SM = Smem<D>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t smem = smem_u32(smem_raw);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Waiter W{smem + SM::BARS, smem + SM::MISC + 4};
  if (smem & 1023u) {  // the swizzled tiles need 1024-byte alignment
    if (tid == 0) atomicOr(&g_trim_error_tc, DEV_ERR_MBAR_TIMEOUT);
    return;
  }
  if (warp == 8) {
    if (lane < NBARS) mbar_init(W.at(lane), lane >= KEMPTY && lane < SEMPTY ? 1 : 4);
    fence_mbar_init();
    if (lane == 0) *reinterpret_cast<volatile uint32_t *>(smem_raw + SM::MISC + 4) = 0u;
  }
  if (warp == 12) tc::alloc(smem + SM::MISC, 256);
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem =
      __shfl_sync(0xffffffffu, *reinterpret_cast<volatile uint32_t *>(smem_raw + SM::MISC), 0);
  const uint32_t each = P.total / gridDim.x, rest = P.total - each * gridDim.x;
  const Walk walk{blockIdx.x * each + min(blockIdx.x, rest), each + (blockIdx.x < rest ? 1u : 0u)};
  griddep_wait();  // the rows' maxima and sums come from the kernel before
  if (warp < 8) sum_role<D>(P, walk, W, smem, tmem, tid);
  else if (warp < 12) dequant_role<D, G>(P, walk, W, smem, tid - 256);
  else mma_role<D>(P, walk, W, smem, tmem);
  __syncwarp();
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (warp == 12) tc::dealloc(tmem, 256);
}

STcParams score_plan(const ScoreParams &S) {
  STcParams P{};
  P.s = S;
  P.rows = S.t.R * S.t.nodes;
  P.passes = (P.rows + RT - 1) / RT;
  P.nctx = static_cast<int>((S.t.S + KT - 1) / KT);
  P.tiles = P.nctx + (S.t.ndraft + KT - 1) / KT;
  return P;
}

template <int D, int G>
int launch_score(const STcParams &P, cudaStream_t st) {
  static bool configured[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = 0;
  if (!configured[dev]) {
    const int rc = cuda_status(cudaFuncSetAttribute(
        score_tc<D, G>, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<D>::BYTES));
    if (rc) return rc;
    configured[dev] = true;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(std::min<uint32_t>(2u * sm_count(), P.total));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = Smem<D>::BYTES;
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, score_tc<D, G>, P));
}

}  // namespace

// For the calls that tree_tc takes, with at least one row and one key (the rows'
// statistics are in terms of the same operands).
int score_tc_run(const ScoreParams &S, cudaStream_t st) {
  STcParams P = score_plan(S);
  const int64_t total = S.t.B * S.t.Hkv * P.tiles;
  if (total >= (int64_t(1) << 31)) return KV4_ERR_UNSUPPORTED;
  P.total = static_cast<uint32_t>(total);
  if (S.t.d == 64) {
    switch (S.t.G) {
      case 16: return launch_score<64, 16>(P, st);
      case 32: return launch_score<64, 32>(P, st);
      default: return launch_score<64, 64>(P, st);
    }
  }
  switch (S.t.G) {
    case 16: return launch_score<128, 16>(P, st);
    case 32: return launch_score<128, 32>(P, st);
    case 64: return launch_score<128, 64>(P, st);
    default: return launch_score<128, 128>(P, st);
  }
}

int trim_tc_take_device_error(int *v) {
  int zero = 0;
  int rc = cuda_status(cudaMemcpyFromSymbol(v, g_trim_error_tc, sizeof(int)));
  if (rc) return rc;
  return cuda_status(cudaMemcpyToSymbol(g_trim_error_tc, &zero, sizeof(int)));
}

}  // namespace kv4
