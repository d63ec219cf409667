// Tree attention on the 5th-generation tensor cores (tcgen05), for bf16
// queries over caches with bf16 scales and head sizes 64 and 128.
//
// The mathematics is branch.cu's.  All rows (node, q head of the group) that
// read one KV head form the M dimension, 128 at a time, so a tile of 128 keys
// is dequantized once for up to 256 rows.  One CTA per SM, 20 warps:
//
//   warps 0-7    softmax: two streams of 128 threads, a thread per row.  A
//                stream reads its scores from tensor memory, keeps the running
//                maximum and sum, writes the weights back as f16 over the
//                scores, and rescales its output accumulator when the maximum
//                moved by more than 2^8 (seldom).
//   warps 8-15   dequantization, four warps each for K and V: chunks of 16 bytes
//                (32 codes), loaded a tile ahead into registers, to f16 tiles
//                in the swizzled layout of the matrix descriptors, double-buffered.
//   warp 16      an elected lane issues S = Q K^T and O += P V for both streams.
//   warps 17-19  turn the mask bytes of drafted tiles into 128 bits per row.
//
// With more than 128 rows the streams are two row tiles that share every
// dequantized key tile; with fewer they are the even and odd key tiles of one
// row tile, joined at the end through shared memory.  Either way the tensor
// cores work on one stream while the other is in its softmax.
//
// Work is cut evenly: the (unit, key tile) pairs of all sequences lie end to
// end and CTA c takes pairs [c W / n, (c + 1) W / n).  A unit that falls into
// several CTAs leaves partial rows in the workspace, column by column (a warp
// then writes 32 rows of a column in one piece), which tree_tc_merge joins in a
// fixed order.  Lengths are read on the device.
//
// Operands are f16: q times a power of two per row that brings its largest
// element to [2^13, 2^14) (exact for bf16), K and V values exactly (tc.cuh).
// Weights enter the second product rounded to f16, times 2^7 (at most 2^15);
// their sum is taken before that rounding, in fp32.
//
// Bound: the chain scores -> maximum -> weights -> products of a stream, 5000 cycles
// a tile with both streams at it, where products and exponentials need 2048 each.
// Measured: 64 nodes x 16K x 64 heads over 8, batch 4, 149 us (755 TFLOP/s); 63 nodes
// x 4K x 32 heads, batch 8, 54 us, of which about 5 pass before the first product.
#include <algorithm>

#include "branch.cuh"
#include "tc_rows.cuh"

namespace kv4 {

// device error word of this file (folded into kv4_device_error)
__device__ int g_branch_error_tc = 0;

namespace {

constexpr int KT = 128;      // keys per tile
constexpr int THREADS = 640;  // five warpgroups of 96 registers a thread, shared out below
constexpr int DQ = 128;       // threads that dequantize K, and V
constexpr float kWeightShift = 7.0f;  // weights are written times 2^7: f16 then resolves 2^-31 of the largest
constexpr uint32_t kWaitPolls = 1u << 11;  // of at most 1 ms each

struct TcParams {
  TreeParams t;
  int rows, blocks;  // rows per KV head; blocks of 256 of them
  int dtiles;        // tiles of drafted rows
  int2 *shares;      // workspace, per unit and block: slot of its first share (-1:
                     // it was whole in one CTA) and CTA of its last
};
constexpr int WS_ROWS = 256;  // rows of a partial slot, [column][row]

__device__ __forceinline__ int ctx_tiles(const TcParams &P, int b, int *err = nullptr) {
  return static_cast<int>((static_cast<uint32_t>(context_len(P.t, b, err)) + KT - 1) / KT);
}
__device__ __forceinline__ int unit_tiles(const TcParams &P, int b, int *err = nullptr) {
  return ctx_tiles(P, b, err) + P.dtiles;
}

// one CTA's share of one unit
struct Segment {
  int b, kvh, row0, nrows;  // rows [row0, row0 + nrows) of KV head kvh of sequence b
  int tile, ntiles;         // key tiles [tile, tile + ntiles)
  bool whole, last;         // all of the unit's tiles; its last one among them
  bool first;               // the CTA's first segment
};

// rows of a 128-row tile that differ: up to 64 (32) lie in it twice (four times)
__device__ __forceinline__ int tile_rows(const Segment &s) {
  return s.nrows > 64 ? 128 : s.nrows > 32 ? 64 : 32;
}

// walks a CTA's segments; every role walks its own copy
struct Walk {
  uint32_t left;            // tiles still to do
  int b, kvh, blk, t;
  bool first;
  __device__ __forceinline__ bool next(const TcParams &P, Segment &s) {
    if (left == 0) return false;
    int T = unit_tiles(P, b);
#pragma unroll 1
    while (T == 0) T = unit_tiles(P, ++b);  // units without keys have no work
    s.b = b;
    s.kvh = kvh;
    s.row0 = blk * 256;
    s.nrows = min(256, P.rows - s.row0);
    s.tile = t;
    s.ntiles = static_cast<int>(min(static_cast<uint32_t>(T - t), left));
    s.whole = s.ntiles == T;
    s.last = t + s.ntiles == T;
    s.first = first;
    first = false;
    left -= s.ntiles;
    t += s.ntiles;
    if (t == T) {
      t = 0;
      if (++blk == P.blocks) {
        blk = 0;
        if (++kvh == P.t.Hkv) {
          kvh = 0;
          ++b;
        }
      }
    }
    return true;
  }
};

template <int D>
struct Smem {
  static constexpr int TILE = KT * D * 2;  // 128 rows of D 16-bit values
  static constexpr int Q = 0, K = 2 * TILE, V = 4 * TILE, END = 6 * TILE;
  static constexpr int ML = END;            // float2 [2][128]
  static constexpr int MASK = ML + 2048;    // uint4 [2][128]: a row's visible keys of a drafted tile
  static constexpr int QC = MASK + 4096;    // float [2][128]: a row's factor from scores to base-2 exponents
  static constexpr int BAD = QC + 1024;   // uint32 [4 + 2][4]: drafted keys without a usable scale in K, V
  static constexpr int TOPS = BAD + 96;     // uint32 [2][4]: by K's and by V's warps: each one's largest scales
  static constexpr int POWERS = TOPS + 32;  // int16 [4][2]: powers of two of K and of V in the last four tiles
  static constexpr int BARS = POWERS + 16;  // mbarriers
  static constexpr int MISC = BARS + 176;   // TMEM address, abort flag, walk start
  static constexpr int BYTES = MISC + 64;
};

// barriers (pairs: by stage or by stream) and their arrival counts
enum Bar { KFULL = 0, VFULL = 2, KEMPTY = 4, VEMPTY = 6, SFULL = 8, PREADY = 10, OREADY = 12,
           MFULL = 14, MEMPTY = 16, QREADY = 18, QFREE = 19, QSEEN = 20, NBARS = 21 };
__device__ __forceinline__ int bar_count(int i) {
  if (i < KEMPTY) return 4;           // dequantizing warps of K, of V
  if (i < PREADY) return 1;           // commits
  if (i < OREADY) return 4;           // a stream's warps
  if (i < MFULL) return 1;
  if (i < MEMPTY) return 3;           // mask warps
  return i < QREADY ? 4 : 8;
}

struct Waiter {
  uint32_t bars, flag;
  __device__ __forceinline__ uint32_t at(int i) const { return bars + 8 * i; }
  // wait for phase number n of barrier i; after a time-out nobody waits any
  // more: the CTA runs through its loops, reports, and its output is not valid
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
    atomicOr(&g_branch_error_tc, DEV_ERR_MBAR_TIMEOUT);
  }
};

__device__ __forceinline__ void bar_softmax() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

// ---------------------------------------------------------------------------
// Four warps dequantize K, four V, each at their own pace: scores are asked for a
// tile ahead of the products with V, so that V must not hold up K.
template <int D, int G>
__device__ __forceinline__ void dequant_role(const TcParams &P, Walk walk, const Waiter &W,
                                             uint32_t smem, bool is_v, int tid) {
  constexpr int RSTEP = DQ / Chunk<D>::CPR;  // rows between a thread's chunks
  constexpr int NCH = KT / RSTEP;            // chunks per thread and tile
  constexpr int NS = G < 32 ? 2 : 1;         // scales per chunk
  using SM = Smem<D>;
  struct Regs {
    uint4 w[NCH];
    uint16_t s[NCH * NS], sv[NCH * NS];  // scales; K's warps: V's beside them
    bool draft;
  };
  const TreeParams &T = P.t;
  const Chunk<D> own(tid);
  const int r0 = own.row, c = own.c;

  Segment s;
  int nctx = 0, len = 0, rem = 0;
  Source src{}, vsrc{};
  auto load = [&](Regs &r, int i) {  // tile i of the segment
    const int tile = s.tile + i;
    r.draft = tile >= nctx;
    if (i == 0 || tile == nctx) {
      const int t0 = (r.draft ? tile - nctx : tile) * KT + r0;
      rem = (r.draft ? T.ndraft : len) - t0;
      src = source_of<D, G, DQ>(T, r.draft, is_v, s.b, s.kvh, t0, c);
      if (!is_v) vsrc = source_of<D, G, DQ>(T, r.draft, true, s.b, s.kvh, t0, c);
    } else {
      src.p += static_cast<int64_t>(NCH) * src.pst;
      src.s += static_cast<int64_t>(NCH) * src.sst;
      vsrc.s += static_cast<int64_t>(NCH) * vsrc.sst;
      rem -= KT;
    }
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      r.w[k] = make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int e = NS * k; e < NS * k + NS; ++e) r.s[e] = r.sv[e] = 0;
      if (RSTEP * k < rem) {
        r.w[k] = __ldg(reinterpret_cast<const uint4 *>(src.p + static_cast<int64_t>(k) * src.pst));
#pragma unroll
        for (int e = 0; e < NS; ++e) {
          r.s[NS * k + e] = __ldg(src.s + static_cast<int64_t>(k) * src.sst + e);
          if (!is_v) r.sv[NS * k + e] = __ldg(vsrc.s + static_cast<int64_t>(k) * vsrc.sst + e);
        }
      }
    }
  };
  bool big = false;
  int least = 0;   // smallest power of two in V's tiles of the segment
  uint32_t n = 0;  // tiles so far
  auto turn_over = [&](Regs &r) {  // a loaded tile to shared memory
    const uint32_t st = n & 1u, use = n >> 1;
    // marks of drafted keys: K's of the last four tiles, V's of the last two
    // (when a stage is free again, the marks of the tile that far back have been read)
    const uint32_t bad = smem + SM::BAD + 16 * (is_v ? 4 + st : n & 3u);
    const uint32_t tile = smem + (is_v ? SM::V : SM::K) + st * SM::TILE;
    // The tile's powers of two (see tc.cuh).  K's warps find V's as well, from the
    // same scales by the same rule, so that the softmax warps have it with the
    // scores and need not wait for V (2 % of a tile).
    bool odd = tc::scales_odd(r.s);
    if (!is_v) odd = odd || tc::scales_odd(r.sv);
    W.wait((is_v ? VEMPTY : KEMPTY) + st, use + 1u);  // passes at once for the first use of a stage
    if (r.draft && tid < 4) asm volatile("st.shared.u32 [%0], %1;" ::"r"(bad + 4 * tid), "r"(0u) : "memory");
    int shift = 0, vshift = 0;
    __syncwarp();
    odd = tc::barrier_any(is_v ? 3 : 2, odd);
    if (odd) {
      // the four warps put their largest scales together (low half: their own)
      const uint32_t tops = smem + SM::TOPS + 16 * is_v;
      uint32_t top = tc::scales_top(r.s);
      if (!is_v) top |= tc::scales_top(r.sv) << 16;
      if ((tid & 31) == 0) asm volatile("st.shared.u32 [%0], %1;" ::"r"(tops + 4 * (tid >> 5)), "r"(top) : "memory");
      asm volatile("bar.sync %0, 128;" ::"r"(is_v ? 3 : 2) : "memory");
      const uint4 t = lds128(tops);  // (not written again before the next tile's first barrier)
      const uint32_t m = __vmaxu2(__vmaxu2(t.x & 0x7FFF7FFFu, t.y & 0x7FFF7FFFu),
                                  __vmaxu2(t.z & 0x7FFF7FFFu, t.w & 0x7FFF7FFFu));
      const uint32_t not_exact = t.x | t.y | t.z | t.w;
      if (not_exact & 0x8000u) shift = tc::scale_shift(m & 0xFFFFu);
      if (not_exact >> 31) vshift = tc::scale_shift(m >> 16);
    }
    // V's sums of earlier tiles move up by 2^48 at most, which they can
    (is_v ? shift : vshift) = min(is_v ? shift : vshift, least + 48);
    least = min(least, is_v ? shift : vshift);
    if (!is_v && tid == 0)
      asm volatile("st.shared.u32 [%0], %1;" ::"r"(smem + SM::POWERS + 4 * (n & 3u)),
                   "r"((static_cast<uint32_t>(shift) & 0xFFFFu) | static_cast<uint32_t>(vshift) << 16)
                   : "memory");
    if (odd || shift != 0) {
      const float up = tc::pow2(shift);
#pragma unroll
      for (int k = 0; k < NCH * NS; ++k) {
        r.s[k] = tc::scale_shifted(r.s[k], up);
        if (r.s[k] != 0x7F80u) continue;
        big = true;
        if (r.draft) {  // seen by some rows only: out of the product, those rows are marked
          const int row = r0 + RSTEP * (k / NS);
          r.s[k] = 0;
          asm volatile("red.shared.or.b32 [%0], %1;" ::"r"(bad + 4 * (row >> 5)), "r"(1u << (row & 31)) : "memory");
        }
      }
    }
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      uint32_t sp[NS];
#pragma unroll
      for (int e = 0; e < NS; ++e) sp[e] = tc::scale_pair(r.s[NS * k + e]);
      store_chunk<D, NS>(tile, r0 + RSTEP * k, c, r.w[k], sp);
    }
    tc::fence_smem();
    __syncwarp();
    if ((tid & 31) == 0) mbar_arrive(W.at((is_v ? VFULL : KFULL) + st));
    ++n;
  };
  // the next tile is on its way while one waits for its stage and is stored
  Regs a;
  bool narrow = false;  // the segment before had one row tile
#pragma unroll 1
  for (uint32_t seg = 0; walk.next(P, s); ++seg) {
    len = static_cast<int>(context_len(T, s.b, nullptr));
    nctx = (len + KT - 1) / KT;
    least = tc::kMaxShift;
    load(a, 0);
    // The segment's queries, a row tile by K's warps and one by V's: as soon as
    // the scores of the segment before are out and the softmax warps have its
    // factors, beside its last softmax and its epilogue; behind that epilogue where
    // its exchange uses the queries' place.  QSEEN is waited for in every segment:
    // it keeps QREADY from running ahead of a softmax warp by two phases, which a
    // wait by parity takes for none, and says that segment seg - 2 is over, without
    // which the wait for QFREE could pass a phase early.
    if (seg > 0) {
      W.wait(KEMPTY + ((n - 1) & 1u), (n - 1) >> 1);
      W.wait(QSEEN, seg - 1);
      if (narrow) W.wait(QFREE, seg - 1);
    }
    const bool two = s.nrows > 128;
    narrow = !two;
    if (two || !is_v) {
      const int row = s.row0 + (two ? 128 * is_v + tid : tid & (tile_rows(s) - 1));
      const float c0 = load_query_row<D>(T, P.rows, s.b, s.kvh, row, smem + SM::Q + is_v * SM::TILE, tid);
      asm volatile("st.shared.f32 [%0], %1;" ::"r"(smem + SM::QC + 4 * (128 * is_v + tid)), "f"(c0) : "memory");
    }
    tc::fence_smem();
    __syncwarp();
    if ((tid & 31) == 0) mbar_arrive(W.at(QREADY));
#pragma unroll 1
    for (int i = 0; i < s.ntiles; ++i) {
      turn_over(a);
      if (i + 1 < s.ntiles) load(a, i + 1);
    }
  }
  if (big) atomicOr(&g_branch_error_tc, DEV_ERR_F16_RANGE);
}

// ---------------------------------------------------------------------------
// The whole warp runs this converged; one elected lane issues.
template <int D>
__device__ __forceinline__ void mma_role(const TcParams &P, Walk walk, const Waiter &W,
                                         uint32_t smem, uint32_t tmem) {
  using SM = Smem<D>;
  constexpr uint32_t id_s = tc::idesc(128, false), id_o = tc::idesc(D, true);
  Segment s;
  uint32_t base = 0, seg = 0;         // tiles before this segment; segments
  uint32_t np0 = 0, np1 = 0;          // steps of each stream before this segment
  while (walk.next(P, s)) {
    const bool two = s.nrows > 128;   // two row tiles, or even and odd key tiles
    const int nt = s.ntiles;
    const int s0 = two ? nt : (nt + 1) / 2, s1 = two ? nt : nt / 2;
    W.wait(QREADY, seg);
    // S0(0) S1(0) | O0(i) S0(i+1) O1(i) S1(i+1) | ...: scores go out behind the
    // product that reads the weights they overwrite
#pragma unroll 1
    for (int i = -1; i < s0; ++i) {
#pragma unroll 1
      for (int x = 0; x < 2; ++x) {
        const int steps = x ? s1 : s0;
        const bool last = !two || x == 1;  // stream that uses a tile last
        if (i >= 0 && i < steps) {
          const uint32_t n = base + (two ? i : 2 * i + x), st = n & 1u;
          const uint64_t dv = tc::desc(smem + SM::V + st * SM::TILE, tc::PANEL, 1024);
          W.wait(VFULL + st, n >> 1);
          W.wait(PREADY + x, (x ? np1 : np0) + i);
          tc::fence_after();
          if (tc::elect()) {
#pragma unroll
            for (int j = 0; j < KT / 16; ++j)
              tc::mma_ts(tmem + 256 + 128 * x, tmem + 128 * x + 8 * j, dv + j * 128, id_o,
                         (i > 0 || j > 0) ? 1u : 0u);
            tc::commit(W.at(OREADY + x));
            if (last) tc::commit(W.at(VEMPTY + st));
          }
          __syncwarp();
        }
        if (i + 1 < steps) {
          const uint32_t n = base + (two ? i + 1 : 2 * (i + 1) + x), st = n & 1u;
          const uint64_t dq = tc::desc(smem + SM::Q + (two ? x : 0) * SM::TILE, 16, 1024);
          const uint64_t dk = tc::desc(smem + SM::K + st * SM::TILE, 16, 1024);
          W.wait(KFULL + st, n >> 1);
          tc::fence_after();
          if (tc::elect()) {
#pragma unroll
            for (int j = 0; j < D / 16; ++j) {
              const uint64_t off = ((j >> 2) * tc::PANEL + (j & 3) * 32) / 16;
              tc::mma_ss(tmem + 128 * x, dq + off, dk + off, id_s, j > 0 ? 1u : 0u);
            }
            tc::commit(W.at(SFULL + x));
            if (last) tc::commit(W.at(KEMPTY + st));
          }
          __syncwarp();
        }
      }
    }
    np0 += s0;
    np1 += s1;
    base += nt;
    ++seg;
  }
}

// ---------------------------------------------------------------------------
// Three warps turn the mask of each drafted tile into four words per row; a
// warp takes every third node, a lane every 32nd key.
template <int D>
__device__ __forceinline__ void mask_role(const TcParams &P, Walk walk, const Waiter &W,
                                          uint32_t smem, int part, int lane) {
  using SM = Smem<D>;
  const TreeParams &T = P.t;
  if (!T.mask || P.dtiles == 0) return;
  Segment s;
  uint32_t nm0 = 0, nm1 = 0;  // drafted tiles of each stream so far
  while (walk.next(P, s)) {
    const bool two = s.nrows > 128;
    const int nctx = ctx_tiles(P, s.b);
#pragma unroll 1
    for (int j = max(0, nctx - s.tile); j < s.ntiles; ++j) {
      const int j0 = (s.tile + j - nctx) * KT;
#pragma unroll 1
      for (int x = 0; x < 2; ++x) {
        if (!two && (j & 1) != x) continue;
        W.wait(MEMPTY + x, (x ? nm1 : nm0) + 1u);
        const int ra = s.row0 + (two ? 128 * x : 0), rb = min(ra + 128, P.rows);
#pragma unroll 1
        for (int nd = ra / T.R + part; nd * T.R < rb; nd += 3) {
          const uint8_t *m = T.mask + s.b * T.ms[0] + nd * T.ms[1];
          uint32_t byte[4], word[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int jj = j0 + 32 * q + lane;
            byte[q] = jj < T.ndraft ? __ldg(m + jj * T.ms[2]) : 0u;
          }
#pragma unroll
          for (int q = 0; q < 4; ++q) word[q] = __ballot_sync(0xffffffffu, byte[q] != 0u);
#pragma unroll 1
          for (int r = max(nd * T.R, ra) + lane; r < min((nd + 1) * T.R, rb); r += 32)
            tc::sts128(smem + SM::MASK + 16 * (128 * x + r - ra), word[0], word[1], word[2], word[3]);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(W.at(MFULL + x));
        if (x) ++nm1;
        else ++nm0;
      }
    }
  }
}

// ---------------------------------------------------------------------------
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// A score, or -infinity where the row does not see its column (bit `e` of `bits`).
template <bool MASKED>
__device__ __forceinline__ float seen(uint32_t s, int e, uint32_t bits) {
  const float f = __uint_as_float(s);
  return !MASKED || ((bits >> e) & 1u) ? f : -INFINITY;
}

__device__ __forceinline__ uint32_t word_of(const uint4 &v, int i) {
  return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}

// largest visible score of 16 columns
template <bool MASKED>
__device__ __forceinline__ void max16(const uint32_t (&s)[16], uint32_t bits, float &m0, float &m1) {
#pragma unroll
  for (int e = 0; e < 16; e += 4) {
    m0 = max3(m0, seen<MASKED>(s[e], e, bits), seen<MASKED>(s[e + 1], e + 1, bits));
    m1 = max3(m1, seen<MASKED>(s[e + 2], e + 2, bits), seen<MASKED>(s[e + 3], e + 3, bits));
  }
}

// Both passes take columns [32 cs, 32 ce) 16 at a time, the next ones on their
// way from tensor memory, in rolled loops: the kernel's roles run side by side,
// and the code of all of them has to stay in the instruction cache.
template <bool MASKED>
__device__ __forceinline__ float tile_max(uint32_t tS, const uint4 &bits, int cs, int ce) {
  float m0 = -INFINITY, m1 = -INFINITY;
  uint32_t a[16], b[16];
  tc::ld16(tS + 32 * cs, a);
#pragma unroll 1
  for (int c = cs; c < ce; ++c) {
    const uint32_t bw = MASKED ? word_of(bits, c) : 0u;
    tc::wait_ld16(a);
    tc::ld16(tS + 32 * c + 16, b);
    max16<MASKED>(a, bw, m0, m1);
    tc::wait_ld16(b);
    if (c + 1 < ce) tc::ld16(tS + 32 * c + 32, a);
    max16<MASKED>(b, bw >> 16, m0, m1);
  }
  return fmaxf(m0, m1);
}

// weights 2^(s c0 - m) of 16 scores as f16, added to the sums
template <bool MASKED>
__device__ __forceinline__ void weights16(const uint32_t (&s)[16], uint32_t bits, uint64_t cc,
                                          uint64_t mm, uint64_t &l0, uint64_t &l1, uint32_t to) {
  uint32_t pk[8];
#pragma unroll
  for (int e = 0; e < 16; e += 2) {
    float x0, x1;
    unpair(fma2(pair(seen<MASKED>(s[e], e, bits), seen<MASKED>(s[e + 1], e + 1, bits)), cc, mm), x0, x1);
    x0 = fast_exp2(x0);
    x1 = fast_exp2(x1);
    if (e & 2) l1 = add2(l1, pair(x0, x1));
    else l0 = add2(l0, pair(x0, x1));
    pk[e >> 1] = pack_f16x2(x0, x1);
  }
  tc::st8(to, pk);
}

// ... of a tile's columns, written over its scores; returns their sum
template <bool MASKED>
__device__ __forceinline__ float tile_weights(uint32_t tS, float c0, float m, const uint4 &bits,
                                              int cs, int ce) {
  const uint64_t cc = pair(c0, c0), mm = pair(-m, -m);
  uint64_t l0 = 0, l1 = 0;
  uint32_t a[16], b[16];
  tc::ld16(tS + 32 * cs, a);
#pragma unroll 1
  for (int c = cs; c < ce; ++c) {
    const uint32_t bw = MASKED ? word_of(bits, c) : 0u;
    tc::wait_ld16(a);
    tc::ld16(tS + 32 * c + 16, b);
    // over columns that have been read: 16 c + 7 < 32 c + 16
    weights16<MASKED>(a, bw, cc, mm, l0, l1, tS + 16 * c);
    tc::wait_ld16(b);
    if (c + 1 < ce) tc::ld16(tS + 32 * c + 32, a);
    weights16<MASKED>(b, bw >> 16, cc, mm, l0, l1, tS + 16 * c + 8);
  }
  float s0, s1;
  unpair(add2(l0, l1), s0, s1);
  return s0 + s1;
}

template <int D>
__device__ __forceinline__ void softmax_role(const TcParams &P, Walk walk, const Waiter &W,
                                             uint32_t smem, uint32_t tmem, int tid) {
  using SM = Smem<D>;
  const TreeParams &T = P.t;
  const int x = tid >> 7, r = tid & 127, lane = tid & 31;
  const uint32_t lanes = static_cast<uint32_t>((tid >> 5) & 3) << 21;  // 32 lanes per warp
  const uint32_t tS = tmem + 128 * x + lanes, tO = tmem + 256 + 128 * x + lanes;
  Segment s;
  // steps and drafted tiles of this stream; segments; tiles before this segment
  uint32_t ns = 0, nm = 0, seg = 0, base = 0;
  while (walk.next(P, s)) {
    const bool two = s.nrows > 128;
    const int nt = s.ntiles, steps = two ? nt : (nt + 1 - x) / 2;
    // Up to 64 (32) rows lie in the tile twice (four times): each copy takes a
    // half (a quarter) of every key tile's columns, with a maximum, a sum and an
    // output of its own, so that all warps have work.
    const int RR = tile_rows(s), copies = 128 / RR;
    const int copy = r / RR, cs = copy * 4 / copies, ce = cs + 4 / copies;
    const int row = s.row0 + (two ? 128 * x + r : r & (RR - 1));
    const bool ok = row < P.rows, idle = __all_sync(0xffffffffu, !ok);
    const int node = row / T.R, head = s.kvh * T.R + row - node * T.R;

    const int len = static_cast<int>(context_len(T, s.b, nullptr)), nctx = (len + KT - 1) / KT;
    W.wait(QREADY, seg++);
    const float c0 = __uint_as_float(lds32(smem + SM::QC + 4 * (two ? tid : r & (RR - 1))));
    __syncwarp();
    if (lane == 0) mbar_arrive(W.at(QSEEN));

    float m = -INFINITY, l = 0.0f;
    bool broken = false;  // saw a key without a usable scale
    uint32_t vpower = 0;  // power of two in this stream's output (V's half of a tile's powers)
    for (int i = 0; i < steps; ++i) {
      const int j = two ? i : 2 * i + x, tile = s.tile + j;
      const bool draft = tile >= nctx;
      uint4 bits;
      bool whole = false;
      if (draft && T.mask) {
        W.wait(MFULL + x, nm++);
        bits = lds128(smem + SM::MASK + 16 * (128 * x + (r & (RR - 1))));
        __syncwarp();
        if (lane == 0) mbar_arrive(W.at(MEMPTY + x));
      } else {  // the first `lim` keys of the tile
        int lim;
        if (draft) {
          const int j0 = (tile - nctx) * KT;
          lim = min(KT, T.ndraft - j0);
          if (T.causal) lim = min(lim, node + T.shift + 1 - j0);
        } else {
          lim = len - tile * KT;
        }
        whole = __all_sync(0xffffffffu, lim >= KT);
        auto below = [&](int q) {
          const int k = min(max(lim - 32 * q, 0), 32);
          return k == 32 ? 0xffffffffu : (1u << k) - 1u;
        };
        bits = make_uint4(below(0), below(1), below(2), below(3));
      }
      W.wait(SFULL + x, ns);
      tc::fence_after();
      if (!idle) {  // rows past the last: their weights may be anything
        const uint32_t n = base + j, powers = lds32(smem + SM::POWERS + 4 * (n & 3u));
        auto scale_columns = [](uint32_t at, int from, int to, float f) {
#pragma unroll 1
          for (int col = from; col < to; col += 32) {
            uint32_t o[32];
            tc::ld32(at + col, o);
            tc::wait_ld(o);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            tc::st32(at + col, o);
          }
        };
        if (powers != vpower) {  // seldom
          const int ks = static_cast<int16_t>(powers & 0xFFFFu), vs = static_cast<int16_t>(powers >> 16),
                    was = static_cast<int16_t>(vpower >> 16);
          if (ks != 0) {
            scale_columns(tS, 32 * cs, 32 * ce, tc::pow2(-ks));
            tc::wait_st();
          }
          if (i > 0 && vs != was) {
            W.wait(OREADY + x, ns - 1);
            tc::fence_after();
            scale_columns(tO, 0, D, tc::pow2(vs - was));
            tc::wait_st();
          }
          vpower = powers & 0xFFFF0000u;
        }
        const float mx = (whole ? tile_max<false>(tS, bits, cs, ce) : tile_max<true>(tS, bits, cs, ce)) * c0;
        // the maximum moves only when a score passes it by more than 8, so that
        // weights stay below 2^8 (2^15 as written): seldom after a row's first tile
        const bool up = mx > m + 8.0f;
        if (__any_sync(0xffffffffu, up)) {
          const float alpha = up && m != -INFINITY ? fast_exp2(m - mx) : up ? 0.0f : 1.0f;
          if (up) m = mx;
          l *= alpha;
          if (i > 0) {
            W.wait(OREADY + x, ns - 1);
            tc::fence_after();
            scale_columns(tO, 0, D, alpha);
          }
        }
        const float me = m == -INFINITY ? 0.0f : m - kWeightShift;
        l += whole ? tile_weights<false>(tS, c0, me, bits, cs, ce)
                   : tile_weights<true>(tS, c0, me, bits, cs, ce);
        if (copies > 1) {  // the other copies' columns weigh nothing here
#pragma unroll 1
          for (int c = 0; c < 8; ++c)
            if (c < 2 * cs || c >= 2 * ce) tc::zero8(tS + 8 * c);
        }
        if (draft) {
          W.wait(VFULL + (n & 1u), n >> 1);  // V's marks; K's came with the scores
          const uint4 bk = lds128(smem + SM::BAD + 16 * (n & 3u)), bv = lds128(smem + SM::BAD + 16 * (4 + (n & 1u)));
          const uint4 bad = make_uint4(bk.x | bv.x, bk.y | bv.y, bk.z | bv.z, bk.w | bv.w);
          broken |= ((bad.x & bits.x) | (bad.y & bits.y) | (bad.z & bits.z) | (bad.w & bits.w)) != 0u;
        }
        tc::wait_st();
      }
      tc::fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(W.at(PREADY + x));
      ++ns;
    }
    base += nt;
    m -= kWeightShift;  // what the sum refers to
    if (broken) l = __uint_as_float(0x7fc00000u);

    // ---- this row's sum and output ----
    if (steps > 0) {
      W.wait(OREADY + x, ns - 1);
      tc::fence_after();
    }
    const int64_t unit = static_cast<int64_t>(s.b) * T.Hkv + s.kvh;
    const int64_t slot = 2 * static_cast<int64_t>(blockIdx.x) + (s.first ? 0 : 1);
    if (tid == 0) {
      int2 *at = P.shares + unit * P.blocks + (s.row0 >> 8);
      if (s.tile == 0) at->x = s.whole ? -1 : static_cast<int>(slot);
      if (s.last) at->y = static_cast<int>(blockIdx.x);
    }
    __nv_bfloat16 *out = static_cast<__nv_bfloat16 *>(T.out) + s.b * T.os[0] + head * T.os[1] +
                         node * T.os[2];
    float *part = T.ws_o + slot * D * WS_ROWS + row - s.row0;
    float inv;
    const float down = tc::pow2(-static_cast<int16_t>(vpower >> 16));
    if (two) {
      inv = l > 0.0f ? 1.0f / l : (l == l ? 0.0f : l);
#pragma unroll 1
      for (int col = 0; col < D && !idle; col += 32) {
        uint32_t o[32];
        float v[32];
        tc::ld32(tO + col, o);
        tc::wait_ld(o);
        // accumulator columns 8a.. hold dims 8a + (0,4,1,5,2,6,3,7)
#pragma unroll
        for (int e = 0; e < 32; ++e) v[(e & ~7) + ((e & 1) ? 4 : 0) + ((e & 7) >> 1)] = __uint_as_float(o[e]) * down;
        if (!ok) continue;
        if (s.whole) {
#pragma unroll
          for (int a = 0; a < 4; ++a) {
            const float *p = v + 8 * a;
            reinterpret_cast<uint4 *>(out + col)[a] =
                make_uint4(pack_bf16x2(p[0] * inv, p[1] * inv), pack_bf16x2(p[2] * inv, p[3] * inv),
                           pack_bf16x2(p[4] * inv, p[5] * inv), pack_bf16x2(p[6] * inv, p[7] * inv));
          }
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) part[(col + e) * WS_ROWS] = v[e];
        }
      }
    } else {
      // A row's pieces (two streams, `copies` each) meet in shared memory, 32
      // columns at a time: [piece][dim][row].  Thread t then holds row t mod RR
      // of RR / 8 dims.
      float2 *ml = reinterpret_cast<float2 *>(__cvta_shared_to_generic(smem + SM::ML));
      float *xch = reinterpret_cast<float *>(__cvta_shared_to_generic(smem + SM::Q));
      ml[tid] = make_float2(m, l);
      tc::fence_before();
      bar_softmax();  // all products are complete: Q may be overwritten
      tc::fence_after();
      float M = -INFINITY, total = 0.0f;
#pragma unroll 1
      for (int k = r & (RR - 1); k < 256; k += RR) M = fmaxf(M, ml[k].x);
      const float Me = M == -INFINITY ? 0.0f : M;
#pragma unroll 1
      for (int k = r & (RR - 1); k < 256; k += RR) total = fmaf(ml[k].y, exp2f(ml[k].x - Me), total);
      const float f = steps > 0 ? exp2f(m - Me) * down : 0.0f;
      m = M;
      l = total;
      inv = l > 0.0f ? 1.0f / l : (l == l ? 0.0f : l);
      float *mine = xch + (tid / RR) * 32 * RR + (r & (RR - 1));
      const int nd = RR / 8, d0 = tid / RR * nd;
#pragma unroll 1
      for (int col = 0; col < D; col += 32) {
        if (steps > 0) {
          uint32_t o[32];
          tc::ld32(tO + col, o);
          tc::wait_ld(o);
#pragma unroll
          for (int e = 0; e < 32; ++e)
            mine[((e & ~7) + ((e & 1) ? 4 : 0) + ((e & 7) >> 1)) * RR] = __uint_as_float(o[e]) * f;
        } else {  // a single tile is stream 0's alone
#pragma unroll 1
          for (int e = 0; e < 32; ++e) mine[e * RR] = 0.0f;
        }
        bar_softmax();
#pragma unroll 1
        for (int d = 0; d < nd; d += 4) {
          float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          const float *p = xch + (d0 + d) * RR + (r & (RR - 1));
#pragma unroll 2
          for (int k = 0; k < 2 * copies; ++k, p += 32 * RR) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] += p[e * RR];
          }
          if (!ok) continue;
          if (s.whole) {
            *reinterpret_cast<uint2 *>(out + col + d0 + d) =
                make_uint2(pack_bf16x2(v[0] * inv, v[1] * inv), pack_bf16x2(v[2] * inv, v[3] * inv));
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) part[(col + d0 + d + e) * WS_ROWS] = v[e];
          }
        }
        bar_softmax();
      }
    }
    if (ok && (two || tid < RR)) {
      if (!s.whole) {
        T.ws_ml[slot * WS_ROWS + row - s.row0] = make_float2(m, l);
      } else {
        if (T.stats) T.stats[unit * P.rows + row] = make_float2(m, inv);
        if (T.lse)
          T.lse[s.b * T.ls[0] + head * T.ls[1] + node * T.ls[2]] =
              l == 0.0f ? -INFINITY : (m + log2f(l)) * kBrLn2;
      }
    }
    tc::fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(W.at(QFREE));
  }
}

template <int D, int G>
__global__ void __launch_bounds__(THREADS, 1) tree_tc(const __grid_constant__ TcParams P) {
  using SM = Smem<D>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t smem = smem_u32(smem_raw);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Waiter W{smem + SM::BARS, smem + SM::MISC + 4};
  volatile int *start = reinterpret_cast<volatile int *>(smem_raw + SM::MISC + 8);
  griddep_launch_dependents();  // the merge may be set up: it waits for this grid's end
  if (smem & 1023u) {  // the swizzled tiles need 1024-byte alignment
    if (tid == 0) atomicOr(&g_branch_error_tc, DEV_ERR_MBAR_TIMEOUT);
    return;
  }
  if (warp == 9) {
    if (lane < NBARS) mbar_init(W.at(lane), bar_count(lane));
    fence_mbar_init();
    if (lane < 24) reinterpret_cast<uint32_t *>(smem_raw + SM::BAD)[lane] = 0u;
    if (lane == 0) *reinterpret_cast<volatile uint32_t *>(smem_raw + SM::MISC + 4) = 0u;
  }
  if (warp == 16) tc::alloc(smem + SM::MISC, 512);
  if (warp == 8) {
    // This CTA's share: all tiles of all units lie end to end, W / n of them for
    // each CTA and one more for the first W % n.  Sequences 32 at a time, by
    // prefix sums; work counts fit 31 bits (the host checks).
    const uint32_t per = static_cast<uint32_t>(P.t.Hkv * P.blocks), n = gridDim.x;
    uint32_t total = 0;
#pragma unroll 1
    for (int g = lane; g < P.t.B; g += 32)
      total += unit_tiles(P, g, blockIdx.x == 0 ? &g_branch_error_tc : nullptr);
    total = __reduce_add_sync(0xffffffffu, total) * per;
    const uint32_t each = total / n, rest = total - each * n;
    const uint32_t w0 = blockIdx.x * each + min(blockIdx.x, rest);
    uint32_t left = each + (blockIdx.x < rest ? 1u : 0u), b = 0, before = 0, T = 1;
    if (left > 0) {
#pragma unroll 1
      for (int g = 0;; g += 32) {
        const uint32_t t = g + lane < P.t.B ? unit_tiles(P, g + lane) : 0u;
        uint32_t sum = t * per;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint32_t y = __shfl_up_sync(0xffffffffu, sum, o);
          if (lane >= o) sum += y;
        }
        const uint32_t past = __ballot_sync(0xffffffffu, before + sum > w0);
        if (past || g + 32 >= P.t.B) {
          const int k = past ? __ffs(past) - 1 : 31;
          b = g + k;
          T = __shfl_sync(0xffffffffu, t, k);
          before += __shfl_sync(0xffffffffu, sum, k) - T * per;
          break;
        }
        before += __shfl_sync(0xffffffffu, sum, 31);
      }
    }
    if (lane == 0) {
      const uint32_t u = (w0 - before) / T, h = u / P.blocks;
      start[0] = static_cast<int>(left);
      start[1] = static_cast<int>(b);
      start[2] = static_cast<int>(h);
      start[3] = static_cast<int>(u - h * P.blocks);
      start[4] = static_cast<int>(w0 - before - u * T);
    }
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem =
      __shfl_sync(0xffffffffu, *reinterpret_cast<volatile uint32_t *>(smem_raw + SM::MISC), 0);
  const Walk walk{static_cast<uint32_t>(start[0]), start[1], start[2], start[3], start[4], true};
  // 128 * (2 * 96 + 2 * 104 + 80) = 640 * 96 registers.  Measured at 64 nodes x 16K
  // x 64 heads, batch 4, when it took 146 us: 148 with 104 / 88 / 96; sixteen dequantizing or
  // sixteen softmax warps (896 threads, two to a row there) spill: 160 and 154.
  if (warp < 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
    softmax_role<D>(P, walk, W, smem, tmem, tid);
  } else if (warp < 16) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
    dequant_role<D, G>(P, walk, W, smem, warp >= 12, tid & 127);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    if (warp == 16) mma_role<D>(P, walk, W, smem, tmem);
    else mask_role<D>(P, walk, W, smem, warp - 17, lane);
  }
  __syncwarp();
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (warp == 16) tc::dealloc(tmem, 512);
}

// Joins the partial rows of units that fell into several CTAs; units without
// any key get zeros.  A block takes 32 rows, a lane a row, a warp D / 8 columns.
// Four shares are in flight at a time (one block per SM as the launch bound: at
// the compiler's own choice of 40 registers the loads come one after another).
template <int D>
__global__ void __launch_bounds__(256, 1) tree_tc_merge(const __grid_constant__ TcParams P) {
  constexpr int C = D / 8;
  const TreeParams &T = P.t;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int kvh = blockIdx.y, b = blockIdx.z, row = blockIdx.x * 32 + lane;
  const int unit = b * T.Hkv + kvh;
  float m = -INFINITY, l = 0.0f, acc[C];
#pragma unroll
  for (int k = 0; k < C; ++k) acc[k] = 0.0f;
  griddep_wait();
  if (unit_tiles(P, b) > 0) {
    const int2 share = P.shares[unit * static_cast<int64_t>(P.blocks) + (blockIdx.x >> 3)];
    if (share.x < 0) return;  // written by its CTA
    // the unit is the first segment of every CTA after the one it began in
    constexpr int U = 4;  // shares in flight
#pragma unroll 1
    for (int c = share.x >> 1; c <= share.y; c += U) {
      float2 ml[U];
      float v[U][C];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = min(c + u, share.y);  // rows past the last read what nobody wrote and are dropped
        const int64_t slot = at == share.x >> 1 ? share.x : 2 * static_cast<int64_t>(at);
        ml[u] = T.ws_ml[slot * WS_ROWS + (row & 255)];
        const float *o = T.ws_o + (slot * D + warp * C) * WS_ROWS + (row & 255);
#pragma unroll
        for (int k = 0; k < C; ++k) v[u][k] = o[k * WS_ROWS];
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        // (past the last one: read again, and weighed with nothing)
        const float mu = c + u > share.y ? -INFINITY : ml[u].x;
        const float to = fmaxf(m, mu), base = to == -INFINITY ? 0.0f : to;
        const float f = exp2f(m - base), g = exp2f(mu - base);
        m = to;
        l = fmaf(l, f, g * ml[u].y);
#pragma unroll
        for (int k = 0; k < C; ++k) acc[k] = fmaf(acc[k], f, g * v[u][k]);
      }
    }
  }
  if (row >= P.rows) return;
  const int node = row / T.R, head = kvh * T.R + row - node * T.R;
  const float inv = l > 0.0f ? 1.0f / l : (l == l ? 0.0f : l);
  uint4 *o = reinterpret_cast<uint4 *>(static_cast<__nv_bfloat16 *>(T.out) + b * T.os[0] +
                                       head * T.os[1] + node * T.os[2] + warp * C);
#pragma unroll
  for (int k = 0; k < C; k += 8)
    o[k / 8] = make_uint4(pack_bf16x2(acc[k] * inv, acc[k + 1] * inv),
                          pack_bf16x2(acc[k + 2] * inv, acc[k + 3] * inv),
                          pack_bf16x2(acc[k + 4] * inv, acc[k + 5] * inv),
                          pack_bf16x2(acc[k + 6] * inv, acc[k + 7] * inv));
  if (warp == 0) {
    if (T.stats) T.stats[static_cast<int64_t>(unit) * P.rows + row] = make_float2(m, inv);
    if (T.lse)
      T.lse[b * T.ls[0] + head * T.ls[1] + node * T.ls[2]] =
          l == 0.0f ? -INFINITY : (m + log2f(l)) * kBrLn2;
  }
}

TcParams tc_plan(const TreeParams &T) {
  TcParams P{};
  P.t = T;
  P.rows = T.R * T.nodes;
  P.blocks = (P.rows + 255) / 256;
  P.dtiles = (T.ndraft + KT - 1) / KT;
  return P;
}

int64_t most_tiles(const TcParams &P) {
  return P.t.B * P.t.Hkv * P.blocks * ((P.t.S + KT - 1) / KT + P.dtiles);
}

int tc_ctas(const TcParams &P) {
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(sm_count(), most_tiles(P))));
}

template <int D, int G>
int launch_tc(const TcParams &P, int n, cudaStream_t st) {
  static bool configured[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = 0;
  if (!configured[dev]) {
    const int rc = cuda_status(cudaFuncSetAttribute(
        tree_tc<D, G>, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<D>::BYTES));
    if (rc) return rc;
    configured[dev] = true;
  }
  tree_tc<D, G><<<n, THREADS, Smem<D>::BYTES, st>>>(P);
  int rc = cuda_status(cudaGetLastError());
  if (rc) return rc;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>((P.rows + 31) / 32), static_cast<unsigned>(P.t.Hkv),
                     static_cast<unsigned>(P.t.B));
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, tree_tc_merge<D>, P));
}

}  // namespace

// Whether tree_tc takes the call: bf16 queries and scales (their products are
// exact in f16), the head sizes and groups it is built for, rows that 16-byte
// loads can read.  Everything else is branch.cu's.
bool tree_tc_takes(const TreeParams &T) {
  if (T.q_dtype != KV4_BF16 || T.s_dtype != KV4_BF16) return false;
  if (T.d != 64 && T.d != 128) return false;
  if (T.G != 16 && T.G != 32 && T.G != 64 && T.G != 128) return false;
  if (T.G > T.d) return false;
  if (!rows_ok(T.cache, T.B, T.Hkv, T.S) || !rows_ok(T.draft, T.B, T.Hkv, T.ndraft)) return false;
  if (!al16(T.q) || !al16(T.out) || T.qs[3] != 1 || T.os[3] != 1) return false;
  const int64_t n[3] = {T.B, static_cast<int64_t>(T.Hkv) * T.R, T.nodes};
  for (int i = 0; i < 3; ++i)
    if (n[i] > 1 && (T.qs[i] % 8 || T.os[i] % 8)) return false;
  return T.B < 65536 && T.Hkv < 65536 && most_tiles(tc_plan(T)) < (int64_t(1) << 31);
}

int64_t tree_tc_workspace(const TreeParams &T) {
  const TcParams P = tc_plan(T);
  return 2 * static_cast<int64_t>(tc_ctas(P)) * WS_ROWS * (static_cast<int64_t>(T.d) * 4 + 8) +
         T.B * T.Hkv * P.blocks * 8;
}

int tree_tc_run(TreeParams &T, void *workspace, int64_t bytes, cudaStream_t st) {
  if (!workspace || bytes < tree_tc_workspace(T)) return KV4_ERR_WORKSPACE;
  TcParams P = tc_plan(T);
  const int n = tc_ctas(P);
  P.t.ws_o = static_cast<float *>(workspace);
  P.t.ws_ml = reinterpret_cast<float2 *>(P.t.ws_o + 2 * static_cast<int64_t>(n) * WS_ROWS * T.d);
  P.shares = reinterpret_cast<int2 *>(P.t.ws_ml + 2 * static_cast<int64_t>(n) * WS_ROWS);
  if (T.d == 64) {
    switch (T.G) {
      case 16: return launch_tc<64, 16>(P, n, st);
      case 32: return launch_tc<64, 32>(P, n, st);
      default: return launch_tc<64, 64>(P, n, st);
    }
  }
  switch (T.G) {
    case 16: return launch_tc<128, 16>(P, n, st);
    case 32: return launch_tc<128, 32>(P, n, st);
    case 64: return launch_tc<128, 64>(P, n, st);
    default: return launch_tc<128, 128>(P, n, st);
  }
}

int branch_tc_take_device_error(int *v) {
  int zero = 0;
  int rc = cuda_status(cudaMemcpyFromSymbol(v, g_branch_error_tc, sizeof(int)));
  if (rc) return rc;
  return cuda_status(cudaMemcpyToSymbol(g_branch_error_tc, &zero, sizeof(int)));
}

}  // namespace kv4
