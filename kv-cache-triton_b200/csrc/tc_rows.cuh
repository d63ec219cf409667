// Packed rows and queries on their way to tensor-core tiles, shared by the
// tcgen05 kernels of branch_tc.cu and trim_tc.cu.
#pragma once

#include "branch.cuh"
#include "tc.cuh"

namespace kv4 {
namespace {

__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float &a, float &b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// 16 bytes global -> shared, zeros instead of the source bytes past `n`
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, uint32_t n) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// A thread's place in the packed rows of K or V: its 16-byte chunk and its
// scales in one row, and how far (bytes; elements) the row of its next chunk is.
struct Source {
  const uint8_t *p;
  const uint16_t *s;
  int pst, sst;
};

template <int D, int G, int THREADS>
__device__ __noinline__ Source source_of(const TreeParams &T, bool draft, bool v, int b, int h, int row,
                                         int c) {
  constexpr int RSTEP = THREADS / (D / 32);
  const RowSource &S = draft ? T.draft : T.cache;
  const int64_t *ps = v ? S.vps : S.kps, *ss = v ? S.vss : S.kss;
  Source o;
  o.p = (v ? S.vp : S.kp) + b * ps[0] + h * ps[1] + row * ps[2] + 16 * c;
  o.s = static_cast<const uint16_t *>(v ? S.vs : S.ks) + b * ss[0] + h * ss[1] + row * ss[2] + c * 32 / G;
  o.pst = static_cast<int>(ps[2]) * RSTEP;
  o.sst = static_cast<int>(ss[2]) * RSTEP;
  return o;
}

// Which 16-byte chunk (32 codes) of which row a thread takes: eight neighbouring
// lanes hold two chunks of four rows that share a 64-element panel, so that
// their 16-byte stores fall into eight different columns of the swizzle.
template <int D>
struct Chunk {
  static constexpr int CPR = D / 32;  // chunks per row
  int row, c;
  // of the four warps that take a tile, the one that row r is with
  static __device__ __forceinline__ int warp_of(int r) { return (D == 128 ? r >> 3 : r >> 4) & 3; }
  __device__ __forceinline__ explicit Chunk(int tid) {
    const int lane = tid & 31;
    if (D == 128) {
      c = (lane & 1) | ((lane >> 2) & 2);
      row = (tid >> 5) * 8 + ((lane >> 1) & 3) + ((lane >> 2) & 4);
    } else {
      c = lane & 1;
      row = tid >> 1;
    }
  }
};

// Chunk c of row `row` of a K or V tile, dequantized.
template <int D, int NS>
__device__ __forceinline__ void store_chunk(uint32_t tile, int row, int c, const uint4 &w,
                                            const uint32_t (&scale)[NS]) {
  const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
  const uint32_t at = tile + (c >> 1) * tc::PANEL + row * 128;
  const uint32_t col = ((c & 1) * 4) ^ (row & 7);  // 16-byte column of the chunk's first word
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t v[4];
    tc::dequant_word(ws[j], scale[NS == 2 ? j >> 1 : 0], v);
    tc::sts128(at + ((col ^ j) << 4), v[0], v[1], v[2], v[3]);
  }
}

// Row `row` of a KV head's queries (row = node * R + head of the group) as f16
// in row r of a tile, times the power of two that brings its largest element to
// [2^13, 2^14): copied as it is to its place in shared memory (D / 8 lanes a
// row), then converted there by its own thread.  The calling warp holds 32
// consecutive rows, r = 0 mod 32 in lane 0; rows at or past `rows` become
// zeros.  Returns the factor from scores to base-2 exponents.
template <int D>
__device__ __forceinline__ float load_query_row(const TreeParams &T, int rows, int b, int kvh,
                                                int row, uint32_t tile, int r) {
  constexpr int LPR = D / 8, RPI = 32 / LPR;  // lanes per row, rows at a time
  const int lane = threadIdx.x & 31;
  {
    const int k = lane % LPR, rl = lane / LPR, first = row - lane;
    const __nv_bfloat16 *q = static_cast<const __nv_bfloat16 *>(T.q) + b * T.qs[0] +
                             static_cast<int64_t>(kvh * T.R) * T.qs[1] + 8 * k;
    const int dn = RPI / T.R, dh = RPI - dn * T.R;
    const int qn = (first + rl) / T.R;
    int qh = first + rl - qn * T.R;  // head of this lane's row
    const __nv_bfloat16 *p = q + qh * T.qs[1] + qn * T.qs[2];
    const int64_t step = dh * T.qs[1] + dn * T.qs[2], wrap = T.qs[2] - T.R * T.qs[1];
    const uint32_t to = tile + (k >> 3) * tc::PANEL + (r & ~31) * 128;
#pragma unroll 4
    for (int g = rl; g < 32; g += RPI) {
      const bool in = first + g < rows;
      cp_async16(to + g * 128 + (((k & 7) ^ (g & 7)) << 4), in ? p : static_cast<const __nv_bfloat16 *>(T.q),
                 in ? 16u : 0u);
      p += step;
      qh += dh;
      if (qh >= T.R) {
        qh -= T.R;
        p += wrap;
      }
    }
    cp_async_wait_all();
    __syncwarp();
  }
  uint32_t top2 = 0;  // largest |q| as bits: bf16 magnitudes order like integers
#pragma unroll 4
  for (int k = 0; k < D / 8; ++k) {
    const uint4 w = lds128(tile + tc::tile_off(r, k));
    top2 = __vmaxu2(top2, __vmaxu2(__vmaxu2(w.x & 0x7FFF7FFFu, w.y & 0x7FFF7FFFu),
                                   __vmaxu2(w.z & 0x7FFF7FFFu, w.w & 0x7FFF7FFFu)));
  }
  const uint32_t top = max(top2 & 0xFFFFu, top2 >> 16);
  int ex = 13 - (static_cast<int>(top >> 7) - 127);
  ex = top == 0 ? 0 : min(max(ex, -126), 126);
  const float up = __uint_as_float(static_cast<uint32_t>(ex + 127) << 23);
#pragma unroll 4
  for (int k = 0; k < D / 8; ++k) {
    const uint32_t at = tile + tc::tile_off(r, k);
    const uint4 w = lds128(at);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
    float f[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f[2 * e] = bf16lo_to_f32(u[e]) * up;
      f[2 * e + 1] = bf16hi_to_f32(u[e]) * up;
    }
    tc::sts128(at, pack_f16x2(f[0], f[4]), pack_f16x2(f[1], f[5]), pack_f16x2(f[2], f[6]),
               pack_f16x2(f[3], f[7]));
  }
  return T.scale_log2 * __uint_as_float(static_cast<uint32_t>(127 - ex) << 23);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
inline bool al16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

inline bool rows_ok(const RowSource &S, int64_t B, int Hkv, int64_t T) {
  if (T == 0) return true;
  if (!al16(S.kp) || !al16(S.vp)) return false;
  for (const int64_t *st : {S.kps, S.vps}) {
    if (st[3] != 1 || st[2] % 16 || (Hkv > 1 && st[1] % 16) || (B > 1 && st[0] % 16)) return false;
    if (st[2] < 0 || st[2] >= (1 << 20)) return false;  // 64 of them fit 32 bits
  }
  for (const int64_t *st : {S.kss, S.vss})
    if (st[3] != 1 || st[2] < 0 || st[2] >= (1 << 20)) return false;
  return true;
}

inline int sm_count() {
  static int n[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (!n[dev]) {
    int v = 0;
    if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || v <= 0)
      v = 148;
    n[dev] = v;
  }
  return n[dev];
}

}  // namespace
}  // namespace kv4
