// tcgen05 / tensor-memory wrappers of the branch and trim kernels (sm_100a).
#pragma once

#include "common.cuh"

namespace kv4 {
namespace tc {

constexpr int PANEL = 128 * 128;  // 128 rows of a 64-element-wide 16-bit panel (bytes)

__device__ __forceinline__ void fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_smem() {  // generic writes before tensor-core reads
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// Shared-memory matrix descriptor, 128-byte swizzle, version 1: `lbo` is the
// distance of 64-element panels of an MN-major operand, `sbo` of 8-row groups.
__device__ __forceinline__ uint64_t desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
  return static_cast<uint64_t>((addr & 0x3FFFFu) >> 4) |
         (static_cast<uint64_t>(lbo >> 4) << 16) | (static_cast<uint64_t>(sbo >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}

// Instruction descriptor: f32 accumulators, f16 A and B, M = 128, A K-major,
// B K-major or (mn) MN-major, N columns.
__host__ __device__ constexpr uint32_t idesc(uint32_t n, bool mn) {
  return (1u << 4) | ((mn ? 1u : 0u) << 16) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}

// One lane of a converged warp.  The issuing warp runs its loops converged and
// elects the lane only around the instructions themselves, so that descriptors
// stay in uniform registers: issued from a one-lane branch, each product of
// the tree kernel took about 250 cycles to get out, four times its run time.
__device__ __forceinline__ uint32_t elect() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(p));
  return p;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(id), "r"(acc)
      : "memory");
}
// A from tensor memory: rows on the lanes, pairs of 16-bit K values per column
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(id), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
      : "memory");
}

__device__ __forceinline__ void alloc(uint32_t slot, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot),
               "r"(cols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void dealloc(uint32_t tmem, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols)
               : "memory");
}

// 32 consecutive columns of this thread's lane; wait_ld() before use
__device__ __forceinline__ void ld32(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
      "%11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, "
      "%28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr)
      : "memory");
}
// the loads issued so far have landed in r (tying r keeps its uses behind the wait)
__device__ __forceinline__ void wait_ld(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                 "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                 "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]),
                 "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                 "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}
__device__ __forceinline__ void ld16(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
      "%11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void wait_ld16(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                 "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                 "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}
__device__ __forceinline__ void st16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
      "%11, %12, %13, %14, %15, %16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void st32(uint32_t addr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
      "%11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, "
      "%28, %29, %30, %31, %32};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
      "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
      "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void st8(uint32_t addr, const uint32_t (&r)[8]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
      : "memory");
}
__device__ __forceinline__ void zero8(uint32_t addr) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %1, %1, %1, %1, %1, %1, %1};" ::"r"(addr),
      "r"(0u)
      : "memory");
}
__device__ __forceinline__ void wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// byte offset of 16-byte chunk c of row r in a tile of 128 rows of 64-element
// panels, 128-byte swizzle
__device__ __forceinline__ uint32_t tile_off(int r, int c) {
  return static_cast<uint32_t>((c >> 3) * PANEL + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

__device__ __forceinline__ void sts128(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d)
               : "memory");
}

__device__ __forceinline__ uint32_t hsub2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// what a * b loses when it is rounded to p (exact above the subnormals)
__device__ __forceinline__ uint32_t hrest2(uint32_t a, uint32_t b, uint32_t p) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(p ^ 0x80008000u));
  return r;
}
// f16 pair (1024 + code) of nibbles 0 and 4 of x
__device__ __forceinline__ uint32_t nib_pair(uint32_t x) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(x), "r"(0x000F000Fu), "r"(0x64006400u));
  return r;
}

// Eight codes of a packed word times a scale (f16, in both halves), in the dim
// order 0,4,1,5,2,6,3,7: (1024 + code) - 1032 is exact, and so is the product
// of a 4-bit code and a bf16 scale's 8 significant bits (in the range below).
__device__ __forceinline__ void dequant_word(uint32_t w, uint32_t scale, uint32_t (&v)[4]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = hmul2(hsub2(nib_pair(w >> (4 * e)), 0x64086408u), scale);
}

// ---- bf16 scales in f16 operands ----
// A scale of 8 significant bits times a code is exact in f16 while the scale lies
// in [2^-17, 2^12): f16 steps by 2^-24 at its lower end, and 8 * 2^12 is below its
// upper.  Scales elsewhere are first multiplied by a power of two 2^e, the same
// for all scales of a key tile (or of a warp's step), and the fp32 sums that they
// go into by 2^-e: with the largest brought to [2^10, 2^11), all down to 2^-27 of
// it are exact.  e = 0 while all lie in that range as they are.
constexpr uint32_t kExactLo = 110u << 7, kExactSpan = 29u << 7;  // bits of 2^-17; of 2^-17 .. 2^12
constexpr uint32_t kUsableEnd = 227u << 7;                       // 2^100: a larger scale is reported, not used
constexpr int kMaxShift = 96;

__device__ __forceinline__ uint32_t scale_bits(uint32_t bf) { return bf & 0x7FFFu; }  // |scale|, ordered
__device__ __forceinline__ bool scale_usable(uint32_t bits) { return bits < kUsableEnd; }
__device__ __forceinline__ bool scale_exact(uint32_t bits) {
  return bits == 0u || bits - kExactLo < kExactSpan;
}
// Whether some of N scales are not exact as they are.
template <int N>
__device__ __forceinline__ bool scales_odd(const uint16_t (&x)[N]) {
  uint32_t lo = 0xFFFFFFFFu, hi = 0;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    lo = min(lo, scale_bits(x[k]) - 1u);  // zeros last
    hi = max(hi, scale_bits(x[k]));
  }
  return lo < kExactLo - 1u || hi >= kExactLo + kExactSpan;
}
// A warp's largest usable scale (bits), and bit 15 where some are not exact.
template <int N>
__device__ __forceinline__ uint32_t scales_top(const uint16_t (&x)[N]) {
  uint32_t top = 0;
  bool exact = true;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const uint32_t u = scale_bits(x[k]);
    exact = exact && scale_exact(u);
    if (scale_usable(u)) top = max(top, u);
  }
  return __reduce_max_sync(0xffffffffu, top) | (__all_sync(0xffffffffu, exact) ? 0u : 0x8000u);
}
// 2^e for e <= 127; 0 below the normal numbers
__device__ __forceinline__ float pow2(int e) {
  return __uint_as_float(static_cast<uint32_t>(max(e + 127, 0)) << 23);
}
// e for the largest usable scale (as bits)
__device__ __forceinline__ int scale_shift(uint32_t top) {
  return min(10 + 127 - static_cast<int>(top >> 7), kMaxShift);
}
// a bf16 scale times 2^e (exact); one that is not usable becomes infinite
__device__ __forceinline__ uint16_t scale_shifted(uint16_t bf, float up) {
  if (!scale_usable(scale_bits(bf))) return 0x7F80u;
  return static_cast<uint16_t>(__float_as_uint(__uint_as_float(static_cast<uint32_t>(bf) << 16) * up) >> 16);
}
// a bf16 scale as f16 in both halves; an infinite one stays so
__device__ __forceinline__ uint32_t scale_pair(uint16_t bf) {
  const uint32_t h = __half_as_ushort(__float2half_rn(__uint_as_float(static_cast<uint32_t>(bf) << 16)));
  return h | (h << 16);
}
// barrier `id` of 128 threads (whole warps); true where `p` is for any of them
__device__ __forceinline__ bool barrier_any(int id, bool p) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %2, 0;\n\t"
      "bar.red.or.pred q, %1, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(id), "r"(p ? 1u : 0u)
      : "memory");
  return r != 0u;
}

}  // namespace tc
}  // namespace kv4
