// Joining the partial rows that key ranges of one (sequence, KV head) leave.
#pragma once

#include "branch.cuh"

namespace kv4 {

// how tree_generic's or tree_mma's work was cut; units = B * Hkv
struct GenPlan {
  int64_t units;
  int rows, row_tiles, parts, warps, ld;
  size_t smem;
};

// The run that tree_run makes of P (branch.cu); not for branch_tc.cu's kernel.
GenPlan tree_plan(const TreeParams &P);

// One warp joins row `at` of `parts` key ranges: ws_o [parts][rows][d]
// unnormalised, ws_ml [parts][rows] (base-2 maximum, sum).
template <int DC>
__device__ __forceinline__ void merge_row(const TreeParams &P, const GenPlan &L, int64_t at, int lane) {
  const int64_t n = L.units * L.rows;
  float m = -INFINITY, l = 0.0f, acc[DC];
#pragma unroll
  for (int k = 0; k < DC; ++k) acc[k] = 0.0f;
#pragma unroll 4
  for (int p = 0; p < L.parts; ++p) {
    const float2 ml = P.ws_ml[p * n + at];
    float v[DC];
#pragma unroll
    for (int k = 0; k < DC; ++k)
      v[k] = lane + 32 * k < P.d ? P.ws_o[(p * n + at) * P.d + lane + 32 * k] : 0.0f;
    const float to = fmaxf(m, ml.x), base = to == -INFINITY ? 0.0f : to;
    const float f = exp2f(m - base), g = exp2f(ml.x - base);
    m = to;
    l = fmaf(l, f, g * ml.y);
#pragma unroll
    for (int k = 0; k < DC; ++k) acc[k] = fmaf(acc[k], f, g * v[k]);
  }
  const int64_t unit = at / L.rows, b = unit / P.Hkv;
  const int row = static_cast<int>(at - unit * L.rows), i = row / P.R;
  const int h = static_cast<int>(unit - b * P.Hkv) * P.R + row - i * P.R;
  const float inv = l > 0.0f ? 1.0f / l : (l == l ? 0.0f : l);
#pragma unroll
  for (int k = 0; k < DC; ++k)
    if (lane + 32 * k < P.d)
      store_from_f32(P.out, P.q_dtype,
                     b * P.os[0] + h * P.os[1] + i * P.os[2] + (lane + 32 * k) * P.os[3],
                     acc[k] * inv);
  if (lane == 0) {
    if (P.stats) P.stats[at] = make_float2(m, inv);
    if (P.lse)
      P.lse[b * P.ls[0] + h * P.ls[1] + i * P.ls[2]] =
          l == 0.0f ? -INFINITY : (m + log2f(l)) * kBrLn2;
  }
}

}  // namespace kv4
