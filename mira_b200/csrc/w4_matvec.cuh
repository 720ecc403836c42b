// Products of a few rows with 4-bit weights under group scales:
//   y[m, n] = steps(sum_g s[n, g] sum_{k in g} x[m, k] (w[n, k] - 8)).
#pragma once
#include <cstdint>

#include "paged_kv.cuh"

namespace mira {

struct W4Params {
  const void* x;
  const uint8_t* w;
  const void* scales;
  void* out;
  int64_t ld_x, ld_w, ld_scales, ld_out;
  int m, n, k, group;
  int x_dtype, scale_dtype, out_dtype;
  int n_steps;
  mira_epi_step steps[MIRA_EPI_MAX_STEPS];
};

// The epilogue steps on one f32 result.
__device__ __forceinline__ float w4_steps(const W4Params& p, float y, int m, int n) {
  for (int s = 0; s < p.n_steps; ++s) {
    const mira_epi_step& st = p.steps[s];
    if (st.operand == MIRA_OPND_NONE) {
      y = apply_unary(st.op, y);
      continue;
    }
    float o = st.scalar;
    if (st.operand == MIRA_OPND_CHANNEL) o = __ldg(st.ptr + n);
    else if (st.operand == MIRA_OPND_ROW) o = __ldg(st.ptr + m);
    else if (st.operand == MIRA_OPND_FULL) o = __ldg(st.ptr + int64_t(m) * st.ld + n);
    y = st.swapped ? apply_binary(st.op, o, y) : apply_binary(st.op, y, o);
  }
  return y;
}

constexpr int W4_WARPS = 8;
constexpr int W4_ROWS = 4;     // rows of x per pass over the weights

// One warp per weight row: lanes stride over words of eight weights, each group's sum is scaled once.
__global__ void __launch_bounds__(W4_WARPS * 32) w4_matvec_kernel(const __grid_constant__ W4Params p) {
  const int lane = threadIdx.x & 31;
  const int n = blockIdx.x * W4_WARPS + (threadIdx.x >> 5);
  if (n >= p.n) return;
  for (int m0 = blockIdx.y * W4_ROWS; m0 < p.m; m0 += gridDim.y * W4_ROWS) {
    float acc[W4_ROWS] = {};
    const int words = (p.k + 7) / 8;
    for (int j = lane; j < words; j += 32) {
      const uint32_t w = __ldg(reinterpret_cast<const uint32_t*>(p.w + n * p.ld_w) + j);
      const float s = dt_load(p.scales, n * p.ld_scales + j * 8 / p.group, p.scale_dtype);
#pragma unroll
      for (int r = 0; r < W4_ROWS; ++r) {
        if (m0 + r >= p.m) break;
        float part = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int k = j * 8 + e;
          if (k < p.k)
            part = fmaf(dt_load(p.x, (m0 + r) * p.ld_x + k, p.x_dtype), float(int((w >> (4 * e)) & 15) - 8), part);
        }
        acc[r] = fmaf(part, s, acc[r]);
      }
    }
#pragma unroll
    for (int r = 0; r < W4_ROWS; ++r) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) acc[r] += __shfl_xor_sync(0xffffffffu, acc[r], o);
      if (lane == 0 && m0 + r < p.m)
        dt_store(p.out, (m0 + r) * p.ld_out + n, p.out_dtype, w4_steps(p, acc[r], m0 + r, n));
    }
  }
}

}  // namespace mira
