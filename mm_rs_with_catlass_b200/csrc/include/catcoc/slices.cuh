// Attention whose keys are cut into slices: the merge of a row's pieces, for the kernels that leave them (flash_attn.cu, window_attn.cu).
#pragma once
#include <cstdint>
#include "catcoc/ptx.cuh"
#include "catcoc/softmax_row.cuh"

namespace catcoc {
namespace attn {

// The slices of a row, a warp each; every row has a slice that it sees something of unless it sees nothing at all. A slice of which
// the row sees nothing is left out, not weighed with zero: its piece is zero times values that the row's tile may not see either, where
// an infinity makes a NaN. (A sum that is not zero, a NaN, is no such slice.)
template <int D, int FMT>
__global__ void __launch_bounds__(128) flash_slices_kernel(const float* part_o, const float* part_ml, void* out, int64_t rows, int slices) {
  constexpr int kPer = D / 32;                     // columns per lane
  const int64_t r = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  ptx::grid_dependency_wait();
  if (r >= rows) return;
  const float2 ml = lane < slices ? *reinterpret_cast<const float2*>(part_ml + (lane * rows + r) * 2) : make_float2(-INFINITY, 0.0f);
  float mx = ml.x;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  const float w = ml.x == -INFINITY ? 0.0f : ptx::ex2_approx(ml.x - mx);
  const uint32_t seen = __ballot_sync(0xffffffffu, !(ml.x == -INFINITY && ml.y == 0.0f));
  float l = w * ml.y, acc[kPer];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
#pragma unroll
  for (int e = 0; e < kPer; ++e) acc[e] = 0.0f;
#pragma unroll 4
  for (int c = 0; c < slices; ++c) {
    const float wc = __shfl_sync(0xffffffffu, w, c);
    const float* src = part_o + (c * rows + r) * D + lane * kPer;
    float o[kPer] = {};
    if ((seen >> c) & 1u) {
      if constexpr (kPer == 4) *reinterpret_cast<float4*>(o) = *reinterpret_cast<const float4*>(src);
      else *reinterpret_cast<float2*>(o) = *reinterpret_cast<const float2*>(src);
    }
#pragma unroll
    for (int e = 0; e < kPer; ++e) acc[e] += wc * o[e];
  }
  const float inv = l > 0.0f ? 1.0f / l : 0.0f;
  uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(out) + (r * D + lane * kPer) * 2);
#pragma unroll
  for (int e = 0; e < kPer / 2; ++e) dst[e] = pack16<FMT>(acc[2 * e] * inv, acc[2 * e + 1] * inv);
}

}  // namespace attn
}  // namespace catcoc
