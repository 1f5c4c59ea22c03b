// Sums over the lanes of a power-of-two group by lane moves in the vector
// registers: __shfl_xor goes through the LDS crossbar (~100 cycles a step),
// these stay in the ALU (~8).  Every lane of the group gets the group's sum,
// added in the same order whatever the lane.
#pragma once

#include <hip/hip_runtime.h>

namespace st {

template <int CTRL>
__device__ __forceinline__ float dpp_move(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
// v of the lane 16 (32) away, by swapping odd rows of one copy with even rows of another
__device__ __forceinline__ float other_row(float v) {
  const unsigned u = __builtin_bit_cast(unsigned, v);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return __builtin_bit_cast(float, (threadIdx.x & 16) ? r[0] : r[1]);
}
__device__ __forceinline__ float other_half(float v) {
  const unsigned u = __builtin_bit_cast(unsigned, v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __builtin_bit_cast(float, (threadIdx.x & 32) ? r[0] : r[1]);
}

// Sum over groups of LANES (2..64) consecutive lanes.
template <int LANES>
__device__ __forceinline__ float group_sum(float v) {
  if constexpr (LANES >= 2) v += dpp_move<0xB1>(v);   // quad_perm [1,0,3,2]
  if constexpr (LANES >= 4) v += dpp_move<0x4E>(v);   // quad_perm [2,3,0,1]
  if constexpr (LANES >= 8) v += dpp_move<0x141>(v);  // row_half_mirror: the other four of eight
  if constexpr (LANES >= 16) v += dpp_move<0x140>(v); // row_mirror: the other eight of sixteen
  if constexpr (LANES >= 32) v += other_row(v);
  if constexpr (LANES >= 64) v += other_half(v);
  return v;
}

}  // namespace st
