// Sums over neighbouring lanes of a wave.
#pragma once
#include <hip/hip_runtime.h>

namespace advoc {

// v of the lane that a data-parallel-primitive control names, within rows of 16 lanes
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float lane_value(float v, int lane) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
}

// Sum over groups of N consecutive lanes, in every lane of the group.  Within 16 lanes the partners come with the addition itself
// (eight cycles a step); a shuffle goes through LDS (over a hundred), and a row's sums are on the way of everything behind them.
template <int N>
__device__ __forceinline__ float lanes_sum(float v) {
  v += dpp<0xB1>(v);                       // quad_perm 1 0 3 2
  v += dpp<0x4E>(v);                       // quad_perm 2 3 0 1
  v += dpp<0x141>(v);                      // row_half_mirror: the other quad of eight
  if constexpr (N >= 16) v += dpp<0x140>(v);      // row_mirror: the other eight of sixteen
  if constexpr (N == 32) v += __shfl_xor(v, 16, 64);
  if constexpr (N == 64) v = (lane_value(v, 0) + lane_value(v, 16)) + (lane_value(v, 32) + lane_value(v, 48));
  return v;
}

}  // namespace advoc
