// dsa_lanes.h — sums over the lanes of a wave (gfx950) without a trip through LDS.
#pragma once

#include "dsa_common.h"

namespace dsa {
namespace hid {

// One data-parallel step of a sum over the lanes of a row of 16 (the
// instruction's own lane patterns: no trip through LDS).
template <int CTRL>
DSA_DEV float dpp(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
DSA_DEV float lane_value(float x, int lane) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), lane));
}
// The sum of x over each L neighbouring lanes, in a fixed order, in every lane.
template <int L>
DSA_DEV float lanes_sum(float x) {
  static_assert(L == 16 || L == 32 || L == 64, "");
  x += dpp<0xB1>(x);   // quad_perm [1, 0, 3, 2]
  x += dpp<0x4E>(x);   // quad_perm [2, 3, 0, 1]
  x += dpp<0x141>(x);  // row_half_mirror: the other quad of eight lanes
  x += dpp<0x140>(x);  // row_mirror: the other eight of sixteen
  if constexpr (L == 32) x += __shfl_xor(x, 16);
  if constexpr (L == 64) x = (lane_value(x, 0) + lane_value(x, 16)) + (lane_value(x, 32) + lane_value(x, 48));
  return x;
}

}  // namespace hid
}  // namespace dsa
