// wave.hpp — exchanges and sums over the 64 lanes of a wave with vector
// operations only: no LDS round trips (a ds_bpermute costs ~130 cycles before
// its result can be used, and a sum needs six of them in a row).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mlxq {

// The value of the lane whose number differs in bit J: vector operations only
// (4 is 3 then 7; halves and rows of 16 are swapped between two registers).
template <int J>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v, int lane) {
  if constexpr (J == 1) return __builtin_amdgcn_mov_dpp(v, 0xB1, 0xF, 0xF, false);
  else if constexpr (J == 2) return __builtin_amdgcn_mov_dpp(v, 0x4E, 0xF, 0xF, false);
  else if constexpr (J == 4)
    return __builtin_amdgcn_mov_dpp(__builtin_amdgcn_mov_dpp(v, 0x1B, 0xF, 0xF, false), 0x141, 0xF, 0xF, false);
  else if constexpr (J == 8) return __builtin_amdgcn_mov_dpp(v, 0x128, 0xF, 0xF, false);
  else if constexpr (J == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return lane & 16 ? r[0] : r[1];
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return lane & 32 ? r[0] : r[1];
  }
}
template <int J>
__device__ __forceinline__ float lane_xor(float v, int lane) {
  return __uint_as_float(lane_xor<J>(__float_as_uint(v), lane));
}

// Over all lanes, the same in each.
__device__ __forceinline__ float wave_sum(float v, int lane) {
  v += lane_xor<1>(v, lane);
  v += lane_xor<2>(v, lane);
  v += lane_xor<4>(v, lane);
  v += lane_xor<8>(v, lane);
  v += lane_xor<16>(v, lane);
  return v + lane_xor<32>(v, lane);
}
__device__ __forceinline__ float wave_max(float v, int lane) {
  v = fmaxf(v, lane_xor<1>(v, lane));
  v = fmaxf(v, lane_xor<2>(v, lane));
  v = fmaxf(v, lane_xor<4>(v, lane));
  v = fmaxf(v, lane_xor<8>(v, lane));
  v = fmaxf(v, lane_xor<16>(v, lane));
  return fmaxf(v, lane_xor<32>(v, lane));
}

}  // namespace mlxq
