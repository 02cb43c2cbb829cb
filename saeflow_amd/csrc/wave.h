// Sums over a wavefront's 64 lanes.
#pragma once

#include <hip/hip_runtime.h>

// Sum of v over the wave, returned in every lane, with DPP moves (VALU) instead of LDS
// permutes: xor-1 and xor-2 within quads, the half-row and row mirrors give each 16-lane row
// its total, row_bcast:15 / row_bcast:31 carry row totals upward, lane 63 ends with the sum.
template <int CTRL, int ROW_MASK>
__device__ __forceinline__ float dpp_add(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, ROW_MASK, 0xF, false));
}
__device__ __forceinline__ float wave_sum(float v) {
  v = dpp_add<0xB1, 0xF>(v);   // quad_perm [1,0,3,2]
  v = dpp_add<0x4E, 0xF>(v);   // quad_perm [2,3,0,1]
  v = dpp_add<0x141, 0xF>(v);  // row_half_mirror
  v = dpp_add<0x140, 0xF>(v);  // row_mirror
  v = dpp_add<0x142, 0xA>(v);  // row_bcast:15 into rows 1 and 3
  v = dpp_add<0x143, 0xC>(v);  // row_bcast:31 into rows 2 and 3
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// What v_permlane32_swap_b32 and v_permlane16_swap_b32 leave of a and b, added: of a in the lower 32 lanes (the even rows of
// 16 lanes) each lane's value plus that of the lane 32 (16) above, of b the same in the others.
template <int LANES>
__device__ __forceinline__ float swap_add(float a, float b) {
  static_assert(LANES == 32 || LANES == 16, "");
  const auto r = LANES == 32 ? __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false)
                             : __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Wave sums of 8 values at once: afterwards every lane l holds the total of v[(l >> 3) & 7].
// A reduce-scatter: each of three exchanges (lanes 32, 16 and 8 apart) keeps half of the values
// a lane still carries and adds its partner's copy of that half, then DPP moves sum the 8-lane
// groups (quads, then the half-row mirror). The first two are swaps of register halves, so no value is
// selected and none goes through LDS (against 7 permutes: the backward pass over the features of 1000 tokens x 1000 x
// 10007 features in fp16 41 -> 38 us).
__device__ __forceinline__ float wave_sum8(const float (&v)[8], int lane) {
  float w[4], x[2];
#pragma unroll
  for (int k = 0; k < 4; ++k) w[k] = swap_add<32>(v[k], v[k + 4]);
#pragma unroll
  for (int k = 0; k < 2; ++k) x[k] = swap_add<16>(w[k], w[k + 2]);
  const bool b3 = lane & 8;
  float y = b3 ? x[1] : x[0];
  y += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(b3 ? x[0] : x[1]), 0x128, 0xF, 0xF, false));  // row_ror:8
  y = dpp_add<0xB1, 0xF>(y);   // quad_perm [1,0,3,2]
  y = dpp_add<0x4E, 0xF>(y);   // quad_perm [2,3,0,1]
  return dpp_add<0x141, 0xF>(y);  // row_half_mirror: the other quad of the 8-lane group
}
