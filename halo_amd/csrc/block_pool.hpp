// What the block-pool kernels share: positions to blocks and rows.
#pragma once

#include "common.hpp"

namespace halo {

// x / d for 0 <= x < 2^31 by one product: with 2^(s-1) < d <= 2^s and M =
// ceil(2^(31+s) / d), M d - 2^(31+s) < 2^s, so x M / 2^(31+s) is above x / d by
// less than 1 / d and has the same whole part.  d = 1 has no such M below 2^32.
struct Div {
  int d;
  uint32_t mul, shift, one;
};
inline Div make_div(int d) {
  if (d == 1) return {1, 0, 0, 0xffffffffu};
  uint32_t s = 1;
  while ((1ll << s) < d) ++s;
  return {d, (uint32_t)(((1ull << (31 + s)) + d - 1) / d), s - 1, 0};
}
__device__ __forceinline__ int div_by(int x, Div v) {
  return (int)((__umulhi((uint32_t)x, v.mul) >> v.shift) | ((uint32_t)x & v.one));
}

// Inclusive sums over the 64 lanes, in registers.
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_or_zero(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_or_zero(float v) {
  return __int_as_float(dpp_or_zero<CTRL, ROWS>(__float_as_int(v)));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ int64_t dpp_or_zero(int64_t v) {
  const uint32_t lo = (uint32_t)dpp_or_zero<CTRL, ROWS>((int)(uint32_t)v);
  return (int64_t)(((uint64_t)(uint32_t)dpp_or_zero<CTRL, ROWS>((int)(v >> 32)) << 32) | lo);
}
template <typename T>
__device__ __forceinline__ T wave_prefix(T v) {
  v += dpp_or_zero<0x111, 0xf>(v);  // row_shr 1, 2, 4, 8: within 16 lanes
  v += dpp_or_zero<0x112, 0xf>(v);
  v += dpp_or_zero<0x114, 0xf>(v);
  v += dpp_or_zero<0x118, 0xf>(v);
  v += dpp_or_zero<0x142, 0xa>(v);  // lane 15 of each row to the row behind it
  v += dpp_or_zero<0x143, 0xc>(v);  // lane 31 to the upper half
  return v;
}

// The value of one lane, the same for all.
__device__ __forceinline__ int lane_of(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
__device__ __forceinline__ float lane_of(float v, int lane) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
}
__device__ __forceinline__ int64_t lane_of(int64_t v, int lane) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
  return (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32) | lo);
}

}  // namespace halo
