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

}  // namespace halo
