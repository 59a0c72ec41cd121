// What the block-pool kernels share: positions to blocks and rows.
#pragma once

#include "common.hpp"

namespace halo {

// x / d and x % d for 0 <= x < 2^31; `shift` >= 0 where d is a power of two.
struct Div {
  int d, shift;
};
inline Div make_div(int d) {
  int s = -1;
  if ((d & (d - 1)) == 0)
    for (s = 0; (1 << s) < d; ++s) {
    }
  return {d, s};
}
__device__ __forceinline__ int div_by(int x, Div v) {
  return v.shift >= 0 ? x >> v.shift : (int)((uint32_t)x / (uint32_t)v.d);
}

}  // namespace halo
