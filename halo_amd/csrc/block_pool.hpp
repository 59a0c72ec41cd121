// What the block-pool kernels share: pools, positions to blocks and rows.
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
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_or_zero(double v) {
  return __builtin_bit_cast(double, dpp_or_zero<CTRL, ROWS>(__builtin_bit_cast(int64_t, v)));
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
__device__ __forceinline__ double lane_of(double v, int lane) {
  return __builtin_bit_cast(double, lane_of(__builtin_bit_cast(int64_t, v), lane));
}

// A pool as the kernels address it.
struct PoolView {
  char* k;
  char* v;
  int64_t sl, sb, sh, sr;  // strides in bytes
  int layers, blocks, H_kv, D_bytes;
  Div bs;
};

template <int PB>
struct Piece;
template <>
struct Piece<16> {
  typedef __attribute__((ext_vector_type(4))) uint32_t type;
};
template <>
struct Piece<4> {
  typedef uint32_t type;
};
template <>
struct Piece<2> {
  typedef uint16_t type;
};

inline int check_pool(const halo_block_pool* pool, PoolView* out) {
  HALO_CHECK_ARG(pool && pool->k && pool->v, "null pool");
  HALO_CHECK_ARG(pool->dtype == HALO_F32 || pool->dtype == HALO_BF16 || pool->dtype == HALO_F16, "bad pool dtype");
  HALO_CHECK_ARG(pool->layers > 0 && pool->blocks > 0 && pool->H_kv > 0 && pool->block_size > 0 && pool->D > 0,
                 "pool sizes must be positive");
  HALO_CHECK_ARG((int64_t)pool->blocks * pool->block_size < (1ll << 31), "a pool holds at most 2^31 - 1 rows");
  const int64_t es = elem_size(pool->dtype);
  out->k = static_cast<char*>(pool->k);
  out->v = static_cast<char*>(pool->v);
  out->sl = pool->stride_l * es;
  out->sb = pool->stride_b * es;
  out->sh = pool->stride_h * es;
  out->sr = pool->stride_r * es;
  out->layers = pool->layers;
  out->blocks = pool->blocks;
  out->H_kv = pool->H_kv;
  out->D_bytes = (int)(pool->D * es);
  out->bs = make_div(pool->block_size);
  return HALO_OK;
}

// The widest piece that every row start is a multiple of.
inline int piece_bytes(const PoolView& p, uint64_t more) {
  const uint64_t all = reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v) | (uint64_t)p.sl |
                       (uint64_t)p.sb | (uint64_t)p.sh | (uint64_t)p.sr | (uint64_t)p.D_bytes | more;
  return all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 2;
}

}  // namespace halo
