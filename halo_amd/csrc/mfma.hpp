// Matrix-core helpers of the prefill and tree attention kernels (gfx950): the
// 32x32x16 products of 16-bit operands, wave-uniform values, and the moves of
// their accumulator layout.
#pragma once

#include "common.hpp"

namespace halo {

typedef __attribute__((ext_vector_type(16))) float pf32x16;

template <int DT>
struct PMfma;
template <>
struct PMfma<HALO_BF16> {
  typedef __attribute__((ext_vector_type(8))) __bf16 v8;
  __device__ static __forceinline__ pf32x16 run(const uint4& a, const uint4& b, pf32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
  __device__ static __forceinline__ uint32_t pack(float a, float b) {
    typedef __attribute__((ext_vector_type(2))) __bf16 b2;
    const b2 v = {(__bf16)a, (__bf16)b};  // round to nearest even
    return __builtin_bit_cast(uint32_t, v);
  }
};
template <>
struct PMfma<HALO_F16> {
  typedef __attribute__((ext_vector_type(8))) _Float16 v8;
  __device__ static __forceinline__ pf32x16 run(const uint4& a, const uint4& b, pf32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
  __device__ static __forceinline__ uint32_t pack(float a, float b) {
    typedef __attribute__((ext_vector_type(2))) _Float16 h2;
    const h2 v = {(_Float16)a, (_Float16)b};  // round to nearest even
    return __builtin_bit_cast(uint32_t, v);
  }
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t prsrc(const char* base, int64_t bytes) {
  const int nrec = bytes <= 0 ? 0 : (bytes > 0x7fffffffLL ? 0x7fffffff : (int)bytes);
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, nrec, 0x00020000);
}

template <typename T>
__device__ __forceinline__ T uni(T v) {
  return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ int64_t uni64(int64_t v) {
  const uint64_t u = (uint64_t)v;
  return (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(u >> 32)) << 32) |
                   (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)u));
}
__device__ __forceinline__ const char* uniptr(const void* p) {
  return reinterpret_cast<const char*>((uintptr_t)uni64((int64_t)(uintptr_t)p));
}

// value of lane l ^ 32 next to the own value: {lanes 0-31 of v, lanes 32-63 of v}
__device__ __forceinline__ float half_max(float v) {
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float half_sum(float v) {
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

// ds_read_b64_tr_b16: within each 16-lane group, lane i receives element i%4
// of the 8-byte reads of lanes 4e + i/4 (e = 0..3).
typedef short pv4i16_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ uint2 pf_tr16(const char* p) {
  const pv4i16_t r = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) pv4i16_t*)(__attribute__((address_space(3))) char*)(p));
  return __builtin_bit_cast(uint2, r);
}

}  // namespace halo
