// What the matrix-core decode kernels (decode_mfma.hip, decode8.hip) share.
#pragma once

#include "pa_common.hpp"

namespace pa {

typedef float f32x4m __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8m __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8m __attribute__((ext_vector_type(8)));
typedef unsigned int u32x4m __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2m __attribute__((ext_vector_type(2)));

template <typename T>
__device__ __forceinline__ f32x4m mfma16(u32x4m a, u32x4m b, f32x4m c);
template <>
__device__ __forceinline__ f32x4m mfma16<bf16_t>(u32x4m a, u32x4m b, f32x4m c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8m, a), __builtin_bit_cast(bf16x8m, b), c,
                                                 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x4m mfma16<f16_t>(u32x4m a, u32x4m b, f32x4m c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8m, a), __builtin_bit_cast(f16x8m, b), c, 0,
                                                0, 0);
}

// NT: streaming loads, for rows no other workgroup reads.
template <typename V, bool NT>
__device__ __forceinline__ V row_load(const void* p) {
  if constexpr (NT) return __builtin_nontemporal_load(reinterpret_cast<const V*>(p));
  return *reinterpret_cast<const V*>(p);
}

}  // namespace pa
