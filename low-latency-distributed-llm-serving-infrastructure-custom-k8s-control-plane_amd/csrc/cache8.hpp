// The 8-bit cache: e4m3 codes (OCP, no infinities) with one fp32 scale per
// block, KV head and tensor ([num_layers, total_blocks, num_kv_heads]); an
// element is code * scale.
//
// Scales are powers of two, and the kernels read nothing but their exponent.
// So code * scale is exact in bf16 (e4m3 has four significant bits), and the
// conversion to 16 bits takes the scale along in the same instruction
// (v_cvt_scalef32_pk_*_fp8).  In fp16 it is exact as well down to fp16's own
// smallest step.  A power of two costs e4m3 at most one of its 18 binades of
// range, and no precision: rounding is relative to each value's own exponent.
// When a block's scale grows, its older rows keep their values but where they
// fall among the subnormal codes.
#pragma once

#include "pa_common.hpp"

namespace pa {

struct code8_t {
  uint8_t bits;
};

// Least scale: 2^-64, so that a block of zeros has one and no product of a
// code, a scale and a probability is lost among fp32's subnormals.
constexpr int kMinScaleExp = -64;
// Largest magnitude a row may hold: the largest four-bit value below its type's
// maximum (the next one, 2^16 in fp16 and 2^128 in bf16 and fp32, would read
// back as an infinity).
template <typename T>
constexpr float kMaxRow8 = Elem<T>::kDtype == PA_DTYPE_F16 ? 61440.f : 0x1.ep127f;

typedef __bf16 bf16x2c8 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2c8 __attribute__((ext_vector_type(2)));

// The power of two a stored scale stands for.
__device__ __forceinline__ float scale_pow2(float s) {
  return __uint_as_float(__float_as_uint(s) & 0x7f800000u);
}
// The smallest power of two >= amax / 448: with amax = m * 2^e (1 <= m < 2)
// and 448 = 1.75 * 2^8 it is 2^(e-8), or 2^(e-7) for m > 1.75.
__device__ __forceinline__ float scale_for(float amax) {
  const uint32_t b = __float_as_uint(amax);
  int e = static_cast<int>(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = max(e, kMinScaleExp);
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}
// 1 / s of a power of two between 2^-126 and 2^126.
__device__ __forceinline__ float inverse_pow2(float s) {
  return __uint_as_float((254u << 23) - __float_as_uint(s));
}

// Two floats as codes in the low bits (round to nearest even; an infinity or
// a NaN becomes NaN, the only one of the two e4m3 has).
__device__ __forceinline__ uint32_t pack_codes2(float lo, float hi) {
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(lo, hi, 0, false)) & 0xffffu;
}
__device__ __forceinline__ uint32_t pack_codes4(float a, float b, float c, float d) {
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true));
}
// Code i of a word as a float.
template <int I>
__device__ __forceinline__ float code_to_f32(uint32_t w) {
  return __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(w), I);
}

// Codes (2 HIGH, 2 HIGH + 1) of a word times a scale as a packed pair of a
// 16-bit type.
template <typename T, bool HIGH>
__device__ __forceinline__ uint32_t codes_to_half2(uint32_t w, float scale);
template <>
__device__ __forceinline__ uint32_t codes_to_half2<bf16_t, false>(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(static_cast<int>(w), scale, false));
}
template <>
__device__ __forceinline__ uint32_t codes_to_half2<bf16_t, true>(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(static_cast<int>(w), scale, true));
}
template <>
__device__ __forceinline__ uint32_t codes_to_half2<f16_t, false>(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(w), scale, false));
}
template <>
__device__ __forceinline__ uint32_t codes_to_half2<f16_t, true>(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(w), scale, true));
}

}  // namespace pa
