// Rows in 8 bits: e4m3 codes with one power of two for every 128 values of a row, kept as
// its biased exponent (e8m0: 127 + log2 of the scale; 1 .. 254 here, 255 is NaN).
//
// The scale of a group is the smallest power of two s, not below 2^-126, with |v| <= 448 s
// for the group's finite values; the code is e4m3(v / s), rounded once, from f32, and NaN
// where v is NaN or infinite. A power of two costs e4m3, itself a floating type, no
// precision down to its subnormals, v / s is exact, and the matrix instructions apply it
// (their block exponents), so that a product has no work for it.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "hs_model_dev.h"

namespace hs {

constexpr int kFp8Group = 128;  // values of a scale

typedef int i32x8_t __attribute__((ext_vector_type(8)));

// the bits of |v|, 0 where v is NaN or infinite
__device__ __forceinline__ uint32_t finite_bits(float v) {
  const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}

// The scale's exponent byte for a group whose largest finite |v| has these bits: 448 is
// 1.75 2^8, so the exponent of |v| over 2^8, one more where its mantissa is above 1.75.
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits) {
  const int e = (int)((amax_bits + 0x1fffffu) >> 23) - 8;
  return (uint32_t)(e < 1 ? 1 : e);  // at most 247
}
// 1 / scale
__device__ __forceinline__ float scale_inverse(uint32_t byte) {
  return __uint_as_float((254u - byte) << 23);
}

// the code of NaN and the infinities is NaN: as NaN itself, whatever the conversion does
// with infinities
__device__ __forceinline__ float nan_unless_finite(float v) {
  return fabsf(v) < __builtin_inff() ? v : __builtin_nanf("");
}

// codes of four values that are finite or NaN
__device__ __forceinline__ uint32_t finite_codes4(const float* v, float inv) {
  int w = 0;
  w = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inv, v[1] * inv, w, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inv, v[3] * inv, w, true);
  return (uint32_t)w;
}

// codes of 32 bf16 values (in pairs; finite or NaN) under the scale of exponent `byte`
// (v_cvt_scalef32_pk_fp8_bf16: the quotient by the scale, to nearest even)
__device__ __forceinline__ i32x8_t scaled_codes32(const uint32_t (&v)[16], uint32_t byte) {
  typedef short i16x2_t __attribute__((ext_vector_type(2)));
  typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
  const float scale = __uint_as_float(byte << 23);
  i32x8_t codes;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    i16x2_t w = {0, 0};
    w = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(w, __builtin_bit_cast(bf16x2_t, v[2 * i]), scale,
                                                  false);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(w, __builtin_bit_cast(bf16x2_t, v[2 * i + 1]),
                                                  scale, true);
    codes[i] = __builtin_bit_cast(int, w);
  }
  return codes;
}

// the largest of the lanes l, l ^ 16, l ^ 32 and l ^ 48
__device__ __forceinline__ float quad_max(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// codes of four values (v_cvt_pk_fp8_f32: round to nearest even; finite |v / s| <= 448)
__device__ __forceinline__ uint32_t codes4(const float* v, float inv) {
  int w = 0;
  w = __builtin_amdgcn_cvt_pk_fp8_f32(nan_unless_finite(v[0]) * inv, nan_unless_finite(v[1]) * inv,
                                      w, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(nan_unless_finite(v[2]) * inv, nan_unless_finite(v[3]) * inv,
                                      w, true);
  return (uint32_t)w;
}

// the largest of the 16 lanes of a DPP row, in every lane
__device__ __forceinline__ uint32_t row16_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, false));
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, false));
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xF, 0xF, false));
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x128, 0xF, 0xF, false));
  return v;
}

// Codes of 8 values a lane, 16 lanes a group: all lanes of the row take part, lanes past the
// row's end with zeros. Returns the scale's byte.
__device__ __forceinline__ uint32_t group_codes8(const float (&v)[8], uint2& codes) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, finite_bits(v[i]));
  const uint32_t byte = scale_byte(row16_max(m));
  const float inv = scale_inverse(byte);
  codes = make_uint2(codes4(v, inv), codes4(v + 4, inv));
  return byte;
}

}  // namespace hs
