// Rows of a cache in 8 bits, as the kernels read and write them.
//
// A row of 128 elements is 128 codes of the type e4m3 (sign, 4 bits of exponent, 3 of mantissa, the largest 448, code 0x7f
// NaN) and one byte of the type e8m0, the biased exponent of its scale 2^(b - 127); 255 is NaN.  The rows of a plane lie
// wherever their codes do: the scale of the row whose codes begin at byte x of a layer is byte x / 128 of the layer's
// scales.  A power of two as scale costs e4m3 nothing (its error is relative down to 2^-9 of a row's scale) and makes every
// step exact but one, the rounding of x / 2^e to four significant bits: what is read back is a 16-bit value as it stands.
#pragma once

#include "common.hpp"

namespace ellm {

typedef short i16x2 __attribute__((ext_vector_type(2)));

constexpr uint32_t kScaleNan = 255;

// The scale of a row as the conversions take it (they look at the exponent field alone, as e8m0: 0 is 2^-127, 255 NaN).
__device__ __forceinline__ float scale_of(uint32_t byte) { return __builtin_bit_cast(float, byte << 23); }

// Two codes of a register (the low or the high pair) times a scale as two 16-bit values: exact, where the type has the value.
template <typename T>
struct Codes;
template <>
struct Codes<F16> {
  template <bool HI>
  static __device__ __forceinline__ uint32_t pair(uint32_t codes, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, HI));
  }
  // the largest value of four significant bits: what a row's values are cut to ahead of their rounding
  static constexpr float kLargest = 61440.0f;   // 1.875 x 2^15
};
template <>
struct Codes<BF16> {
  template <bool HI>
  static __device__ __forceinline__ uint32_t pair(uint32_t codes, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, HI));
  }
  static constexpr float kLargest = 0x1.ep127f;
};

// Four codes as four 16-bit values.
template <typename T>
__device__ __forceinline__ u32x2 values4(uint32_t codes, float scale) {
  return u32x2{Codes<T>::template pair<false>(codes, scale), Codes<T>::template pair<true>(codes, scale)};
}

// Eight codes of a row as eight 16-bit values.
template <typename T>
__device__ __forceinline__ u32x4 values8(u32x2 codes, uint32_t scale) {
  const u32x2 lo = values4<T>(codes[0], scale_of(scale)), hi = values4<T>(codes[1], scale_of(scale));
  return u32x4{lo[0], lo[1], hi[0], hi[1]};
}
// The scales that a key row and its value row are taken with.  The key of a value row whose scale is NaN has a scale of NaN too: rows
// that see it get weights of NaN, and so both results.  A chunk's kernels take the value row itself as what its codes say (zeros,
// where the cache wrote them): rows that do not see it yet give it a weight of exactly 0, and 0 x NaN would be NaN.
__device__ __forceinline__ uint32_t key_scale(uint32_t k, uint32_t v) { return v == kScaleNan ? kScaleNan : k; }
__device__ __forceinline__ uint32_t value_scale(uint32_t v) { return v == kScaleNan ? 127u : v; }

// The byte of the smallest scale 2^e with top <= 448 2^e, e >= -126; `top`: the bits of the row's largest magnitude (those of
// infinities and NaN: the scale is NaN).  448 is 1.75 x 2^8: a mantissa above 1.75 (0x600000) carries into the exponent.
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
  const uint32_t b = (top + 0x1fffffu) >> 23;
  return top >= 0x7f800000u ? kScaleNan : b > 9 ? b - 8 : 1;
}

// x of the lane 1, 2, 4 or 8 apart, in a row of sixteen lanes of which the lanes that STEP's earlier ones joined hold the same x:
// there lane 7 - i stands for i ^ 4, and 15 - i for i ^ 8.  No trip through LDS, as an exchange of any two lanes is.
template <int STEP>
__device__ __forceinline__ uint32_t from_partner16(uint32_t x) {
  constexpr int kCtrl = STEP == 1 ? 0xb1 : STEP == 2 ? 0x4e : STEP == 4 ? 0x141 : 0x140;   // quad_perm 1 0 3 2, 2 3 0 1; mirrors
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, kCtrl, 0xf, 0xf, true);
}
__device__ __forceinline__ float sum16(float x) {
  auto with = [&](uint32_t y) { x = x + __builtin_bit_cast(float, y); };
  with(from_partner16<1>(__builtin_bit_cast(uint32_t, x)));
  with(from_partner16<2>(__builtin_bit_cast(uint32_t, x)));
  with(from_partner16<4>(__builtin_bit_cast(uint32_t, x)));
  with(from_partner16<8>(__builtin_bit_cast(uint32_t, x)));
  return x;
}
__device__ __forceinline__ uint32_t max16(uint32_t x) {
  x = max(x, from_partner16<1>(x));
  x = max(x, from_partner16<2>(x));
  x = max(x, from_partner16<4>(x));
  return max(x, from_partner16<8>(x));
}

template <typename T>
__device__ __forceinline__ void unpack8(u32x4 raw, float (&x)[8]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[2 * e] = Mfma<T>::to_float((uint16_t)(raw[e] & 0xffffu));
    x[2 * e + 1] = Mfma<T>::to_float((uint16_t)(raw[e] >> 16));
  }
}

// The key row that lane c of sixteen holds eight elements of, normalised and rotated: the formulas of norm_rope_row16
// (common.hpp) in binary32, one rounding an operation, but the squares added as a tree (a lane's eight in order, then
// across lanes 1, 2, 4, 8 apart) and the results not rounded: the codes are taken of them as they are.
template <typename T>
__device__ __forceinline__ void norm_rope8(float (&x)[8], u32x4 turn, float eps) {
#pragma clang fp contract(off)
  float sum = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) sum = sum + x[e] * x[e];
  sum = sum16(sum);
  const float rrms = 1.0f / (sqrtf(sum / (float)kHeadDim) + eps);
  float w[8];
  unpack8<T>(turn, w);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float a = x[2 * e] * rrms, b = x[2 * e + 1] * rrms;
    x[2 * e] = a * w[2 * e] - b * w[2 * e + 1];
    x[2 * e + 1] = a * w[2 * e + 1] + b * w[2 * e];
  }
}

// Sixteen lanes hold a row, eight values each: their codes, and the scale's byte.  Every lane of the wave must call this.
template <typename T>
__device__ __forceinline__ u32x2 row_codes16(const float (&x)[8], uint32_t& byte) {
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, __builtin_bit_cast(uint32_t, x[e]) & 0x7fffffffu);
  byte = scale_byte(max16(top));
  const float scale = scale_of(byte);
  u32x2 codes;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    float c[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      c[e] = __builtin_amdgcn_fmed3f(x[4 * w + e], -Codes<T>::kLargest, Codes<T>::kLargest);
    i16x2 to = {0, 0};
    to = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(to, c[0], c[1], scale, false);
    to = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(to, c[2], c[3], scale, true);
    codes[w] = byte == kScaleNan ? 0u : __builtin_bit_cast(uint32_t, to);   // (a row that is NaN holds no values)
  }
  return codes;
}

}  // namespace ellm
