// Rows in 8 bits: e4m3 codes beside one power of two (E8M0) for each row.
//
// The power 2^e of a row is the least whose 448 (the largest code) reaches max |x|; being a
// power of two it costs no precision (codes of values down to 2^-15 of the largest keep the
// four bits that e4m3 has), and codes times it are exact in bf16, and in fp16 down to the
// step of its smallest numbers.  A conversion makes two features of T of two codes and the
// power in one instruction: half of one a feature, for half of the bytes.
#pragma once
#include "mfma.h"

namespace vafa {

namespace {

// 16 codes times 2^(byte - 127) as two 16-byte pieces of T.  The conversion takes the
// exponent field of `scale`.
__device__ __forceinline__ float row_scale(uint32_t byte) {
  return __uint_as_float(byte != 0 ? byte << 23 : 0x00400000u);
}
template <typename T>
__device__ __forceinline__ uint32_t two_of_codes(uint32_t codes, float scale, bool high);
template <>
__device__ __forceinline__ uint32_t two_of_codes<bf16>(uint32_t codes, float scale, bool high) {
  return __builtin_bit_cast(
      uint32_t, high ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, true)
                     : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, false));
}
template <>
__device__ __forceinline__ uint32_t two_of_codes<f16>(uint32_t codes, float scale, bool high) {
  return __builtin_bit_cast(
      uint32_t, high ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, true)
                     : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, false));
}
template <typename T>
__device__ __forceinline__ void from_codes(u32x4 x, float scale, u32x4 &lo, u32x4 &hi) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    lo[2 * i] = two_of_codes<T>(x[i], scale, false);
    lo[2 * i + 1] = two_of_codes<T>(x[i], scale, true);
    hi[2 * i] = two_of_codes<T>(x[2 + i], scale, false);
    hi[2 * i + 1] = two_of_codes<T>(x[2 + i], scale, true);
  }
}

// The exponent of a row whose largest finite magnitude is amax: the least e with
// amax <= 448 * 2^e (448 = 1.75 * 2^8), 0 for a row of zeros; and the limit of the scaled
// values.  At the largest exponent that limit is 240, whose value is the largest code's that
// T holds: beyond it, in the last binade of T, a code would stand for infinity.
template <typename T>
constexpr int kTopExponent = std::is_same_v<T, bf16> ? 120 : 8;

template <typename T>
__device__ __forceinline__ int row_exponent(float amax, float *limit) {
  const uint32_t bits = __float_as_uint(amax);
  int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = e < -126 ? -126 : e;
  e = e > kTopExponent<T> ? kTopExponent<T> : e;
  if (amax == 0.f) e = 0;
  *limit = e == kTopExponent<T> ? 240.f : 448.f;
  return e;
}
// x / 2^e within the limit, rounded to nearest even; infinities and NaN become NaN.
__device__ __forceinline__ float to_code_range(float x, float inv, float limit) {
  const float y = __builtin_amdgcn_fmed3f(x * inv, -limit, limit);
  return fabsf(x) < __builtin_inff() ? y : __builtin_nanf("");
}
// Eight values, times inv within 448 (or NaN), as codes.
__device__ __forceinline__ u32x2 to_codes(const float *x, float inv) {
  u32x2 r;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i] * inv, x[4 * i + 1] * inv, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2] * inv, x[4 * i + 3] * inv, w, true);
    r[i] = (uint32_t)w;
  }
  return r;
}

}  // namespace

}  // namespace vafa
