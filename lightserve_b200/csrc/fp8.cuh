// e4m3 rows with one power-of-two scale: the storage format of the quantised
// KV cache.
//
// A row of D values (one token of one head of K or V) is stored as D e4m3
// bytes and one e8m0 byte E, value = e4m3 * 2^(E - 127). E is the smallest
// for which the row's largest finite magnitude stays at or below 448, e4m3's
// largest value. e4m3 is a floating-point format, so a power of two costs no
// relative precision against an arbitrary scale, and it makes both the scaling
// before the rounding and the product after it exact: the one rounding of the
// format is the conversion to e4m3 (3 mantissa bits, off by at most 2^-4 of
// the value, or 2^-10 of 2^(E - 127) below 2^-6 of it).
#pragma once

#include <stdint.h>

#include "common.cuh"

namespace lsb {

// Two fp32 values to e4m3 (round to nearest even), the first in the low byte.
__device__ __forceinline__ uint32_t cvt_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// Two e4m3 bytes to fp16 (exact), the low byte in the low half.
__device__ __forceinline__ uint32_t cvt_e4m3x2_f16x2(uint16_t x) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(x));
  return r;
}

__device__ __forceinline__ float2 f16x2_to_float2(uint32_t x) {
  return __half22float2(*reinterpret_cast<const __half2*>(&x));
}

// The four values of a word of e4m3 bytes.
__device__ __forceinline__ void e4m3x4_to_float(uint32_t w, float (&f)[4]) {
  const float2 a = f16x2_to_float2(cvt_e4m3x2_f16x2((uint16_t)(w & 0xffff)));
  const float2 b = f16x2_to_float2(cvt_e4m3x2_f16x2((uint16_t)(w >> 16)));
  f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
}

// The scale byte of a row whose largest finite magnitude is `amax`:
// amax = m 2^x (1 <= m < 2) fits below 448 = 1.75 2^8 at 2^(x - 8) when
// m <= 1.75 and at 2^(x - 7) above. Rows of zeros and of magnitudes below
// 2^-118 take the smallest scale the writer uses, 2^-126.
__device__ __forceinline__ int e8m0_of_amax(float amax) {
  const uint32_t b = __float_as_uint(amax);
  const int x = (int)(b >> 23);  // biased exponent
  const int e = x - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return max(e, 1);
}

// 2^(E - 127); 2^-127 is subnormal in fp32, 255 is e8m0's NaN.
__device__ __forceinline__ float e8m0_to_float(int e) {
  const uint32_t bits = e == 0 ? 0x00400000u : (e == 255 ? 0x7fc00000u : (uint32_t)e << 23);
  return __uint_as_float(bits);
}

// 2^(127 - E) for the scale bytes the writer makes (1 <= E <= 247).
__device__ __forceinline__ float e8m0_inverse(int e) { return __uint_as_float((uint32_t)(254 - e) << 23); }

// |x| for the row maximum: NaN and infinities do not take part.
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a <= 3.402823466e38f ? a : 0.f;
}

// x 2^(127 - E) ready for the e4m3 conversion. x - x is NaN for an infinity
// or a NaN and 0 otherwise, so both are stored as e4m3's NaN (it has no
// infinity, and the conversion would saturate them to 448).
__device__ __forceinline__ float scaled_for_e4m3(float x, float inv) { return fmaf(x, inv, x - x); }

// Rounding to e4m3 can lift a value at the top of T's range past it (65504
// becomes 65536): a dequantised row, and an fp16 attention output made of such
// values, stays at T's largest finite value (a wider type's values of that size
// are past what attention's fp32 sums hold). NaN stays NaN.
template <typename T> struct FiniteMax;
template <> struct FiniteMax<float> { static constexpr float v = 3.402823466e38f; };
template <> struct FiniteMax<__nv_bfloat16> { static constexpr float v = 3.38953139e38f; };
template <> struct FiniteMax<__half> { static constexpr float v = 65504.f; };

template <typename T>
__device__ __forceinline__ float clamp_finite(float x) {
  constexpr float M = FiniteMax<T>::v;
  x = x > M ? M : x;
  return x < -M ? -M : x;
}

}  // namespace lsb
