// The 8-bit form that activations are kept in for the backward pass: e4m3 values with one power-of-two scale
// for each group of 32 along the last dimension.
//
//   scale byte s stands for 2^(s - 127): the least power of two (s >= 0) with max|x| <= 448 * 2^(s - 127)
//   code = e4m3(x * 2^(127 - s)), to nearest even;  value = code * 2^(s - 127)
//
// Scaling by a power of two is exact, so a value is rounded once, to 4 significant bits (fewer below 2^-14 of
// its group's largest).  The scale goes by the finite values of the group; a NaN or an infinity becomes NaN.
#pragma once

#include <cuda_fp16.h>

#include "kernels.cuh"

namespace gsa {

constexpr int kGroup = 32;

// Scale byte of a group from the bits of its largest finite |x| (fp32).  448 = 1.75 * 2^8: the byte is the
// exponent field less 8, one more where the significand is above 1.75.
__device__ __forceinline__ int scale_byte(uint32_t amax_bits) {
  const int s = (int)(amax_bits >> 23) - 8 + ((amax_bits & 0x7fffffu) > 0x600000u);
  return max(s, 0);
}
__device__ __forceinline__ float pow2_of(int s) {  // 2^(s - 127); s = 0 is below the normal range
  return __int_as_float(s ? s << 23 : 0x00400000);
}
__device__ __forceinline__ float inv_pow2_of(int s) { return __int_as_float((254 - s) << 23); }  // s <= 247

// Two values to two e4m3 codes (x0 in the low byte).  The conversion saturates infinities, which have no
// code: they go in as NaN.
__device__ __forceinline__ uint16_t to_e4m3x2(float x0, float x1) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(x1), "f"(x0));
  return r;
}
__device__ __forceinline__ float2 from_e4m3x2(uint16_t c) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(c));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
__device__ __forceinline__ uint32_t finite_abs_bits(float x) {
  const uint32_t a = __float_as_uint(x) & 0x7fffffffu;
  return a >= 0x7f800000u ? 0u : a;
}
__device__ __forceinline__ float inf_to_nan(float x) { return isinf(x) ? __int_as_float(0x7fc00000) : x; }

}  // namespace gsa
