// 8-bit floating point with scales: e4m3 codes (a sign, 4 bits of exponent, 3
// of mantissa; 0x7f and 0xff are NaN) and one fp32 scale for every block of 128
// elements along a row, or of 128 x 128.  A block whose largest magnitude is m
// has the scale m / 448, 448 being the largest code, and the codes of
// y (448 / m), rounded to nearest even.  A block of 2^-100 or less is 0, with
// the scale 0 (448 / m would leave fp32's range); one that holds an infinity or
// a NaN is NaN throughout.
#pragma once
#include <cuda_fp8.h>
#include "types.cuh"

namespace pvb2 {

constexpr int kGroup8 = 128;  // elements of one scale along a row

// magnitudes as integers: they compare as the numbers do, and a NaN above all
__device__ __forceinline__ uint32_t abs_bits(float y) { return __float_as_uint(y) & 0x7fffffffu; }

struct Scale8 {
  float scale, inv;
};
__device__ __forceinline__ Scale8 scale8(uint32_t most_bits) {
  const float most = __uint_as_float(most_bits);
  // (a NaN is not below)
  if (most <= 0x1p-100f) return {0.f, 0.f};
  return {__fdiv_rn(most, 448.f), __fdiv_rn(448.f, most)};
}

// two codes, the first in the low byte
__device__ __forceinline__ uint32_t codes2(float a, float b) {
  return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
  return codes2(a, b) | (codes2(c, d) << 16);
}
__device__ __forceinline__ float2 values2(uint32_t codes) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes & 0xffffu), __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

}  // namespace pvb2
