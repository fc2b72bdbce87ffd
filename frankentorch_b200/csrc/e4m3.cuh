// 8-bit floating point of a cache (e4m3: 4 bits of exponent, 3 of mantissa, largest 448, no infinities) and the scale of a block.
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

namespace ftk {

constexpr float E4M3_MOST = 448.f;

// Two values, rounded to nearest even; what is beyond 448 (of finite values nothing is, under their block's scale) and NaN become NaN.
__device__ __forceinline__ uint32_t e4m3_pair(float a, float b) {
  a = fabsf(a) <= E4M3_MOST ? a : __int_as_float(0x7fffffff);
  b = fabsf(b) <= E4M3_MOST ? b : __int_as_float(0x7fffffff);
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
  return r;
}
// The same of values of up to 448 and NaN
__device__ __forceinline__ uint32_t e4m3_finite(float a, float b) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
  return r;
}
// Two values of the low 16 bits as fp16, which holds every one of them
__device__ __forceinline__ uint32_t e4m3_up(uint32_t pair) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)pair));
  return r;
}
__device__ __forceinline__ float2 e4m3_floats(uint32_t pair) {
  const uint32_t h = e4m3_up(pair);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
// The smallest power of two, 2^-100 at least, of which 448 times reaches `a` >= 0.  A finer scale would gain nothing: the type's
// precision is relative, the power of two costs one of its 17 binades, and scales that grow keep the bits of the values in place.
__host__ __device__ __forceinline__ float e4m3_scale(float a) {
#ifdef __CUDA_ARCH__
  const uint32_t bits = __float_as_uint(a);
#else
  union { float f; uint32_t u; } x = {a};
  const uint32_t bits = x.u;
#endif
  int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u);      // 448 = 1.75 * 2^8
  e = e < -100 ? -100 : e;
#ifdef __CUDA_ARCH__
  return __int_as_float((e + 127) << 23);
#else
  union { int i; float f; } y = {(e + 127) << 23};
  return y.f;
#endif
}
__device__ __forceinline__ float finite_size(float x) {      // |x|, or 0 for infinities and NaN
  const float a = fabsf(x);
  return a <= 3.402823466e38f ? a : 0.f;
}

}  // namespace ftk
