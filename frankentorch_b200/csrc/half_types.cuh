// bf16 and fp16 as element types of one kernel: eight values of 16 bytes to fp32 and back, one rounding each way out.
#pragma once
#include <cuda_fp16.h>
#include "ft_sm100.cuh"

namespace ftk {

template <typename T> struct Half16;
template <> struct Half16<__nv_bfloat16> {
  static __device__ __forceinline__ float2 up(uint32_t u) { return unpack_bf16(u); }
  static __device__ __forceinline__ uint32_t down(float a, float b) { return pack_bf16(a, b); }
  static __device__ __forceinline__ float one(__nv_bfloat16 x) { return __bfloat162float(x); }
  static __device__ __forceinline__ __nv_bfloat16 round(float x) { return __float2bfloat16_rn(x); }
};
template <> struct Half16<__half> {
  static __device__ __forceinline__ float2 up(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
  static __device__ __forceinline__ uint32_t down(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float one(__half x) { return __half2float(x); }
  static __device__ __forceinline__ __half round(float x) { return __float2half_rn(x); }
};
template <typename T> __device__ __forceinline__ void up8(const uint4& u, float* f) {
  const float2 a = Half16<T>::up(u.x), b = Half16<T>::up(u.y), c = Half16<T>::up(u.z), d = Half16<T>::up(u.w);
  f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y; f[4] = c.x; f[5] = c.y; f[6] = d.x; f[7] = d.y;
}
template <typename T> __device__ __forceinline__ uint4 down8(const float* f) {
  return make_uint4(Half16<T>::down(f[0], f[1]), Half16<T>::down(f[2], f[3]), Half16<T>::down(f[4], f[5]),
                    Half16<T>::down(f[6], f[7]));
}

}  // namespace ftk
