// The angle of a position.
#pragma once
#include <cuda_runtime.h>

namespace ftk {

// (cosine, sine) of position * inv_freq: formed and reduced to a fraction of a turn in 64 bits, since far positions turn thousands of times
__device__ __forceinline__ float2 turn_of(long long position, double inv_freq) {
  const double turns = (double)position * inv_freq * 0.15915494309189533577;      // 1 / (2 pi)
  float s, c;
  sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
  return make_float2(c, s);
}

}  // namespace ftk
