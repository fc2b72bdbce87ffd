// Logits of a step on their way to a choice: penalties for repeated tokens, biases, a grammar's mask.
//
// A CTA owns a slice of one row's vocabulary.  It counts the row's history for its slice in shared memory - occurrences among the
// generated tokens in the low 31 bits, "occurred at all" in bit 31; whole numbers, so the order of the additions does not
// matter - then passes over the slice once.  fp32 arithmetic, one rounding on the way out.
#include <math.h>

#include "ft_sm100.cuh"
#include "half_types.cuh"
#include "launch.cuh"
#include "ftk_api.h"

extern "C" int* ftk_status_word(void);

namespace ftk {

constexpr int LOGITS_SLICE = 8192;

__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float load1(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ void store1(float* p, float x) { *p = x; }
__device__ __forceinline__ void store1(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }
__device__ __forceinline__ void store1(__half* p, float x) { *p = __float2half_rn(x); }

template <typename T, typename O>
__global__ void __launch_bounds__(256) logits_kernel(const FtkLogitsDesc d, int* status) {
  __shared__ unsigned seen[LOGITS_SLICE];
  pdl_wait();
  pdl_trigger();
  const long long r = blockIdx.y, v0 = (long long)blockIdx.x * LOGITS_SLICE;
  const int n = (int)min((long long)LOGITS_SLICE, d.V - v0);
  for (int i = threadIdx.x; i < n; i += 256) seen[i] = 0;
  __syncthreads();
  if (d.tokens) {
    long long len = d.L, prompt = 0;
    if (d.lengths) {
      len = d.lengths[r];
      if (len < 0 || len > d.L) ft_index_ok(-1, 1, status);
      len = len < 0 ? 0 : (len > d.L ? d.L : len);
    }
    if (d.prompts) prompt = d.prompts[r];
    for (long long j = threadIdx.x; j < len; j += 256) {
      const long long id = d.tokens[r * d.ldt + j];
      if (!ft_index_ok(id, d.V, status)) continue;
      if (id < v0 || id >= v0 + n) continue;
      if (j >= prompt) atomicAdd(&seen[id - v0], 1u);
      atomicOr(&seen[id - v0], 0x80000000u);
    }
    __syncthreads();
  }
  const float rep = d.rep_rows ? d.rep_rows[r] : (float)d.rep, freq = d.freq_rows ? d.freq_rows[r] : (float)d.freq;
  const float pres = d.pres_rows ? d.pres_rows[r] : (float)d.pres;
  const T* in = (const T*)d.logits + r * d.ld + v0;
  O* out = (O*)d.out + r * d.ldo + v0;
  for (int i = threadIdx.x; i < n; i += 256) {
    float x = load1(in + i);
    const unsigned c = seen[i];
    if (c) {
      x = x > 0.f ? x / rep : x * rep;
      const unsigned k = c & 0x7fffffffu;
      if (k) x = x - freq * (float)k - pres;
    }
    if (d.bias) x += d.bias[r * d.bias_rs + v0 + i];
    if (d.allowed && !((unsigned)d.allowed[r * d.allowed_rs + ((v0 + i) >> 5)] >> ((v0 + i) & 31) & 1u)) x = -INFINITY;
    store1(out + i, x);
  }
}

template <typename T, typename O>
static int launch(const FtkLogitsDesc& d, cudaStream_t s) {
  return launch_pdl(logits_kernel<T, O>, dim3((unsigned)((d.V + LOGITS_SLICE - 1) / LOGITS_SLICE), (unsigned)d.R), dim3(256), 0, s, d,
                    ftk_status_word());
}

}  // namespace ftk
using namespace ftk;

extern "C" int ftk_logits(const FtkLogitsDesc* d, void* stream) {
  if (!d || d->R <= 0 || d->R > 65535 || d->V <= 0 || d->V > 0x7fffffff || !d->logits || !d->out) return -2;
  cudaStream_t s = (cudaStream_t)stream;
  if (d->type == FTK_T_FP32 && d->out_type == FTK_T_FP32) return launch<float, float>(*d, s);
  if (d->type == FTK_T_BF16 && d->out_type == FTK_T_FP32) return launch<__nv_bfloat16, float>(*d, s);
  if (d->type == FTK_T_FP16 && d->out_type == FTK_T_FP32) return launch<__half, float>(*d, s);
  if (d->type == FTK_T_BF16 && d->out_type == FTK_T_BF16) return launch<__nv_bfloat16, __nv_bfloat16>(*d, s);
  if (d->type == FTK_T_FP16 && d->out_type == FTK_T_FP16) return launch<__half, __half>(*d, s);
  return -2;
}
