// Attention of one new token per sequence over a paged key-value cache.
//
// Mathematics.  With scores x_t = scale q . k_t the running maximum m, the sum l = sum_t exp(x_t - m) and the accumulator
// a = sum_t exp(x_t - m) v_t are carried over the tokens; a larger maximum rescales l and a by exp(m_old - m_new).  Two parts join
// the same way.  o = a / l, lse = m + log(l); a part of no tokens has m = -inf, l = 0.
#include <math.h>

#include "ft_sm100.cuh"
#include "half_types.cuh"
#include "launch.cuh"
#include "ftk_api.h"
#include "paged_cache.h"

extern "C" int* ftk_status_word(void);

namespace ftk {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// One CTA per sequence and query head; each of its four warps takes every fourth token.
template <typename T, int HD>
__global__ void __launch_bounds__(128) paged_attn_kernel(const FtkPagedAttnDesc d, int* status) {
  pdl_wait();
  pdl_trigger();
  constexpr int V = HD / 32;       // elements of a row per lane
  const int b = blockIdx.y, h = blockIdx.x, g = h / (int)(d.Hq / d.Hkv);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const PagedTable t = {d.table, d.table_stride, d.table_cols, d.n_pages, (int)d.page_shift};
  bool bad;
  const long long n = paged_length(t, d.lengths[b], bad);
  if (bad) ft_index_ok(-1, 1, status);
  const T* q = (const T*)d.q + b * d.q_bs + h * d.q_hs;
  float qv[V], acc[V], m = -INFINITY, l = 0.f;
  const float sc = (float)d.scale * LOG2E;
#pragma unroll
  for (int i = 0; i < V; ++i) qv[i] = Half16<T>::one(q[lane * V + i]) * sc, acc[i] = 0.f;
  for (long long p = warp; p < n; p += 4) {
    const long long page = paged_page(t, b, p);
    if (page < 0) {
      ft_index_ok(-1, 1, status);
      continue;
    }
    const T* k = (const T*)d.k_pages + page * d.kp_ps + g * d.kp_hs + paged_row(t, p) * d.kp_rs + lane * V;
    const T* v = (const T*)d.v_pages + page * d.vp_ps + g * d.vp_hs + paged_row(t, p) * d.vp_rs + lane * V;
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) x += qv[i] * Half16<T>::one(k[i]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    const float top = fmaxf(m, x), base = top == -INFINITY ? 0.f : top;
    const float f = exp2f(m - base), e = exp2f(x - base);
    m = top;
    l = l * f + e;
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = acc[i] * f + e * Half16<T>::one(v[i]);
  }
  __shared__ float sa[4][HD], sm[4], sl[4];
#pragma unroll
  for (int i = 0; i < V; ++i) sa[warp][lane * V + i] = acc[i];
  if (lane == 0) sm[warp] = m, sl[warp] = l;
  __syncthreads();
  const float top = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3])), base = top == -INFINITY ? 0.f : top;
  float f[4], sum = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) f[w] = exp2f(sm[w] - base), sum += f[w] * sl[w];
  for (int i = threadIdx.x; i < HD; i += 128) {
    float a = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) a += f[w] * sa[w][i];
    ((T*)d.o)[b * d.o_bs + h * d.o_hs + i] = Half16<T>::round(sum == 0.f ? 0.f : a / sum);
  }
  if (threadIdx.x == 0) d.lse[(long long)b * d.Hq + h] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * LN2;
}

template <typename T, int HD>
static int launch(const FtkPagedAttnDesc& d, cudaStream_t s) {
  return launch_pdl(paged_attn_kernel<T, HD>, dim3((unsigned)d.Hq, (unsigned)d.B), dim3(128), 0, s, d, ftk_status_word());
}

}  // namespace ftk
using namespace ftk;

extern "C" int ftk_paged_attn(const FtkPagedAttnDesc* d, void* stream) {
  if (!d || d->B <= 0 || d->B > 65535 || d->Hkv <= 0 || d->Hq <= 0 || d->Hq % d->Hkv || d->Hq > 65535) return -2;
  if (!d->q || !d->o || !d->lse || !d->k_pages || !d->v_pages || !d->table || !d->lengths || d->page_shift < 0 || d->page_shift > 30)
    return -2;
  cudaStream_t s = (cudaStream_t)stream;
  if (d->type == FTK_T_BF16 && d->hd == 64) return launch<__nv_bfloat16, 64>(*d, s);
  if (d->type == FTK_T_BF16 && d->hd == 128) return launch<__nv_bfloat16, 128>(*d, s);
  if (d->type == FTK_T_FP16 && d->hd == 64) return launch<__half, 64>(*d, s);
  if (d->type == FTK_T_FP16 && d->hd == 128) return launch<__half, 128>(*d, s);
  return -2;
}
