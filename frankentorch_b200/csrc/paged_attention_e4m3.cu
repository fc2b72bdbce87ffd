// Attention of one new token per sequence over a paged key-value cache held in 8 bits (e4m3) with a scale per block of rows and head.
//
// Mathematics.  x_t = scale ks_t (q . k_t), o = sum_t softmax_t(x) vs_t v_t, lse = log sum_t exp(x_t): a running maximum m, the sum l and
// the accumulator, rescaled when the maximum grows.
//
// A CTA per query head; its warps take tokens in turn.
#include <math.h>

#include "e4m3.cuh"
#include "ft_sm100.cuh"
#include "half_types.cuh"
#include "launch.cuh"
#include "ftk_api.h"
#include "paged_cache.h"

extern "C" int* ftk_status_word(void);

namespace ftk {

constexpr int A8_WARPS = 4;

template <typename T, int HD>
__global__ void __launch_bounds__(A8_WARPS * 32) paged_attn_e4m3_kernel(const __grid_constant__ FtkPagedAttnDesc d, int* status) {
  constexpr int N = HD / 32;
  __shared__ float sm[A8_WARPS], sl[A8_WARPS], sa[A8_WARPS][HD];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long b = blockIdx.x / d.Hq;
  const int h = (int)(blockIdx.x % d.Hq), kv = h / (int)(d.Hq / d.Hkv);
  pdl_wait();
  pdl_trigger();
  const PagedTable table = {d.table, d.table_stride, d.table_cols, d.n_pages, (int)d.page_shift};
  bool bad;
  const long long n = paged_length(table, d.lengths[b], bad);
  if (bad) ft_index_ok(-1, 1, status);
  float q[N], a[N] = {}, m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) q[i] = Half16<T>::one(((const T*)d.q)[b * d.q_bs + h * d.q_hs + lane * N + i]);
  for (long long t = warp; t < n; t += A8_WARPS) {
    const long long page = paged_page(table, b, t), row = paged_row(table, t);
    if (page < 0) {
      ft_index_ok(-1, 1, status);
      continue;
    }
    const unsigned char* k = (const unsigned char*)d.k_pages + page * d.kp_ps + kv * d.kp_hs + row * d.kp_rs + lane * N;
    const unsigned char* v = (const unsigned char*)d.v_pages + page * d.vp_ps + kv * d.vp_hs + row * d.vp_rs + lane * N;
    const float ks = d.k_scales[page * d.ks_ps + kv * d.ks_hs + (row >> d.block_shift)], vs = d.v_scales[page * d.vs_ps + kv * d.vs_hs + (row >> d.block_shift)];
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float2 y = e4m3_floats(*reinterpret_cast<const uint16_t*>(k + i));
      x += q[i] * y.x + q[i + 1] * y.y;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    x *= ks * (float)d.scale;
    const float top = fmaxf(m, x), base = top == -INFINITY ? 0.f : top, grow = expf(m - base), e = expf(x - base);
    m = top;
    l = l * grow + e;
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float2 y = e4m3_floats(*reinterpret_cast<const uint16_t*>(v + i));
      a[i] = a[i] * grow + e * vs * y.x, a[i + 1] = a[i + 1] * grow + e * vs * y.y;
    }
  }
  if (lane == 0) sm[warp] = m, sl[warp] = l;
#pragma unroll
  for (int i = 0; i < N; ++i) sa[warp][lane * N + i] = a[i];
  __syncthreads();
  float top = -INFINITY, sum = 0.f;
  for (int w = 0; w < A8_WARPS; ++w) top = fmaxf(top, sm[w]);
  const float base = top == -INFINITY ? 0.f : top;
  for (int w = 0; w < A8_WARPS; ++w) sum += expf(sm[w] - base) * sl[w];
  for (int i = threadIdx.x; i < HD; i += A8_WARPS * 32) {
    float v = 0.f;
    for (int w = 0; w < A8_WARPS; ++w) v += expf(sm[w] - base) * sa[w][i];
    ((T*)d.o)[b * d.o_bs + h * d.o_hs + i] = Half16<T>::round(sum == 0.f ? 0.f : v / sum);
  }
  if (threadIdx.x == 0) d.lse[b * d.Hq + h] = sum == 0.f ? -INFINITY : top + logf(sum);
}

static bool refused(const FtkPagedAttnDesc* d) {
  return !d || d->B <= 0 || d->B > (1 << 30) || d->Hkv <= 0 || d->Hq <= 0 || d->Hq % d->Hkv || d->Hq > (1 << 20) || (d->hd != 64 && d->hd != 128) ||
         (d->type != FTK_T_BF16 && d->type != FTK_T_FP16) || d->page_shift < 0 || d->page_shift > 30 || d->table_cols <= 0 ||
         d->table_cols > (0x7fffff00ll >> d->page_shift) || d->n_pages <= 0 || d->n_pages > 0x7fffffff || d->B * d->Hq > 0x7fffffff ||
         d->block_shift < 0 || d->block_shift > 6 || d->block_shift > d->page_shift;
}

}  // namespace ftk
using namespace ftk;

extern "C" long long ftk_paged_attn_e4m3_scratch(const FtkPagedAttnDesc* d) { return refused(d) ? -2 : 0; }

extern "C" int ftk_paged_attn_e4m3(const FtkPagedAttnDesc* d, void* scratch, void* stream) {
  if (refused(d) || !d->q || !d->o || !d->lse || !d->k_pages || !d->v_pages || !d->k_scales || !d->v_scales || !d->table || !d->lengths) return -2;
  const bool bf = d->type == FTK_T_BF16;
  const auto kernel = d->hd == 64 ? (bf ? paged_attn_e4m3_kernel<__nv_bfloat16, 64> : paged_attn_e4m3_kernel<__half, 64>)
                                  : (bf ? paged_attn_e4m3_kernel<__nv_bfloat16, 128> : paged_attn_e4m3_kernel<__half, 128>);
  return launch_pdl(kernel, dim3((unsigned)(d->B * d->Hq)), dim3(A8_WARPS * 32), 0, (cudaStream_t)stream, *d, ftk_status_word());
}
