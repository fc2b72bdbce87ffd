// The choice of a token from the logits of a step: temperature, top-k, top-p, min-p, and a given random number.
//
// Mathematics.  Weights are whole numbers, w_i = round(2^43 exp((x_i - max x) / T)), so their sums (63 bits for up to 2^20 tokens) are exact
// whatever their order, and a row's choice is a function of its logits, settings and random number alone.  With tokens in the order of
// their logits (equal ones by their ids): the first k; of those the ones before which less than p of the sum lies; of those the ones of
// at least min_p of the largest; then the first by id whose running sum passes u times the sum.
//
// A CTA per row.  The border of top-k and of top-p is a logit and a number of equal ones: digits of eight bits, the highest first, with
// counts or sums of weights per digit.
#include <math.h>

#include "ft_sm100.cuh"
#include "half_types.cuh"
#include "launch.cuh"
#include "ftk_api.h"

namespace ftk {

constexpr int SA_THREADS = 512;
typedef unsigned long long u64;

__device__ __forceinline__ float logit_of(const float* p) { return *p; }
template <typename T> __device__ __forceinline__ float logit_of(const T* p) { return Half16<T>::one(*p); }
// Whole numbers in the order of the logits (0 and -0 are equal)
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
// f * n for 0 <= f < 1, rounded down or up
template <bool UP> __device__ __forceinline__ u64 share_of(u64 n, float f) {
  if (!(f > 0.f)) return 0;
  int e;
  const u64 m = (u64)(frexpf(f, &e) * 16777216.f);      // f = m 2^(e - 24), exactly
  const int s = 24 - e;
  const u64 lo = n * m, hi = __umul64hi(n, m);
  if (s >= 128) return UP && n ? 1 : 0;
  const u64 down = s < 64 ? (hi << (64 - s)) | (lo >> s) : hi >> (s - 64);
  if (!UP) return down;
  const bool rest = s < 64 ? (lo << (64 - s)) != 0 : lo != 0 || (s > 64 && (hi << (128 - s)) != 0);
  return down + rest;
}
template <typename V> __device__ __forceinline__ V block_sum(V v, V* buf) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
  for (int w = 0; w < SA_THREADS / 32; ++w) v += buf[w];
  return v;
}

template <typename T>
__global__ void __launch_bounds__(SA_THREADS) sample_kernel(const __grid_constant__ FtkSampleDesc d) {
  __shared__ u64 hist[256], part[SA_THREADS + 1], buf[SA_THREADS / 32], found[4];
  const int tid = threadIdx.x, V = (int)d.V;
  const long long r = blockIdx.x;
  pdl_wait();
  pdl_trigger();
  const T* x = (const T*)d.logits + r * d.ld;
  const auto at = [&](int i) { return logit_of(x + i); };
  const float t = d.temp_rows ? d.temp_rows[r] : (float)d.temp, p = d.p_rows ? d.p_rows[r] : (float)d.p, least = d.min_rows ? d.min_rows[r] : (float)d.min_p;
  const float u = d.uniform[r];
  const long long k0 = d.k_rows ? d.k_rows[r] : d.k;
  float top = -INFINITY;
  bool odd = !(t >= 0.f) || p != p || least != least || u != u;
  for (int i = tid; i < V; i += SA_THREADS) top = fmaxf(top, at(i)), odd |= at(i) != at(i);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if ((tid & 31) == 0) part[tid >> 5] = order_of(top);
  odd = __syncthreads_or(odd);
  uint32_t most = 0;
  for (int w = 0; w < SA_THREADS / 32; ++w) most = max(most, (uint32_t)part[w]);
  top = __uint_as_float(most & 0x80000000u ? most & 0x7fffffffu : ~most);
  if (odd || top == -INFINITY) {
    if (tid == 0) d.token[r] = -1, d.logprob[r] = odd ? NAN : -INFINITY;
    return;
  }
  const double by = t > 0.f ? 1.0 / (double)t : 0.0;
  const auto weight = [&](float y) -> u64 {
    if (y == top) return 1ull << 43;
    if (y == -INFINITY || t == 0.f || top == INFINITY) return 0;
    return (u64)rint(exp(((double)y - (double)top) * by) * 0x1p43);
  };
  const long long k = t == 0.f ? 1 : (k0 <= 0 || k0 > V ? V : k0);
  uint32_t border = 0;      // kept: what is larger, and equal ones up to id `last`
  int last = V;
  const auto kept = [&](int i, float y) {
    const uint32_t o = order_of(y);
    return o > border || (o == border && i <= last);
  };
  // Moves the border to where the running sum of counts or weights of what is kept reaches `limit` > 0
  const auto cut = [&](bool mass, u64 limit) {
    uint32_t high = 0;
    u64 before = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += SA_THREADS) hist[i] = 0;
      __syncthreads();
      for (int i = tid; i < V; i += SA_THREADS) {
        const float y = at(i);
        const uint32_t o = order_of(y);
        if (!kept(i, y) || (shift < 24 && (o >> (shift + 8)) != (high >> (shift + 8)))) continue;
        const u64 w = mass ? weight(y) : 1;
        if (w) atomicAdd(&hist[o >> shift & 255], w);
      }
      __syncthreads();
      if (tid == 0) {
        int digit = 255;
        for (; digit > 0 && before + hist[digit] < limit; --digit) before += hist[digit];
        found[0] = digit, found[1] = before;
      }
      __syncthreads();
      high |= (uint32_t)found[0] << shift, before = found[1];
      __syncthreads();
    }
    // of the equal ones: as many as are needed, by their ids
    const float y = __uint_as_float(high & 0x80000000u ? high & 0x7fffffffu : ~high);
    const u64 one = mass ? weight(y) : 1, need = one ? (limit - before + one - 1) / one : 0;
    const int seg = (V + SA_THREADS - 1) / SA_THREADS, i0 = min(V, tid * seg), i1 = min(V, i0 + seg);
    u64 n = 0;
    for (int i = i0; i < i1; ++i) n += order_of(at(i)) == high && kept(i, at(i));
    part[tid] = n;
    if (tid == 0) found[2] = V;
    __syncthreads();
    u64 front = 0;
    for (int j = 0; j < tid; ++j) front += part[j];
    if (front < need && need <= front + n) {
      for (int i = i0; i < i1; ++i)
        if (order_of(at(i)) == high && kept(i, at(i)) && ++front == need) {
          found[2] = i;
          break;
        }
    }
    __syncthreads();
    border = high, last = (int)found[2];
    __syncthreads();
  };
  if (k < V) cut(false, (u64)k);
  if (p < 1.f) {
    u64 sum = 0;
    for (int i = tid; i < V; i += SA_THREADS)
      if (kept(i, at(i))) sum += weight(at(i));
    const u64 limit = share_of<true>(block_sum(sum, buf), p);
    cut(true, limit > 0 ? limit : 1);
  }
  const u64 low = least >= 1.f ? 1ull << 43 : (u64)ceil(fmax((double)least, 0.0) * 0x1p43);
  const auto final = [&](int i, float y) -> u64 {
    const u64 w = kept(i, y) ? weight(y) : 0;
    return w >= low ? w : 0;
  };
  const int seg = (V + SA_THREADS - 1) / SA_THREADS, i0 = min(V, tid * seg), i1 = min(V, i0 + seg);
  u64 sum = 0;
  for (int i = i0; i < i1; ++i) sum += final(i, at(i));
  part[tid] = sum;
  __syncthreads();
  u64 front = 0, total = 0;
  for (int j = 0; j < SA_THREADS; ++j) {
    if (j < tid) front += part[j];
    total += part[j];
  }
  const u64 target = u >= 1.f ? total - 1 : min(share_of<false>(total, u), total - 1);
  if (front <= target && target < front + sum) {
    for (int i = i0; i < i1; ++i) {
      const u64 w = final(i, at(i));
      if (target < front + w) {
        d.token[r] = i, d.logprob[r] = (float)log((double)w / (double)total);
        return;
      }
      front += w;
    }
  }
}

}  // namespace ftk
using namespace ftk;

extern "C" int ftk_sample(const FtkSampleDesc* d, void* stream) {
  if (!d || !d->logits || !d->uniform || !d->token || !d->logprob || d->R <= 0 || d->R > 0x7fffffff || d->V <= 0 || d->V > (1 << 20)) return -2;
  const auto kernel = d->type == FTK_T_FP32 ? sample_kernel<float> : d->type == FTK_T_BF16 ? sample_kernel<__nv_bfloat16> : sample_kernel<__half>;
  if (d->type < FTK_T_BF16 || d->type > FTK_T_FP32) return -2;
  return launch_pdl(kernel, dim3((unsigned)d->R), dim3(SA_THREADS), 0, (cudaStream_t)stream, *d);
}
