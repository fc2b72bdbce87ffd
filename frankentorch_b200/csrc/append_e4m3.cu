// Keys and values of new tokens into a paged cache of 8-bit floating point (e4m3) with a scale per block of rows and head, the keys
// turned by position on the way.
//
// Mathematics.  A block's new elements x (keys after the rotation, in fp32) with the largest finite magnitude a get the scale
// s = 2^e, the smallest with a <= 448 s; a block that has earlier rows keeps the larger of s and its own s', and its rows become
// y s' / s.  An element is x / s, rounded once.
#include "e4m3.cuh"
#include "ft_sm100.cuh"
#include "half_types.cuh"
#include "launch.cuh"
#include "ftk_api.h"
#include "paged_cache.h"
#include "rotary.cuh"

extern "C" int* ftk_status_word(void);

namespace ftk {

constexpr int A8_THREADS = 128;

// A warp per block of rows, head and operand (keys, values).
template <typename T, bool INTER>
__global__ void __launch_bounds__(A8_THREADS) append_e4m3_kernel(const __grid_constant__ FtkRotaryDesc d, const long long blocks, const long long units, int* status) {
  const int lane = threadIdx.x & 31, half = (int)(d.turn >> 1), chunks = (int)(d.hd >> 4);
  pdl_wait();
  pdl_trigger();
  const long long unit = (long long)blockIdx.x * (A8_THREADS / 32) + (threadIdx.x >> 5);
  if (unit >= units) return;
  const int heads = 2 * (int)d.Hkv, g = (int)(unit % heads);
  const long long b = unit / heads / blocks, j = unit / heads % blocks;
  const bool key = g < (int)d.Hkv;
  const int h = key ? g : g - (int)d.Hkv;
  const long long start = d.start[b];
  long long n = d.S;
  if (d.counts) {
    n = d.counts[b];
    if (n < 0 || n > d.S) {
      if (j == 0 && g == 0 && lane == 0) ft_index_ok(-1, 1, status);
      n = n < 0 ? 0 : d.S;
    }
  }
  const long long row0 = ((start >> d.block_shift) + j) << d.block_shift;      // the block's first position
  const long long p0 = max(row0, start), p1 = min(row0 + (1ll << d.block_shift), start + n);
  if (p0 >= p1) return;
  const PagedTable table = {d.table, d.table_stride, d.table_cols, d.n_pages, (int)d.page_shift};
  const long long page = paged_page(table, b, row0);
  if (page < 0) {
    if (lane == 0) ft_index_ok(-1, 1, status);
    return;
  }
  const long long in = paged_row(table, row0);
  unsigned char* rows = key ? (unsigned char*)d.k_pages + page * d.kp_ps + h * d.kp_hs + in * d.kp_rs : (unsigned char*)d.v_pages + page * d.vp_ps + h * d.vp_hs + in * d.vp_rs;
  const long long rs = key ? d.kp_rs : d.vp_rs;
  float* scale = (key ? d.k_scales + page * d.ks_ps + h * d.ks_hs : d.v_scales + page * d.vs_ps + h * d.vs_hs) + (in >> d.block_shift);
  const T* src = key ? (const T*)d.k + b * d.k_bs + h * d.k_hs : (const T*)d.v + b * d.v_bs + h * d.v_hs;
  const long long ss = key ? d.k_ss : d.v_ss;
  const int items = (int)(p1 - p0) * chunks;
  // 16 elements of a token: eight whole pairs
  const auto load = [&](int i, float (&x)[16], int& o0, int& o1) {
    const int t = i / chunks, c = i % chunks;
    const bool turned = key && c * 16 < (int)d.turn, apart = turned && !INTER;
    o0 = apart ? c * 8 : c * 16, o1 = apart ? half + c * 8 : c * 16 + 8;
    const T* at = src + (p0 - start + t) * ss;
    up8<T>(*reinterpret_cast<const uint4*>(at + o0), x);
    up8<T>(*reinterpret_cast<const uint4*>(at + o1), x + 8);
    if (turned) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float2 a = turn_of(p0 + t, d.inv_freq[c * 8 + e]);
        float& u = INTER ? x[2 * e] : x[e];
        float& v = INTER ? x[2 * e + 1] : x[8 + e];
        const float y = u * a.x - v * a.y;
        v = v * a.x + u * a.y;
        u = y;
      }
    }
  };
  float most = 0.f;
  for (int i = lane; i < items; i += 32) {
    float x[16];
    int o0, o1;
    load(i, x, o0, o1);
#pragma unroll
    for (int e = 0; e < 16; ++e) most = fmaxf(most, finite_size(x[e]));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
  float s = e4m3_scale(most);
  if (p0 > row0) {
    const float had = *scale;
    __syncwarp();
    if (!(had >= s)) {      // the rows that are there, under the larger scale
      const float by = had / s;
      for (int i = lane; i < (int)(p0 - row0) * chunks; i += 32) {
        uint2* at = reinterpret_cast<uint2*>(rows + i / chunks * rs + i % chunks * 16);
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          uint2 y = at[w];
          uint32_t* u = reinterpret_cast<uint32_t*>(&y);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float2 lo = e4m3_floats(u[k] & 0xffffu), hi = e4m3_floats(u[k] >> 16);
            u[k] = e4m3_pair(lo.x * by, lo.y * by) | e4m3_pair(hi.x * by, hi.y * by) << 16;
          }
          at[w] = y;
        }
      }
    } else {
      s = had;
    }
  }
  if (lane == 0) *scale = s;
  const float by = 1.f / s;
  for (int i = lane; i < items; i += 32) {
    float x[16];
    int o0, o1;
    load(i, x, o0, o1);
    uint32_t y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = e4m3_pair(x[4 * e] * by, x[4 * e + 1] * by) | e4m3_pair(x[4 * e + 2] * by, x[4 * e + 3] * by) << 16;
    unsigned char* to = rows + (p0 - row0 + i / chunks) * rs;
    *reinterpret_cast<uint2*>(to + o0) = make_uint2(y[0], y[1]);
    *reinterpret_cast<uint2*>(to + o1) = make_uint2(y[2], y[3]);
  }
}

template <typename T>
static int launch(const FtkRotaryDesc& d, long long blocks, cudaStream_t s) {
  const long long units = d.B * blocks * 2 * d.Hkv, ctas = (units + A8_THREADS / 32 - 1) / (A8_THREADS / 32);
  if (ctas > 0x7fffffff) return -2;
  const auto kernel = d.interleaved ? append_e4m3_kernel<T, true> : append_e4m3_kernel<T, false>;
  return launch_pdl(kernel, dim3((unsigned)ctas), dim3(A8_THREADS), 0, s, d, blocks, units, ftk_status_word());
}

}  // namespace ftk
using namespace ftk;

extern "C" int ftk_append_e4m3(const FtkRotaryDesc* d, void* stream) {
  if (!d || d->B <= 0 || d->S <= 0 || d->Hkv <= 0 || d->hd <= 0 || d->hd % 16 || d->turn < 0 || d->turn % 16 || d->turn > d->hd) return -2;
  if ((d->turn && !d->inv_freq) || (d->type != FTK_T_BF16 && d->type != FTK_T_FP16)) return -2;
  if (!d->k || !d->v || !d->k_pages || !d->v_pages || !d->k_scales || !d->v_scales || !d->table || !d->start) return -2;
  if (d->page_shift < 0 || d->page_shift > 30 || d->block_shift < 0 || d->block_shift > 6 || d->block_shift > d->page_shift) return -2;
  if (d->S > 0x3fffffff || d->B > (1 << 30) || d->Hkv > (1 << 20)) return -2;
  if (d->q) {
    FtkRotaryDesc q = *d;
    q.k = q.v = nullptr, q.k_pages = q.v_pages = nullptr;
    const int rc = ftk_rotary(&q, stream);
    if (rc) return rc;
  }
  const long long block = 1ll << d->block_shift, blocks = (d->S + block - 2) / block + 1;
  return d->type == FTK_T_BF16 ? launch<__nv_bfloat16>(*d, blocks, (cudaStream_t)stream) : launch<__half>(*d, blocks, (cudaStream_t)stream);
}
