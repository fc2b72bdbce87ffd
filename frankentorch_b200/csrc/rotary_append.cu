// Rotation of queries and keys by position, in training (forward, and backward with the opposite angle) and on the way into a
// paged key-value cache.
//
// Mathematics.  A pair (x0, x1) of a token at position p is turned by a = p w: (x0 cos a - x1 sin a, x1 cos a + x0 sin a).  The
// backward pass is the inverse rotation of the gradient.  Far positions turn thousands of times, so the angle is formed and
// reduced to a fraction of a turn in 64 bits (2^31 turns leave 2^-22 of a turn); sine and cosine of the fraction and the products
// are fp32, each output is rounded once.
//
// Work is divided into items of 16 elements of one head of one token: two 16-byte vectors that hold eight whole pairs (the
// vectors are turn / 2 apart where pairs are (i, i + turn / 2), else neighbours), so an item can be turned in place.
#include "ft_sm100.cuh"
#include "half_types.cuh"
#include "launch.cuh"
#include "ftk_api.h"
#include "paged_cache.h"

extern "C" int* ftk_status_word(void);

namespace ftk {

__device__ __forceinline__ float2 turn_of(long long position, double inv_freq) {
  const double turns = (double)position * inv_freq * 0.15915494309189533577;      // 1 / (2 pi)
  float s, c;
  sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
  return make_float2(c, s);
}

template <typename T>
__global__ void __launch_bounds__(256) rotary_kernel(const FtkRotaryDesc d, int heads, int* status) {
  pdl_wait();
  pdl_trigger_work(256 * 64);
  const int chunks = (int)(d.hd >> 4), half = (int)(d.turn >> 1);
  const long long items = d.B * d.S * heads * chunks;
  const long long it = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (it >= items) return;
  const int c = (int)(it % chunks);
  const int h = (int)(it / chunks % heads);
  const long long tok = it / chunks / heads;
  const long long b = tok / d.S, s = tok % d.S;
  const long long position = (d.start ? d.start[b] : 0) + s;
  const bool used = !d.counts || s < d.counts[b];
  const int hq = d.q ? (int)d.Hq : 0, hk = d.k ? (int)d.Hkv : 0;
  const T* src;
  T* dst;
  bool turn = c * 16 < d.turn;
  if (h < hq) {
    src = (const T*)d.q + b * d.q_bs + s * d.q_ss + h * d.q_hs;
    dst = (T*)d.q_out + b * d.qo_bs + s * d.qo_ss + h * d.qo_hs;
    turn = turn && used;
  } else {
    const bool is_k = h < hq + hk;
    const int g = is_k ? h - hq : h - hq - hk;
    src = is_k ? (const T*)d.k + b * d.k_bs + s * d.k_ss + g * d.k_hs : (const T*)d.v + b * d.v_bs + s * d.v_ss + g * d.v_hs;
    turn = turn && is_k;
    if (d.k_pages) {
      if (!used) return;
      const PagedTable t = {d.table, d.table_stride, d.table_cols, d.n_pages, (int)d.page_shift};
      const long long page = paged_page(t, b, position);
      if (page < 0) {
        ft_index_ok(-1, 1, status);
        return;
      }
      const long long row = paged_row(t, position);
      dst = is_k ? (T*)d.k_pages + page * d.kp_ps + g * d.kp_hs + row * d.kp_rs
                 : (T*)d.v_pages + page * d.vp_ps + g * d.vp_hs + row * d.vp_rs;
    } else {
      dst = (T*)d.k_out + b * d.ko_bs + s * d.ko_ss + g * d.ko_hs;
    }
  }
  const bool apart = c * 16 < d.turn && !d.interleaved;
  const int o0 = apart ? c * 8 : c * 16, o1 = apart ? half + c * 8 : c * 16 + 8;
  uint4 u0 = *reinterpret_cast<const uint4*>(src + o0), u1 = *reinterpret_cast<const uint4*>(src + o1);
  if (turn) {
    float a[16];
    up8<T>(u0, a);
    up8<T>(u1, a + 8);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 t = turn_of(position, d.inv_freq[c * 8 + i]);
      const float sn = d.inverse ? -t.y : t.y;
      float& x0 = d.interleaved ? a[2 * i] : a[i];
      float& x1 = d.interleaved ? a[2 * i + 1] : a[8 + i];
      const float y0 = x0 * t.x - x1 * sn, y1 = x1 * t.x + x0 * sn;
      x0 = y0;
      x1 = y1;
    }
    u0 = down8<T>(a);
    u1 = down8<T>(a + 8);
  }
  *reinterpret_cast<uint4*>(dst + o0) = u0;
  *reinterpret_cast<uint4*>(dst + o1) = u1;
}

}  // namespace ftk
using namespace ftk;

extern "C" int ftk_rotary(const FtkRotaryDesc* d, void* stream) {
  if (!d || d->B <= 0 || d->S <= 0 || d->hd <= 0 || d->hd % 16 || d->turn < 0 || d->turn % 16 || d->turn > d->hd) return -2;
  if ((d->turn && !d->inv_freq) || (d->q && !d->q_out) || (d->type != FTK_T_BF16 && d->type != FTK_T_FP16)) return -2;
  if (d->k_pages ? !d->k || !d->v || !d->v_pages || !d->table || d->page_shift < 0 || d->page_shift > 30 : (d->k && !d->k_out)) return -2;
  const long long heads = (d->q ? d->Hq : 0) + (d->k ? d->Hkv : 0) + (d->k_pages ? d->Hkv : 0);
  if (heads <= 0 || heads > (1 << 20)) return -2;
  const long long blocks = (d->B * d->S * heads * (d->hd >> 4) + 255) / 256;
  if (blocks > 0x7fffffff) return -2;
  return d->type == FTK_T_BF16
             ? launch_pdl(rotary_kernel<__nv_bfloat16>, dim3((unsigned)blocks), dim3(256), 0, (cudaStream_t)stream, *d, (int)heads, ftk_status_word())
             : launch_pdl(rotary_kernel<__half>, dim3((unsigned)blocks), dim3(256), 0, (cudaStream_t)stream, *d, (int)heads, ftk_status_word());
}
