// Rotation of queries and keys by position, in training (forward, and backward with the opposite angle) and on the way into a
// paged key-value cache.
//
// Mathematics.  A pair (x0, x1) of a token at position p is turned by a = p w: (x0 cos a - x1 sin a, x1 cos a + x0 sin a).  The
// backward pass is the inverse rotation of the gradient.  Far positions turn thousands of times, so the angle is formed and
// reduced to a fraction of a turn in 64 bits (2^31 turns leave 2^-22 of a turn); sine and cosine of the fraction and the products
// are fp32, each output is rounded once.
//
// What bounds it: each element is read once and written once; the copy bandwidth, and for a handful of tokens the latency of a
// position, a page number and a row behind one another.
//
// Work is divided into items of 16 elements of one head of one token: two 16-byte vectors that hold eight whole pairs (the
// vectors are turn / 2 apart where pairs are (i, i + turn / 2), else neighbours), so an item can be turned in place.  A CTA has some
// tokens with all their heads: it requests its items, up to four per thread, forms the angles' sines and cosines once per token and
// pair while they arrive, and turns.
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

constexpr int RO_THREADS = 256;

// Where the tokens of a CTA go: page and row in the cache, or page -1 for none.
struct TokenPlace {
  long long page;
  int row, used;
};
struct RotaryShape {
  int tokens, heads, hblocks;      // of a CTA; CTAs that share the heads of a token
  int hq, hk, chunks;              // heads of the queries and of the cache that take part, items of a head
};

template <typename T, int K, bool INTER>
__global__ void __launch_bounds__(RO_THREADS) rotary_kernel(const __grid_constant__ FtkRotaryDesc d, const RotaryShape w, int* status) {
  extern __shared__ __align__(16) unsigned char smem[];
  const int half = (int)(d.turn >> 1), S = (int)d.S;
  float2* cs = reinterpret_cast<float2*>(smem);                                 // [tokens][half]
  TokenPlace* place = reinterpret_cast<TokenPlace*>(cs + w.tokens * half);      // [tokens]
  pdl_wait();
  pdl_trigger_work(RO_THREADS * 64 * K);
  const long long tok0 = (long long)(blockIdx.x / w.hblocks) * w.tokens, all = d.B * d.S;
  const int h0 = (blockIdx.x % w.hblocks) * w.heads;
  const int heads = min(w.heads, w.hq + w.hk + (d.k_pages ? w.hk : 0) - h0);
  const int tokens = (int)min((long long)w.tokens, all - tok0);
  const long long b0 = tok0 / d.S;
  const unsigned s0 = (unsigned)(tok0 - b0 * d.S);
  const auto token = [&](int t, long long& b, int& s) {
    const unsigned x = s0 + (unsigned)t;
    b = b0 + x / (unsigned)S, s = (int)(x % (unsigned)S);
  };
  const int items = tokens * heads * w.chunks;
  uint4 u0[K], u1[K];
  const auto item = [&](int i, int& t, int& h, int& o0, int& o1, bool& turn) {
    const unsigned c = (unsigned)i % (unsigned)w.chunks, r = (unsigned)i / (unsigned)w.chunks;
    h = h0 + (int)(r % (unsigned)heads), t = (int)(r / (unsigned)heads);
    turn = (int)c * 16 < (int)d.turn;
    const bool apart = turn && !INTER;
    o0 = apart ? c * 8 : c * 16, o1 = apart ? half + c * 8 : c * 16 + 8;
  };
  for (int i0 = 0; i0 < items; i0 += K * RO_THREADS) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int i = i0 + k * RO_THREADS + threadIdx.x;
      if (i >= items) break;
      int t, h, o0, o1, s;
      bool turn;
      long long b;
      item(i, t, h, o0, o1, turn);
      token(t, b, s);
      const T* src = h < w.hq ? (const T*)d.q + b * d.q_bs + s * d.q_ss + h * d.q_hs
                     : h < w.hq + w.hk ? (const T*)d.k + b * d.k_bs + s * d.k_ss + (h - w.hq) * d.k_hs
                                       : (const T*)d.v + b * d.v_bs + s * d.v_ss + (h - w.hq - w.hk) * d.v_hs;
      u0[k] = *reinterpret_cast<const uint4*>(src + o0), u1[k] = *reinterpret_cast<const uint4*>(src + o1);
    }
    if (i0 == 0) {
      for (int t = threadIdx.x; t < tokens; t += RO_THREADS) {
        long long b;
        int s;
        token(t, b, s);
        TokenPlace p = {-1, 0, !d.counts || s < d.counts[b]};
        if (d.k_pages && p.used) {
          const PagedTable table = {d.table, d.table_stride, d.table_cols, d.n_pages, (int)d.page_shift};
          const long long position = (long long)d.start[b] + s;
          p.page = paged_page(table, b, position);
          p.row = (int)paged_row(table, position);
          if (p.page < 0) ft_index_ok(-1, 1, status);
        }
        if (d.counts && d.k_pages && s == 0 && (d.counts[b] < 0 || d.counts[b] > S)) ft_index_ok(-1, 1, status);
        place[t] = p;
      }
      for (int e = threadIdx.x; e < tokens * half; e += RO_THREADS) {
        long long b;
        int s;
        token((int)((unsigned)e / (unsigned)half), b, s);
        const float2 c = turn_of((d.start ? d.start[b] : 0) + (long long)s, d.inv_freq[(unsigned)e % (unsigned)half]);
        cs[e] = make_float2(c.x, d.inverse ? -c.y : c.y);
      }
      __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int i = i0 + k * RO_THREADS + threadIdx.x;
      if (i >= items) break;
      int t, h, o0, o1, s;
      bool turn;
      long long b;
      item(i, t, h, o0, o1, turn);
      token(t, b, s);
      const TokenPlace p = place[t];
      T* dst;
      if (h < w.hq) {
        dst = (T*)d.q_out + b * d.qo_bs + s * d.qo_ss + h * d.qo_hs;
        turn = turn && p.used;
      } else {
        const bool is_k = h < w.hq + w.hk;
        const int g = is_k ? h - w.hq : h - w.hq - w.hk;
        turn = turn && is_k;
        if (d.k_pages) {
          if (p.page < 0) continue;
          dst = is_k ? (T*)d.k_pages + p.page * d.kp_ps + g * d.kp_hs + p.row * d.kp_rs
                     : (T*)d.v_pages + p.page * d.vp_ps + g * d.vp_hs + p.row * d.vp_rs;
        } else {
          dst = (T*)d.k_out + b * d.ko_bs + s * d.ko_ss + g * d.ko_hs;
        }
      }
      if (turn) {
        float a[16];
        up8<T>(u0[k], a);
        up8<T>(u1[k], a + 8);
        const float4* tc = reinterpret_cast<const float4*>(cs + t * half + (INTER ? o0 >> 1 : o0));      // two pairs each
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          const float4 f = tc[j >> 1];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float c = e ? f.z : f.x, sn = e ? f.w : f.y;
            float& x0 = INTER ? a[2 * (j + e)] : a[j + e];
            float& x1 = INTER ? a[2 * (j + e) + 1] : a[8 + j + e];
            const float y0 = x0 * c - x1 * sn, y1 = x1 * c + x0 * sn;
            x0 = y0, x1 = y1;
          }
        }
        u0[k] = down8<T>(a);
        u1[k] = down8<T>(a + 8);
      }
      *reinterpret_cast<uint4*>(dst + o0) = u0[k];
      *reinterpret_cast<uint4*>(dst + o1) = u1[k];
    }
  }
}

template <typename T, int K>
static int launch(const FtkRotaryDesc& d, const RotaryShape& w, long long blocks, cudaStream_t s) {
  const size_t smem = (size_t)w.tokens * ((d.turn >> 1) * sizeof(float2) + sizeof(TokenPlace));
  return d.interleaved ? launch_pdl(rotary_kernel<T, K, true>, dim3((unsigned)blocks), dim3(RO_THREADS), smem, s, d, w, ftk_status_word())
                       : launch_pdl(rotary_kernel<T, K, false>, dim3((unsigned)blocks), dim3(RO_THREADS), smem, s, d, w, ftk_status_word());
}

}  // namespace ftk
using namespace ftk;

extern "C" int ftk_rotary(const FtkRotaryDesc* d, void* stream) {
  if (!d || d->B <= 0 || d->S <= 0 || d->hd <= 0 || d->hd % 16 || d->turn < 0 || d->turn % 16 || d->turn > d->hd) return -2;
  if ((d->turn && !d->inv_freq) || (d->q && !d->q_out) || (d->type != FTK_T_BF16 && d->type != FTK_T_FP16)) return -2;
  if (d->k_pages ? !d->k || !d->v || !d->v_pages || !d->table || d->page_shift < 0 || d->page_shift > 30 : (d->k && !d->k_out)) return -2;
  const long long heads = (d->q ? d->Hq : 0) + (d->k ? d->Hkv : 0) + (d->k_pages ? d->Hkv : 0);
  if (heads <= 0 || heads > (1 << 20)) return -2;
  if (d->S > 0x3fffffff || d->B > (1ll << 40)) return -2;
  RotaryShape w = {};
  w.hq = d->q ? (int)d->Hq : 0, w.hk = d->k ? (int)d->Hkv : 0, w.chunks = (int)(d->hd >> 4);
  // Four items per thread where that still leaves several CTAs for each SM, fewer for small calls; tokens of a CTA share its
  // table of 4096 sines at most
  const long long items = d->B * d->S * heads * w.chunks, full = 148ll * 6 * RO_THREADS;
  const int per = items >= 4 * full ? 4 : (items >= 2 * full ? 2 : 1), most = per * RO_THREADS;
  w.heads = (int)(heads * w.chunks <= most ? heads : (most / w.chunks > 0 ? most / w.chunks : 1));
  w.hblocks = (int)((heads + w.heads - 1) / w.heads);
  long long tokens = w.hblocks > 1 ? 1 : most / (heads * w.chunks);
  const long long cap = d->turn ? 8192 / d->turn : 64;
  tokens = tokens > cap ? cap : tokens;
  tokens = tokens > 64 ? 64 : (tokens < 1 ? 1 : tokens);
  w.tokens = (int)tokens;
  const long long blocks = (d->B * d->S + tokens - 1) / tokens * w.hblocks;
  if (blocks > 0x7fffffff) return -2;
  cudaStream_t s = (cudaStream_t)stream;
  if (d->type == FTK_T_BF16)
    return per == 4 ? launch<__nv_bfloat16, 4>(*d, w, blocks, s) : per == 2 ? launch<__nv_bfloat16, 2>(*d, w, blocks, s) : launch<__nv_bfloat16, 1>(*d, w, blocks, s);
  return per == 4 ? launch<__half, 4>(*d, w, blocks, s) : per == 2 ? launch<__half, 2>(*d, w, blocks, s) : launch<__half, 1>(*d, w, blocks, s);
}
