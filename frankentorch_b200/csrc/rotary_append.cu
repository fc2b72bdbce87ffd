// Rotation of queries and keys by position, in training (forward, and backward with the opposite angle) and on the way into a
// paged key-value cache.
//
// Mathematics.  A pair (x0, x1) of a token at position p is turned by a = p w: (x0 cos a - x1 sin a, x1 cos a + x0 sin a).  The
// backward pass is the inverse rotation of the gradient.  Far positions turn thousands of times, so the angle is formed and
// reduced to a fraction of a turn in 64 bits (2^28 turns at position 2^31 leave 2^-24 of a turn); sine and cosine of the fraction and the products
// are fp32, each output is rounded once.
//
// What bounds it: each element is read once and written once; the copy bandwidth, and for a handful of tokens the latency of a
// position, a page number and a row behind one another.
//
// Work is divided into items of 16 elements of one head of one token: two 16-byte vectors that hold eight whole pairs (the
// vectors are turn / 2 apart where pairs are (i, i + turn / 2), else neighbours), so an item can be turned in place.  A CTA has some
// tokens with all their heads, a thread the same elements of every so-manieth head of them: it requests its items, two at a time,
// and while they arrive the CTA forms the angles' sines and cosines once per token and pair and looks up the tokens' places.
// Offsets of tokens are in shared memory: worked out per item they were the larger part of 250 instructions per 64 bytes.
// Forward and backward of 4 x 2048 tokens of 16 heads of 128 take 48 us, 5.6 TB/s.
#include "ft_sm100.cuh"
#include "half_types.cuh"
#include "launch.cuh"
#include "ftk_api.h"
#include "paged_cache.h"
#include "rotary.cuh"

extern "C" int* ftk_status_word(void);

namespace ftk {

constexpr int RO_THREADS = 128;

// A token of a CTA: offsets of its rows in the inputs and outputs, and whether it takes part
struct Token {
  long long q, k, v, q_out, k_out, v_out;
  int used, placed;      // counted among the sequence's tokens; has a place for its key and value
};
struct RotaryShape {
  int tokens, heads, hblocks;      // of a CTA; CTAs that share the heads of a token
  int hq, hk, chunks;              // heads of the queries and of the cache that take part, items of a head
};

template <typename T, int K, bool INTER>
__global__ void __launch_bounds__(RO_THREADS) rotary_kernel(const __grid_constant__ FtkRotaryDesc d, const __grid_constant__ RotaryShape w,
                                                            int* status) {
  extern __shared__ __align__(16) unsigned char smem[];
  const int half = (int)(d.turn >> 1), S = (int)d.S;
  // Cosines and sines of two pairs, (c, c', s, s'), as [token][two pairs of an item][items]: the items' threads read 16 bytes side by side
  float4* cs = reinterpret_cast<float4*>(smem);
  Token* tok = reinterpret_cast<Token*>(cs + w.tokens * half / 2);        // [tokens]
  pdl_wait();
  pdl_trigger();      // a CTA has 8 KB and more to move
  const bool append = d.k_pages != nullptr;
  const long long tok0 = (long long)(blockIdx.x / (unsigned)w.hblocks) * w.tokens, all = d.B * d.S;
  const int h0 = (int)(blockIdx.x % (unsigned)w.hblocks) * w.heads;
  const int heads = min(w.heads, w.hq + w.hk + (append ? w.hk : 0) - h0);
  const int tokens = (int)min((long long)w.tokens, all - tok0);
  const long long b0 = tok0 / d.S;
  const unsigned s0 = (unsigned)(tok0 - b0 * d.S);
  const auto place = [&](int t, long long& b, int& s) {
    const unsigned x = s0 + (unsigned)t;
    b = b0 + x / (unsigned)S, s = (int)(x % (unsigned)S);
  };
  for (int t = threadIdx.x; t < tokens; t += RO_THREADS) {
    long long b;
    int s;
    place(t, b, s);
    Token& k = tok[t];
    k.q = b * d.q_bs + s * d.q_ss, k.k = b * d.k_bs + s * d.k_ss, k.v = b * d.v_bs + s * d.v_ss;
    k.q_out = b * d.qo_bs + s * d.qo_ss, k.k_out = b * d.ko_bs + s * d.ko_ss;
    k.used = 1;
    if (d.counts) {
      const int n = d.counts[b];
      k.used = s < n;
      if (append && s == 0 && (n < 0 || n > S)) ft_index_ok(-1, 1, status);
    }
  }
  __syncthreads();
  // this thread's elements of a head, and its first head and token
  const int c = threadIdx.x % (unsigned)w.chunks, step = RO_THREADS / (unsigned)w.chunks, lane = threadIdx.x / (unsigned)w.chunks;
  const bool turned = c * 16 < (int)d.turn, apart = turned && !INTER;
  const int o0 = apart ? c * 8 : c * 16, o1 = apart ? half + c * 8 : c * 16 + 8;
  const int dt = step / heads, dh = step % heads;
  int t = lane < step ? lane / heads : tokens, h = lane % heads;
  for (bool first = true; first || t < tokens; first = false) {
    uint4 u0[K], u1[K];
    int tt = t, hh = h;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (tt < tokens) {
        const int g = h0 + hh;
        const T* src = g < w.hq ? (const T*)d.q + tok[tt].q + g * d.q_hs
                       : g < w.hq + w.hk ? (const T*)d.k + tok[tt].k + (g - w.hq) * d.k_hs
                                         : (const T*)d.v + tok[tt].v + (g - w.hq - w.hk) * d.v_hs;
        if (g < w.hq || !append || tok[tt].used) {
          u0[k] = *reinterpret_cast<const uint4*>(src + o0), u1[k] = *reinterpret_cast<const uint4*>(src + o1);
        }
      }
      tt += dt, hh += dh;
      if (hh >= heads) hh -= heads, ++tt;
    }
    if (first) {
      for (int i = threadIdx.x; i < tokens && append; i += RO_THREADS) {
        Token& k = tok[i];
        k.placed = 0;
        if (!k.used) continue;
        long long b;
        int s;
        place(i, b, s);
        const PagedTable table = {d.table, d.table_stride, d.table_cols, d.n_pages, (int)d.page_shift};
        const long long position = (long long)d.start[b] + s, page = paged_page(table, b, position), row = paged_row(table, position);
        if (page < 0) {
          ft_index_ok(-1, 1, status);
          continue;
        }
        k.placed = 1;
        k.k_out = page * d.kp_ps + row * d.kp_rs, k.v_out = page * d.vp_ps + row * d.vp_rs;
      }
      for (int e = threadIdx.x; e < tokens * half; e += RO_THREADS) {
        long long b;
        int s;
        const int i = (int)((unsigned)e % (unsigned)half), t = (int)((unsigned)e / (unsigned)half);
        place(t, b, s);
        const float2 a = turn_of((d.start ? d.start[b] : 0) + (long long)s, d.inv_freq[i]);
        float* to = reinterpret_cast<float*>(cs + t * (half >> 1) + ((i & 7) >> 1) * (half >> 3) + (i >> 3)) + (i & 1);
        to[0] = a.x, to[2] = d.inverse ? -a.y : a.y;
      }
      __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (t < tokens) {
        const int g = h0 + h;
        const bool is_q = g < w.hq, is_k = !is_q && g < w.hq + w.hk;
        const Token& o = tok[t];
        T* dst = is_q ? (T*)d.q_out + o.q_out + g * d.qo_hs
                 : append ? (is_k ? (T*)d.k_pages + o.k_out + (g - w.hq) * d.kp_hs : (T*)d.v_pages + o.v_out + (g - w.hq - w.hk) * d.vp_hs)
                          : (T*)d.k_out + o.k_out + (g - w.hq) * d.ko_hs;
        if (turned && (is_q ? o.used : is_k)) {
          const float4* tc = cs + t * (half >> 1) + c;
          uint32_t* x = reinterpret_cast<uint32_t*>(&u0[k]);      // words of two elements
          uint32_t* y = reinterpret_cast<uint32_t*>(&u1[k]);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float4 f = tc[j * (half >> 3)];
            if (INTER) {          // words 2 j and 2 j + 1 of the item hold a pair each
              uint32_t& p = j < 2 ? x[2 * j] : y[2 * j - 4];
              uint32_t& q = j < 2 ? x[2 * j + 1] : y[2 * j - 3];
              const float2 a = Half16<T>::up(p), b = Half16<T>::up(q);
              p = Half16<T>::down(a.x * f.x - a.y * f.z, a.y * f.x + a.x * f.z);
              q = Half16<T>::down(b.x * f.y - b.y * f.w, b.y * f.y + b.x * f.w);
            } else {              // the first and second elements of two pairs
              const float2 a = Half16<T>::up(x[j]), b = Half16<T>::up(y[j]);
              const f32x2 x0 = pk2(a.x, a.y), x1 = pk2(b.x, b.y), cc = pk2(f.x, f.y), sn = pk2(f.z, f.w);
              const float2 u = up2(fma2(x0, cc, mul2(x1, pk2(-f.z, -f.w)))), v = up2(fma2(x1, cc, mul2(x0, sn)));
              x[j] = Half16<T>::down(u.x, u.y), y[j] = Half16<T>::down(v.x, v.y);
            }
          }
        }
        if (is_q || !append || o.placed) {
          *reinterpret_cast<uint4*>(dst + o0) = u0[k];
          *reinterpret_cast<uint4*>(dst + o1) = u1[k];
        }
      }
      t += dt, h += dh;
      if (h >= heads) h -= heads, ++t;
    }
  }
}

template <typename T, int K>
static int launch(const FtkRotaryDesc& d, const RotaryShape& w, long long blocks, cudaStream_t s) {
  const size_t smem = (size_t)w.tokens * ((d.turn >> 1) * sizeof(float2) + sizeof(Token));
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
  // Two items per thread at a time where that leaves several CTAs for each SM, and up to four rounds of them per CTA in large calls:
  // what a CTA does once (places, sines, its launch) takes as long as two rounds.  4 x 2048 x 16 x 128 twice / 16 ragged prompts: one
  // round 52.0 / 87.6 us, two 47.9 / 67.0, four 49.0 / 59.7, eight 51.6 / 63.9; four items at a time, one round 49.2 / 69.2.
  // Tokens of a CTA share its table of 4096 sines at most.
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const long long items = d->B * d->S * heads * w.chunks, full = 8ll * sms * RO_THREADS;
  const int per = items >= 2 * full ? 2 : 1, rounds = items >= 16 * full ? 4 : (items >= 8 * full ? 2 : 1);
  const int most = rounds * per * (RO_THREADS / w.chunks) * w.chunks;
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
  if (d->type == FTK_T_BF16) return per == 2 ? launch<__nv_bfloat16, 2>(*d, w, blocks, s) : launch<__nv_bfloat16, 1>(*d, w, blocks, s);
  return per == 2 ? launch<__half, 2>(*d, w, blocks, s) : launch<__half, 1>(*d, w, blocks, s);
}
