// Keys and values of new tokens into a paged cache of 8-bit floating point (e4m3) with a scale per block of rows and head, the keys
// turned by position on the way, and the queries with them.
//
// Mathematics.  A block's new elements x (keys after the rotation, in fp32) with the largest finite magnitude a get the scale
// s = 2^e, the smallest with a <= 448 s; a block that has earlier rows keeps the larger of s and its own s', and its rows become
// y s' / s.  An element is x / s, rounded once.
//
// What bounds it: each element is read once, and written once in one or (queries) two bytes; the copy bandwidth, and for a handful of tokens
// the latency of a position, a page number and a scale behind one another.
//
// Work.  A CTA has the tokens of a call that fall into one block of rows of a sequence, and some of their heads: it forms the angles' sines
// and cosines once per token and pair.  A unit is one head of those tokens, of the keys, the values or the queries; a group of as many
// lanes as have one to four items of 16 elements each takes units in turn, holds a unit's elements in registers until their largest is
// known (through shared memory where a group is several warps), and writes them.  Queries in a launch of their own took 75.5 us
// where they took 71.0 with the rest (16 prompts of up to 2048, 16 + 4 heads of 128), and 81.4 against 79.6 (8 x 2048, 16 + 16 heads).
// Measured: those prompts 68.3 us, 3600 GB/s of what the call needs and 4900 with the queries behind the counts, which leave as they came;
// a token of 256 sequences, 16 heads of 128, 4.6 us; one token, 12 heads of 64, 2.8 us.  What holds the long calls are chains of instructions
// of few warps (three or four CTAs to an SM, issuing in 59 % of the cycles).  The rotation is done twice, before the largest is known and
// after: turned elements held as floats are too many registers (with two items a lane 75.9, 90.7 and 34.7 us for the prompts and the two
// calls below, where turning twice took 77.4, 88.6 and 32.0).
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
// Items of a unit that a lane holds: one where a warp has a lane for each, else four, so that a group of few warps holds a block and the
// elements come once.  One, two and four, before the bounds below (us): a token of 256 sequences 5.8, 6.3, 7.5; 8 x 2048 tokens of 16 heads
// of 128 -, 88.3, 81.5; 16 x 2048 of 4 heads without queries -, 32.0, 28.4.
constexpr int A8_ONE = 1, A8_MORE = 4;
// CTAs of an SM that the registers are bounded for.  With one item a lane six, where five fit without a bound: 4.6 us for the 256 sequences
// and 5.8 (seven 5.1).  With four items a lane four or three (152 registers): in groups of up to 64 lanes, 25.3 and 28.2 us for the call without
// queries, 68.3 and 71.1 for 16 ragged prompts, 11.9 and 13.7 for 8 x 1024 tokens of 12 heads of 64; a group of 128 lanes, where all warps
// wait for one another, 83.0 and 79.7 for the 16 heads of 128, 8.9 and 8.3 for 16 x 40 tokens of 16 + 4 heads.
constexpr int A8_CTAS_ONE = 6, A8_CTAS = 4, A8_CTAS_WIDE = 3;

struct AppendShape {
  long long blocks;                    // blocks of rows that a sequence's tokens can touch
  int lanes;                           // of a group: a power of two
  int units, parts;                    // units of a CTA, CTAs that share the units of a block
  int hq;                              // heads of the queries that take part
};

// HELD: items of a lane, CTAS: of an SM.  TABLE: sines and cosines in shared memory; else (more than 200 KB of them) where they are used
template <typename T, bool INTER, bool TABLE, int HELD, int CTAS>
__global__ void __launch_bounds__(A8_THREADS, CTAS) append_e4m3_kernel(const __grid_constant__ FtkRotaryDesc d, const __grid_constant__ AppendShape w, int* status) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float largest[2][A8_THREADS / 32];
  // Cosines and sines of two pairs, (c, c', s, s'), as [token][two pairs of an item][items]: the items' lanes read 16 bytes side by side
  float4* cs = reinterpret_cast<float4*>(smem);
  const int half = (int)(d.turn >> 1), chunks = (int)(d.hd >> 4), L = w.lanes, l = threadIdx.x & (L - 1), group = threadIdx.x / (unsigned)L;
  const int groups = A8_THREADS / (unsigned)L;
  pdl_wait();
  pdl_trigger();
  const long long cta = blockIdx.x / (unsigned)w.parts, b = cta / w.blocks, j = cta % w.blocks;
  const int first = (int)(blockIdx.x % (unsigned)w.parts) * w.units, all = 2 * (int)d.Hkv + w.hq, units = min(w.units, all - first);
  const long long start = d.start[b];
  int count = (int)d.S;
  if (d.counts) {
    count = d.counts[b];
    if (count < 0 || count > d.S) {
      if (j == 0 && first == 0 && threadIdx.x == 0) ft_index_ok(-1, 1, status);
      count = count < 0 ? 0 : (int)d.S;
    }
  }
  const long long row0 = ((start >> d.block_shift) + j) << d.block_shift;      // the block's first position
  const int s0 = (int)max(0ll, row0 - start), s1 = (int)min((long long)d.S, row0 + (1ll << d.block_shift) - start);      // its tokens of the call
  if (s0 >= s1) return;
  const int fresh = max(0, min(s1, count) - s0);      // tokens for the cache
  // this lane's items of a unit: 16 elements of a token, eight whole pairs
  int tok[HELD], chunk[HELD];
#pragma unroll
  for (int k = 0; k < HELD; ++k) tok[k] = (l + k * L) / (unsigned)chunks, chunk[k] = (l + k * L) % (unsigned)chunks;
  const auto place = [&](int c, bool apart, int& o0, int& o1) { o0 = apart ? c * 8 : c * 16, o1 = apart ? half + c * 8 : c * 16 + 8; };
  const auto fetch = [&](int unit, int t, int c, uint4& u, uint4& v) {
    const int g = first + unit, kv = (int)d.Hkv;
    const bool key = g < kv, query = g >= 2 * kv;
    const T* at = key ? (const T*)d.k + b * d.k_bs + g * d.k_hs + (long long)(s0 + t) * d.k_ss
                : query ? (const T*)d.q + b * d.q_bs + (g - 2 * kv) * d.q_hs + (long long)(s0 + t) * d.q_ss
                        : (const T*)d.v + b * d.v_bs + (g - kv) * d.v_hs + (long long)(s0 + t) * d.v_ss;
    int o0, o1;
    place(c, !INTER && c * 16 < (int)d.turn && (key || query), o0, o1);
    u = *reinterpret_cast<const uint4*>(at + o0), v = *reinterpret_cast<const uint4*>(at + o1);
  };
  uint4 u[HELD], v[HELD], u_next[HELD], v_next[HELD];
  const auto fetch_all = [&](int unit) {
    const int n = unit < units ? (first + unit < 2 * (int)d.Hkv ? fresh : s1 - s0) : 0;
#pragma unroll
    for (int k = 0; k < HELD; ++k)
      if (tok[k] < n) fetch(unit, tok[k], chunk[k], u_next[k], v_next[k]);
  };
  fetch_all(group);
  for (int e = threadIdx.x; e < fresh * half && TABLE; e += A8_THREADS) {
    const int i = (int)((unsigned)e % (unsigned)half), t = (int)((unsigned)e / (unsigned)half);
    const float2 a = turn_of(start + s0 + t, d.inv_freq[i]);
    float* to = reinterpret_cast<float*>(cs + t * (half >> 1) + ((i & 7) >> 1) * (half >> 3) + (i >> 3)) + (i & 1);
    to[0] = a.x, to[2] = a.y;
  }
  // where the block is
  const PagedTable table = {d.table, d.table_stride, d.table_cols, d.n_pages, (int)d.page_shift};
  const int old = (int)(row0 < start ? start - row0 : 0);      // rows in front of the new ones
  long long page = -1, in = 0;
  if (fresh > 0) {
    page = paged_page(table, b, row0), in = paged_row(table, row0);
    if (page < 0 && first == 0 && threadIdx.x == 0) ft_index_ok(-1, 1, status);
  }
  __syncthreads();

  // an item in fp32, turned where it is one to turn
  const auto turned = [&](const uint4& a, const uint4& c, int t, int ch, bool turns, float (&x)[16]) {
    up8<T>(a, x), up8<T>(c, x + 8);
    if (!turns || ch * 16 >= (int)d.turn) return;
    const float4* tc = cs + t * (half >> 1) + ch;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float4 f;
      if (TABLE) {
        f = tc[e * (half >> 3)];
      } else {
        const float2 y = turn_of(start + s0 + t, d.inv_freq[ch * 8 + 2 * e]), z = turn_of(start + s0 + t, d.inv_freq[ch * 8 + 2 * e + 1]);
        f = make_float4(y.x, z.x, y.y, z.y);
      }
      if (INTER) {
#pragma unroll
        for (int o = 0; o < 2; ++o) {
          float &p = x[4 * e + 2 * o], &q = x[4 * e + 2 * o + 1];
          const float co = o ? f.y : f.x, si = o ? f.w : f.z, y = p * co - q * si;
          q = q * co + p * si;
          p = y;
        }
      } else {              // the first and second elements of two pairs
        const f32x2 x0 = pk2(x[2 * e], x[2 * e + 1]), x1 = pk2(x[8 + 2 * e], x[8 + 2 * e + 1]), co = pk2(f.x, f.y), si = pk2(f.z, f.w);
        const float2 p = up2(fma2(x0, co, mul2(x1, pk2(-f.z, -f.w)))), q = up2(fma2(x1, co, mul2(x0, si)));
        x[2 * e] = p.x, x[2 * e + 1] = p.y, x[8 + 2 * e] = q.x, x[8 + 2 * e + 1] = q.y;
      }
    }
  };
  int turn_of_units = 0;
  for (int base = 0; base < units; base += groups, turn_of_units ^= 1) {
    const int unit = base + group, g = first + unit;
    const bool key = g < (int)d.Hkv, cache = g < 2 * (int)d.Hkv;
#pragma unroll
    for (int k = 0; k < HELD; ++k) u[k] = u_next[k], v[k] = v_next[k];
    fetch_all(unit + groups);            // the next unit, on its way while this one is worked on
    if (unit < units && !cache) {      // queries: turned, and as they are behind the sequence's tokens
      T* const to = (T*)d.q_out + b * d.qo_bs + (g - 2 * d.Hkv) * d.qo_hs;
      const auto put = [&](int t, int c, const uint4& a, const uint4& e) {
        int o0, o1;
        place(c, !INTER && c * 16 < (int)d.turn, o0, o1);
        T* at = to + (long long)(s0 + t) * d.qo_ss;
        uint4 y0 = a, y1 = e;
        if (t < fresh && c * 16 < (int)d.turn) {
          float x[16];
          turned(a, e, t, c, true, x);
          y0 = down8<T>(x), y1 = down8<T>(x + 8);
        }
        *reinterpret_cast<uint4*>(at + o0) = y0, *reinterpret_cast<uint4*>(at + o1) = y1;
      };
#pragma unroll
      for (int k = 0; k < HELD; ++k)
        if (tok[k] < s1 - s0) put(tok[k], chunk[k], u[k], v[k]);
      for (int i = l + HELD * L; i < (s1 - s0) * chunks; i += L) {
        uint4 a, e;
        fetch(unit, i / chunks, i % chunks, a, e);
        put(i / chunks, i % chunks, a, e);
      }
    }
    float most = 0.f;
    const bool mine = unit < units && cache && page >= 0;
    // the largest: NaN is not counted, and infinities only in the first place
    const auto largest_of = [&](auto finite) {
      float top = 0.f, x[16];
#pragma unroll
      for (int k = 0; k < HELD; ++k) {
        if (tok[k] < fresh) {
          turned(u[k], v[k], tok[k], chunk[k], key, x);
#pragma unroll
          for (int e = 0; e < 16; ++e) top = fmaxf(top, finite() ? finite_size(x[e]) : fabsf(x[e]));
        }
      }
      for (int i = l + HELD * L; i < fresh * chunks; i += L) {
        uint4 a, e;
        fetch(unit, i / chunks, i % chunks, a, e);
        turned(a, e, i / chunks, i % chunks, key, x);
#pragma unroll
        for (int o = 0; o < 16; ++o) top = fmaxf(top, finite() ? finite_size(x[o]) : fabsf(x[o]));
      }
      return top;
    };
    const auto yes = []() { return true; };
    const auto no = []() { return false; };
    if (mine) most = largest_of(no);
    const auto over_group = [&](float most) {
      for (int o = 1; o < min(L, 32); o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
      if (L > 32) {      // (two sets of words: a warp may be a unit ahead)
        if ((threadIdx.x & 31) == 0) largest[turn_of_units][threadIdx.x >> 5] = most;
        __syncthreads();
        for (int o = 0; o < L / 32; ++o) most = fmaxf(most, largest[turn_of_units][group * (L / 32) + o]);
      }
      return most;
    };
    most = over_group(most);
    bool odd = most == INFINITY;         // some are infinite: once more without them
    if (L > 32 ? __syncthreads_or(odd) : __any_sync(0xffffffffu, odd)) most = over_group(odd && mine ? largest_of(yes) : most);
    float* scale = nullptr;
    float s = e4m3_scale(most), had = s;
    if (mine) {
      const int h = key ? g : g - (int)d.Hkv;
      scale = (key ? d.k_scales + page * d.ks_ps + h * d.ks_hs : d.v_scales + page * d.vs_ps + h * d.vs_hs) + (in >> d.block_shift);
      if (old) had = *scale;
    }
    if (old) {      // all of a group have read it before one writes it
      if (L > 32) __syncthreads();
      else __syncwarp();
    }
    if (!mine) continue;
    const int h = key ? g : g - (int)d.Hkv;
    unsigned char* rows = key ? (unsigned char*)d.k_pages + page * d.kp_ps + h * d.kp_hs + in * d.kp_rs : (unsigned char*)d.v_pages + page * d.vp_ps + h * d.vp_hs + in * d.vp_rs;
    const long long rs = key ? d.kp_rs : d.vp_rs;
    if (old) {
      if (!(had >= s)) {      // the rows that are there, under the larger scale
        const float by = had / s;
        for (int i = l; i < old * chunks; i += L) {
          uint4* at = reinterpret_cast<uint4*>(rows + i / chunks * rs + i % chunks * 16);
          uint4 y = *at;
          uint32_t* q = reinterpret_cast<uint32_t*>(&y);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 lo = e4m3_floats(q[k] & 0xffffu), hi = e4m3_floats(q[k] >> 16);
            q[k] = e4m3_pair(lo.x * by, lo.y * by) | e4m3_pair(hi.x * by, hi.y * by) << 16;
          }
          *at = y;
        }
      } else {
        s = had;
      }
    }
    if (l == 0) *scale = s;
    const float by = 1.f / s;
    const auto put = [&](int t, int c, const uint4& a, const uint4& e, auto finite) {
      float x[16];
      turned(a, e, t, c, key, x);
      uint32_t y[4];
#pragma unroll
      for (int o = 0; o < 4; ++o) {
        const float *p = x + 4 * o;
        y[o] = finite() ? e4m3_finite(p[0] * by, p[1] * by) | e4m3_finite(p[2] * by, p[3] * by) << 16
                        : e4m3_pair(p[0] * by, p[1] * by) | e4m3_pair(p[2] * by, p[3] * by) << 16;
      }
      int o0, o1;
      place(c, key && !INTER && c * 16 < (int)d.turn, o0, o1);
      unsigned char* to = rows + (long long)(old + t) * rs;
      if (o1 == o0 + 8) {
        *reinterpret_cast<uint4*>(to + o0) = make_uint4(y[0], y[1], y[2], y[3]);
      } else {
        *reinterpret_cast<uint2*>(to + o0) = make_uint2(y[0], y[1]);
        *reinterpret_cast<uint2*>(to + o1) = make_uint2(y[2], y[3]);
      }
    };
    const auto put_all = [&](auto finite) {
#pragma unroll
      for (int k = 0; k < HELD; ++k)
        if (tok[k] < fresh) put(tok[k], chunk[k], u[k], v[k], finite);
      for (int i = l + HELD * L; i < fresh * chunks; i += L) {
        uint4 a, e;
        fetch(unit, i / chunks, i % chunks, a, e);
        put(i / chunks, i % chunks, a, e, finite);
      }
    };
    if (odd) put_all(no);
    else put_all(yes);
  }
}

template <typename T, int HELD, int CTAS>
static int launch(const FtkRotaryDesc& d, AppendShape w, cudaStream_t s) {
  const long long ctas = d.B * w.blocks * w.parts, tokens = d.S < (1ll << d.block_shift) ? d.S : 1ll << d.block_shift;
  if (ctas > 0x7fffffff) return -2;
  size_t bytes = (size_t)tokens * (d.turn >> 1) * sizeof(float2);
  const bool table = bytes <= 200 * 1024;
  if (!table) bytes = 0;
  const auto kernel = d.interleaved ? (table ? append_e4m3_kernel<T, true, true, HELD, CTAS> : append_e4m3_kernel<T, true, false, HELD, CTAS>)
                                    : (table ? append_e4m3_kernel<T, false, true, HELD, CTAS> : append_e4m3_kernel<T, false, false, HELD, CTAS>);
  if (bytes > 40 * 1024) {
    const int rc = (int)cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
    if (rc) return rc;
  }
  return launch_pdl(kernel, dim3((unsigned)ctas), dim3(A8_THREADS), bytes, s, d, w, ftk_status_word());
}

}  // namespace ftk
using namespace ftk;

extern "C" int ftk_append_e4m3(const FtkRotaryDesc* d, void* stream) {
  if (!d || d->B <= 0 || d->S <= 0 || d->Hkv <= 0 || d->hd <= 0 || d->hd % 16 || d->turn < 0 || d->turn % 16 || d->turn > d->hd) return -2;
  if ((d->turn && !d->inv_freq) || (d->type != FTK_T_BF16 && d->type != FTK_T_FP16) || (d->q && !d->q_out)) return -2;
  if (!d->k || !d->v || !d->k_pages || !d->v_pages || !d->k_scales || !d->v_scales || !d->table || !d->start) return -2;
  if (d->page_shift < 0 || d->page_shift > 30 || d->block_shift < 0 || d->block_shift > 6 || d->block_shift > d->page_shift) return -2;
  if (d->S > 0x3fffffff || d->B > (1 << 30) || d->Hkv > (1 << 20) || (d->q && (d->Hq < 0 || d->Hq > (1 << 20)))) return -2;
  AppendShape w = {};
  w.hq = d->q ? (int)d->Hq : 0;
  const long long block = 1ll << d->block_shift, tokens = d->S < block ? d->S : block, items = tokens * (d->hd >> 4), all = 2 * d->Hkv + w.hq;
  w.blocks = (d->S + block - 2) / block + 1;
  // A lane per item up to a warp's, then up to four items a lane
  for (w.lanes = 4; w.lanes < A8_THREADS && (items > 32 ? w.lanes < 32 || items > (long long)A8_MORE * w.lanes : items > w.lanes);) w.lanes *= 2;
  // Heads are shared out among CTAs where there are too few for the SMs
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const long long groups = A8_THREADS / w.lanes, most = (all + groups - 1) / groups, want = (6ll * sms + d->B * w.blocks - 1) / (d->B * w.blocks);
  const long long parts = want < most ? want : most;
  w.units = (int)((all + parts - 1) / parts);
  w.parts = (int)((all + w.units - 1) / w.units);
  const cudaStream_t s = (cudaStream_t)stream;
  const bool bf = d->type == FTK_T_BF16;
  if (items <= w.lanes) return bf ? launch<__nv_bfloat16, A8_ONE, A8_CTAS_ONE>(*d, w, s) : launch<__half, A8_ONE, A8_CTAS_ONE>(*d, w, s);
  if (w.lanes < A8_THREADS) return bf ? launch<__nv_bfloat16, A8_MORE, A8_CTAS>(*d, w, s) : launch<__half, A8_MORE, A8_CTAS>(*d, w, s);
  return bf ? launch<__nv_bfloat16, A8_MORE, A8_CTAS_WIDE>(*d, w, s) : launch<__half, A8_MORE, A8_CTAS_WIDE>(*d, w, s);
}
