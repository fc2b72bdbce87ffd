// Logits of a step on their way to a choice: penalties for repeated tokens, biases, a grammar's mask.
//
// Mathematics.  x = logit; where the token occurred in the row's history x = x / r if positive, else x r; x -= f n + p [n > 0] with n
// its count among the generated tokens; x += bias; -inf where the mask says no.  fp32, one rounding on the way out.
//
// What bounds it: each logit is read once and written once, a few operations in between; the copy bandwidth, and for a row or two
// the latency of two dependent reads.
//
// Work.  The vocabulary is cut into slices of up to 24 thousand columns; a unit is a slice of a row, and each CTA (two per SM)
// takes an equal run of the units.  For a unit it first counts the row's history into shared memory, a word per column -
// occurrences among the generated tokens in the low 31 bits, "occurred in the prompt" in bit 31; whole numbers, so the order of
// additions does not matter - and a bit per column that has any.  Then it streams the columns, 16 bytes per thread twice per
// tile, with the next tile (of the next unit at the end) and the next history already on their way; while one CTA counts the other
// streams.  Only columns whose bit is set are looked up and cleared.  A history is read once per slice, out of the L2 cache.
#include <math.h>

#include "ft_sm100.cuh"
#include "half_types.cuh"
#include "launch.cuh"
#include "ftk_api.h"

extern "C" int* ftk_status_word(void);

namespace ftk {

constexpr int LG_THREADS = 512;              // threads of a CTA at most
constexpr int LG_TOKENS = 4;                 // tokens of a history that a thread requests ahead
constexpr int LG_SLICE = 24 * 1024;          // columns of a slice at most
template <typename T> struct LgCols { static constexpr int value = 16 / (int)sizeof(T); };      // columns of 16 bytes

// A load that stays where it is written: ahead of what waits for others.  (Plain loads of the next tile end up behind the work on
// this one: 512 x 128003 with a history took 199 us instead.)
__device__ __forceinline__ uint4 load_now(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.cs.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ unsigned load_now(const unsigned char* p) {
  unsigned v;
  asm volatile("ld.global.u8 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ long long load_now(const long long* p) {
  long long v;
  asm volatile("ld.global.s64 %0, [%1];" : "=l"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ int load_now(const int* p) {
  int v;
  asm volatile("ld.global.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ float load_now(const float* p) {
  float v;
  asm volatile("ld.global.f32 %0, [%1];" : "=f"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ float4 load_now(const float4* p) {
  float4 v;
  asm volatile("ld.global.nc.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p) : "memory");
  return v;
}
template <typename T> __device__ __forceinline__ void floats(const uint4& v, float* f) { up8<T>(v, f); }
template <> __device__ __forceinline__ void floats<float>(const uint4& v, float* f) {
  f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y), f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
}
template <int N> __device__ __forceinline__ void write(float* p, const float* f) {
#pragma unroll
  for (int i = 0; i < N; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
}
template <int N, typename T> __device__ __forceinline__ void write(T* p, const float* f) {
  static_assert(N == 8, "16 bytes");
  *reinterpret_cast<uint4*>(p) = down8<T>(f);
}
__device__ __forceinline__ float load1(const float* p) { return *p; }
template <typename T> __device__ __forceinline__ float load1(const T* p) { return Half16<T>::one(*p); }
__device__ __forceinline__ void store1(float* p, float x) { *p = x; }
template <typename T> __device__ __forceinline__ void store1(T* p, float x) { *p = Half16<T>::round(x); }

// A row's history and what it costs.  x / r is x times the rounded 1 / r: off by one unit of fp32 more than a division, which
// would take as long as all the rest of a column.
struct LogitsRow {
  int len, prompt;
  float rep, inv, freq, pres;
  __device__ __forceinline__ float operator()(float x, unsigned c) const {
    const unsigned n = c & 0x7fffffffu;
    const float y = x > 0.f ? x * inv : x * rep;
    return n ? y - freq * (float)n - pres : y;
  }
};
struct LogitsCut {
  int slice, slices;      // columns of a slice (a multiple of 64), slices of the vocabulary
  bool bias16;            // rows of the bias start on 16 bytes
};
// VEC: rows of logits and results start on 16 bytes
template <typename T, typename O, bool HISTORY, bool VEC>
__global__ void __launch_bounds__(LG_THREADS, 2) logits_kernel(const __grid_constant__ FtkLogitsDesc d, const LogitsCut cut, int* status) {
  constexpr int N = LgCols<T>::value;
  extern __shared__ __align__(16) unsigned counts[];             // [slice], then a bit per column [slice / 32]
  unsigned* seen = counts + cut.slice;
  const int tid = threadIdx.x, bd = blockDim.x, slice = cut.slice, step = bd * N, tile = 2 * step;
  const long long units = d.R * cut.slices;
  const long long u0 = units * blockIdx.x / gridDim.x, u1 = units * (blockIdx.x + 1) / gridDim.x;
  if (HISTORY) {
    for (int i = tid; i < slice / 4; i += bd) reinterpret_cast<uint4*>(counts)[i] = make_uint4(0, 0, 0, 0);
    for (int i = tid; i < slice / 32; i += bd) seen[i] = 0;
  }
  pdl_wait();
  pdl_trigger();

  struct Unit {
    long long r, v0;        // row, first column
    int n, left;            // columns; units of the CTA from this one on
  };
  const auto columns_of = [&](long long v0) { return (int)max(0ll, min((long long)slice, d.V - v0)); };
  const auto behind = [&](const Unit& u) {
    const bool wrap = u.r + 1 == d.R;
    const long long v0 = wrap ? u.v0 + slice : u.v0;
    return Unit{wrap ? 0 : u.r + 1, v0, columns_of(v0), u.left - 1};
  };
  struct History {
    LogitsRow w;
    long long id[LG_TOKENS];
  };
  const auto request_history = [&](const Unit& u, History& h) {
    if (u.left <= 0) return;
    if (d.lengths) h.w.len = load_now(d.lengths + u.r);
    if (d.prompts) h.w.prompt = load_now(d.prompts + u.r);
    if (d.rep_rows) h.w.rep = load_now(d.rep_rows + u.r);
    if (d.freq_rows) h.w.freq = load_now(d.freq_rows + u.r);
    if (d.pres_rows) h.w.pres = load_now(d.pres_rows + u.r);
    const long long* p = d.tokens + u.r * d.ldt + tid;
#pragma unroll
    for (int i = 0; i < LG_TOKENS; ++i)
      if (i * bd + tid < d.L) h.id[i] = load_now(p + i * bd);
  };
  const auto count = [&](const Unit& u, const History& h) {
    if ((h.w.len < 0 || h.w.len > d.L) && tid == 0) ft_index_ok(-1, 1, status);
    const long long len = min((long long)h.w.len, d.L);
    const auto one = [&](long long j, long long id) {
      if (!ft_index_ok(id, d.V, status)) return;
      const int at = (int)(id - u.v0);
      if ((unsigned)at >= (unsigned)u.n) return;
      if (j < h.w.prompt) atomicOr(&counts[at], 0x80000000u);
      else atomicAdd(&counts[at], 1u);
      atomicOr(&seen[at >> 5], 1u << (at & 31));
    };
#pragma unroll
    for (int i = 0; i < LG_TOKENS; ++i)
      if (i * bd + tid < len) one(i * bd + tid, h.id[i]);
    for (long long j = (long long)LG_TOKENS * bd + tid; j < len; j += (long long)LG_TOKENS * bd) {
      long long id[LG_TOKENS];
#pragma unroll
      for (int i = 0; i < LG_TOKENS; ++i)
        if (j + i * bd < len) id[i] = load_now(d.tokens + u.r * d.ldt + j + i * bd);
#pragma unroll
      for (int i = 0; i < LG_TOKENS; ++i)
        if (j + i * bd < len) one(j + i * bd, id[i]);
    }
  };

  Unit u = {u0 % d.R, u0 / d.R * slice, 0, (int)(u1 - u0)};
  u.n = columns_of(u.v0);
  // the tile that is requested next: columns and mask bytes of its unit from this thread's on
  struct Tile {
    uint4 x[2];
    unsigned bits[2];
  };
  Unit f = u;
  int ft = 0;
  const T* fx = nullptr;
  const unsigned char* fm = nullptr;
  const auto aim = [&]() {
    fx = (const T*)d.logits + f.r * d.ld + f.v0 + tid * N;
    if (d.allowed) fm = reinterpret_cast<const unsigned char*>(d.allowed + f.r * d.allowed_rs) + ((f.v0 + tid * N) >> 3);
  };
  const auto request = [&](Tile& x) {
    if (f.left <= 0) return;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (ft + i * step + tid * N + N <= f.n) {
        x.x[i] = load_now(reinterpret_cast<const uint4*>(fx + i * step));
        if (d.allowed) x.bits[i] = load_now(fm + i * (step >> 3));
      }
    }
    ft += tile, fx += tile, fm += tile >> 3;
    if (ft >= f.n) {
      ft = 0, f = behind(f);
      aim();
    }
  };
  History h;
  h.w = {(int)min(d.L, 0x7fffffffll), 0, (float)d.rep, 1.f, (float)d.freq, (float)d.pres};
  if (HISTORY) request_history(u, h);
  Tile next;
  if (VEC) {
    aim();
    request(next);
  }
  for (; u.left > 0; u = behind(u)) {
    const int n = u.n;
    const long long r = u.r, v0 = u.v0;
    LogitsRow row = h.w;
    if (HISTORY) {
      __syncthreads();            // the counts and bits of the unit before are read and cleared
      count(u, h);
      row.inv = 1.f / row.rep;
      request_history(behind(u), h);
      __syncthreads();
    }
    O* out = (O*)d.out + r * d.ldo + v0;
    const float* bias = d.bias ? d.bias + r * d.bias_rs + v0 : nullptr;
    const unsigned shift = N == 8 ? 0 : (tid & 1) * 4;       // of this thread's bits in their byte
    for (int t0 = 0; t0 < n; t0 += tile) {
      if (VEC) {
        const Tile x = next;
        request(next);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int at = t0 + i * step + tid * N;
          if (at >= n) continue;
          const bool full = at + N <= n;
          float y[N], b[N];
          unsigned bits = ~0u;
          if (full) {
            floats<T>(x.x[i], y);
            if (d.allowed) bits = x.bits[i] >> shift;
          } else {                // the vocabulary's last columns
            if (d.allowed) bits = (unsigned)d.allowed[r * d.allowed_rs + ((v0 + at) >> 5)] >> (at & 31);
#pragma unroll
            for (int e = 0; e < N; ++e) y[e] = at + e < n ? load1((const T*)d.logits + r * d.ld + v0 + at + e) : 0.f;
          }
          if (bias) {
            if (full && cut.bias16) {
#pragma unroll
              for (int e = 0; e < N; e += 4) {
                const float4 p = __ldg(reinterpret_cast<const float4*>(bias + at + e));
                b[e] = p.x, b[e + 1] = p.y, b[e + 2] = p.z, b[e + 3] = p.w;
              }
            } else {
#pragma unroll
              for (int e = 0; e < N; ++e) b[e] = at + e < n ? __ldg(bias + at + e) : 0.f;
            }
          }
          if (HISTORY) {
            const unsigned k = seen[at >> 5] >> (at & 31) & ((1u << N) - 1);
            if (k) {
#pragma unroll
              for (int e = 0; e < N; ++e)
                if (k >> e & 1u) {
                  y[e] = row(y[e], counts[at + e]);
                  counts[at + e] = 0;
                }
              if (N == 8) reinterpret_cast<unsigned char*>(seen)[at >> 3] = 0;
              else atomicAnd(&seen[at >> 5], ~(15u << (at & 31)));      // the other half of the byte is a neighbour's
            }
          }
          if (bias) {
#pragma unroll
            for (int e = 0; e < N; ++e) y[e] += b[e];
          }
          if (d.allowed) {
#pragma unroll
            for (int e = 0; e < N; ++e) y[e] = bits >> e & 1u ? y[e] : -INFINITY;
          }
          if (full) {
            write<N>(out + at, y);
          } else {
#pragma unroll
            for (int e = 0; e < N; ++e)
              if (at + e < n) store1(out + at + e, y[e]);
          }
        }
      } else {
        for (int at = t0 + tid; at < min(n, t0 + tile); at += bd) {
          float y = load1((const T*)d.logits + r * d.ld + v0 + at);
          if (HISTORY && counts[at]) {
            y = row(y, counts[at]);
            counts[at] = 0;
          }
          if (bias) y += bias[at];
          if (d.allowed && !((unsigned)d.allowed[r * d.allowed_rs + ((v0 + at) >> 5)] >> (at & 31) & 1u)) y = -INFINITY;
          store1(out + at, y);
        }
      }
    }
  }
}

template <typename T, typename O, bool HISTORY, bool VEC>
static int launch(const FtkLogitsDesc& d, cudaStream_t s) {
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const long long places = 2ll * sms;
  // Slices as wide as a CTA holds, but 2048 columns where that keeps more SMs at work; among so many and a few times as many
  // the number that leaves the least to the CTA with the most units
  const long long want = max(2048ll, min((long long)LG_SLICE, (d.V * d.R + places - 1) / places));
  const long long least = (d.V + want - 1) / want;
  LogitsCut cut = {0, 0, ((uintptr_t)d.bias | (uintptr_t)(d.bias_rs * 4)) % 16 == 0};
  long long best = -1;
  for (long long k = least; k <= 4 * least && k < least + 16; ++k) {
    const long long slice = ((d.V + k - 1) / k + 63) / 64 * 64, slices = (d.V + slice - 1) / slice;
    const long long cost = (slices * d.R + places - 1) / places * (slice + (HISTORY ? 4096 : 512));      // a unit's fixed part, in columns
    if (best < 0 || cost < best) best = cost, cut.slice = (int)slice, cut.slices = (int)slices;
  }
  const long long vectors = (cut.slice + 2 * LgCols<T>::value - 1) / (2 * LgCols<T>::value);
  const int threads = (int)min((long long)LG_THREADS, max(128ll, (vectors + 31) / 32 * 32));
  const auto kernel = logits_kernel<T, O, HISTORY, VEC>;
  const auto bytes = [](int slice) { return HISTORY ? slice * 4 + slice / 8 : 0; };
  int rc = (int)cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes(LG_SLICE));
  if (rc) return rc;
  return launch_pdl(kernel, dim3((unsigned)min(places, cut.slices * d.R)), dim3(threads), bytes(cut.slice), s, d, cut, ftk_status_word());
}
template <typename T, typename O>
static int launch(const FtkLogitsDesc& d, cudaStream_t s) {
  const bool vec = ((uintptr_t)d.logits | (uintptr_t)(d.R > 1 ? d.ld * sizeof(T) : 0)) % 16 == 0 &&
                   ((uintptr_t)d.out | (uintptr_t)(d.R > 1 ? d.ldo * sizeof(O) : 0)) % 16 == 0;
  if (d.tokens && d.L > 0) return vec ? launch<T, O, true, true>(d, s) : launch<T, O, true, false>(d, s);
  return vec ? launch<T, O, false, true>(d, s) : launch<T, O, false, false>(d, s);
}

}  // namespace ftk
using namespace ftk;

extern "C" int ftk_logits(const FtkLogitsDesc* d, void* stream) {
  if (!d || d->R <= 0 || d->R > (1ll << 40) || d->V <= 0 || d->V > 0x7fffffff || !d->logits || !d->out) return -2;
  cudaStream_t s = (cudaStream_t)stream;
  if (d->type == FTK_T_FP32 && d->out_type == FTK_T_FP32) return launch<float, float>(*d, s);
  if (d->type == FTK_T_BF16 && d->out_type == FTK_T_FP32) return launch<__nv_bfloat16, float>(*d, s);
  if (d->type == FTK_T_FP16 && d->out_type == FTK_T_FP32) return launch<__half, float>(*d, s);
  if (d->type == FTK_T_BF16 && d->out_type == FTK_T_BF16) return launch<__nv_bfloat16, __nv_bfloat16>(*d, s);
  if (d->type == FTK_T_FP16 && d->out_type == FTK_T_FP16) return launch<__half, __half>(*d, s);
  return -2;
}
