// Logits of a step on their way to a choice: penalties for repeated tokens, biases, a grammar's mask.
//
// Mathematics.  x = logit; where the token occurred in the row's history x = x / r if positive, else x r; x -= f n + p [n > 0] with n
// its count among the generated tokens; x += bias; -inf where the mask says no.  fp32, one rounding on the way out.
//
// What bounds it: each logit is read once and written once, a few operations in between; the copy bandwidth, and for a row or two
// the latency of two dependent reads.
//
// Work.  The rows' columns behind one another, in blocks of 64, are cut into equal runs, one per SM; a run is some pieces of rows.
// For a piece the CTA first counts the row's history into shared memory, 16 bits per column - occurrences among the generated
// tokens in the low 15, "occurred in the prompt" in the highest; whole numbers, so the order of additions does not matter - and a bit
// per column that has any.  (Histories of 32768 tokens and more take 32 bits and half the columns.)  Then it streams the columns, 16
// bytes per thread twice per tile, with the next tile (of the next piece at the end) and the next history already on their way.
//
// What was measured (512 rows of 128003 bf16 columns with bias, mask and 2048 to 4096 tokens / 256 rows of 50257 fp32 columns with
// mask and 1024 to 2048 tokens; the copy bandwidth gives 43 / 16 us):
//   * a history is read once per piece and stops the stream, so pieces are as long as shared memory allows: 85 / 20.5 us with 64
//     thousand columns, 103 / 24 with two CTAs of 40 thousand, 112 / 33 with six narrow slices of every row; a cluster of CTAs that
//     share the counts of a row 185 / 50; warps of their own that count ahead of the stream 105 / 27;
//   * penalties where a column has a history are what the time goes by next: without them the first takes 56 us.  All eight
//     columns of a vector are done where one of them has its bit set, without a branch per column (that takes 89 / 22).
#include <math.h>

#include "ft_sm100.cuh"
#include "half_types.cuh"
#include "launch.cuh"
#include "ftk_api.h"

extern "C" int* ftk_status_word(void);

namespace ftk {

constexpr int LG_THREADS = 896;              // threads of a CTA at most
constexpr int LG_TOKENS = 4;                 // tokens of a history that a thread requests ahead
constexpr int LG_BLOCK = 64;                 // columns that stay together
template <typename T> struct LgCols { static constexpr int value = 16 / (int)sizeof(T); };      // columns of 16 bytes

// A load that stays where it is written: ahead of the work on what came before.
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
// would take as long as all the rest of a column.  Beyond 2^126 or below 2^-126 the normal numbers do not hold 1 / r: there x and r are
// multiplied by 2^-64 or 2^64 first, which is exact for every x whose quotient is neither 0 nor infinite.
struct LogitsRow {
  int len, prompt;
  float rep, up, inv, freq, pres;
  __device__ __forceinline__ void invert() {
    const float r = fabsf(rep);
    up = r < 0x1p-126f ? 0x1p64f : (r > 0x1p126f ? 0x1p-64f : 1.f);
    inv = 1.f / (rep * up);
  }
  __device__ __forceinline__ float operator()(float x, unsigned n) const {
    const float y = x > 0.f ? x * up * inv : x * rep;
    return n ? y - freq * (float)n - pres : y;
  }
};
// Counts of a piece's columns, 16 or 32 bits each in words of shared memory
template <bool WIDE> struct Counts {
  static constexpr int COLUMNS = WIDE ? 32 * 1024 : 64 * 1024;      // of a piece at most
  static constexpr unsigned PROMPT = WIDE ? 0x80000000u : 0x8000u;
  unsigned* words;
  __device__ __forceinline__ void add(int at, unsigned n) {
    if (WIDE) atomicAdd(&words[at], n);
    else atomicAdd(&words[at >> 1], n << (at & 1) * 16);
  }
  __device__ __forceinline__ void mark(int at) {
    if (WIDE) atomicOr(&words[at], PROMPT);
    else atomicOr(&words[at >> 1], PROMPT << (at & 1) * 16);
  }
  __device__ __forceinline__ unsigned operator[](int at) const {      // of the generated tokens
    return (WIDE ? words[at] : reinterpret_cast<const unsigned short*>(words)[at]) & (PROMPT - 1);
  }
  template <int N> __device__ __forceinline__ void clear(int at) {       // N columns from a multiple of N on
    if (WIDE) {
#pragma unroll
      for (int i = 0; i < N; i += 4) *reinterpret_cast<uint4*>(words + at + i) = make_uint4(0, 0, 0, 0);
    } else if (N == 8) {
      *reinterpret_cast<uint4*>(words + at / 2) = make_uint4(0, 0, 0, 0);
    } else {
      *reinterpret_cast<uint2*>(words + at / 2) = make_uint2(0, 0);
    }
  }
};
struct LogitsCut {
  long long blocks;       // of a row
  int columns;            // of a piece at most
  bool bias16;            // rows of the bias start on 16 bytes
};

// VEC: rows of logits and results start on 16 bytes
template <typename T, typename O, bool HISTORY, bool VEC, bool WIDE>
__global__ void __launch_bounds__(LG_THREADS, 1) logits_kernel(const __grid_constant__ FtkLogitsDesc d, const LogitsCut cut, int* status) {
  constexpr int N = LgCols<T>::value;
  extern __shared__ __align__(16) unsigned smem[];               // counts, a bit per column, tokens
  Counts<WIDE> counts = {smem};
  unsigned* seen = smem + cut.columns / (WIDE ? 1 : 2);
  long long* ids = reinterpret_cast<long long*>(seen + cut.columns / 32);      // [LG_TOKENS][threads]
  const int tid = threadIdx.x, bd = blockDim.x, step = bd * N, tile = 2 * step;
  const long long x0 = d.R * cut.blocks * blockIdx.x / gridDim.x, x1 = d.R * cut.blocks * (blockIdx.x + 1) / gridDim.x;
  if (HISTORY) {
    for (int i = tid; i < cut.columns / (WIDE ? 4 : 8); i += bd) reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
    for (int i = tid; i < cut.columns / 32; i += bd) seen[i] = 0;
  }
  pdl_wait();
  pdl_trigger();

  struct Unit {
    int r, v0, left, n;           // row, first column; blocks of the CTA from here on; columns
  };
  const auto unit = [&](int r, int v0, int left) {
    return Unit{r, v0, left, min(min(left, cut.columns / LG_BLOCK) * LG_BLOCK, (int)d.V - v0)};
  };
  const auto behind = [&](const Unit& u) {
    const int v = u.v0 + u.n, left = u.left - (u.n + LG_BLOCK - 1) / LG_BLOCK;
    return v == (int)d.V ? unit(u.r + 1, 0, left) : unit(u.r, v, left);
  };
  // a thread's tokens of the next history wait in shared memory, for itself
  const auto request_history = [&](const Unit& u, LogitsRow& w) {
    if (u.left <= 0) return;
    if (d.lengths) w.len = load_now(d.lengths + u.r);
    if (d.prompts) w.prompt = load_now(d.prompts + u.r);
    if (d.rep_rows) w.rep = load_now(d.rep_rows + u.r);
    if (d.freq_rows) w.freq = load_now(d.freq_rows + u.r);
    if (d.pres_rows) w.pres = load_now(d.pres_rows + u.r);
    const long long* p = d.tokens + u.r * d.ldt + tid;
#pragma unroll
    for (int i = 0; i < LG_TOKENS; ++i)
      if (i * bd + tid < (int)d.L)
        asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_u32(ids + i * bd + tid)), "l"(p + i * bd) : "memory");
  };
  const auto count = [&](const Unit& u, const LogitsRow& w) {
    asm volatile("cp.async.wait_all;" ::: "memory");
    if ((w.len < 0 || w.len > (int)d.L) && tid == 0) ft_index_ok(-1, 1, status);
    const int len = min(w.len, (int)d.L);
    const auto one = [&](int j, long long id) {
      if (!ft_index_ok(id, d.V, status)) return;
      const int at = (int)(id - u.v0);
      if ((unsigned)at >= (unsigned)u.n) return;
      if (j < w.prompt) counts.mark(at);
      else counts.add(at, 1);
      atomicOr(&seen[at >> 5], 1u << (at & 31));
    };
#pragma unroll
    for (int i = 0; i < LG_TOKENS; ++i)
      if (i * bd + tid < len) one(i * bd + tid, ids[i * bd + tid]);
    for (int j = LG_TOKENS * bd + tid; j < len; j += bd) one(j, d.tokens[u.r * d.ldt + j]);
  };

  Unit u = unit((int)(x0 / cut.blocks), (int)(x0 % cut.blocks) * LG_BLOCK, (int)(x1 - x0));
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
  LogitsRow h = {(int)d.L, 0, (float)d.rep, 1.f, 1.f, (float)d.freq, (float)d.pres};
  if (HISTORY) request_history(u, h);
  Tile next;
  if (VEC) {
    aim();
    request(next);
  }
  for (; u.left > 0; u = behind(u)) {
    const int n = u.n, v0 = u.v0;
    const long long r = u.r;
    LogitsRow row = h;
    if (HISTORY) {
      __syncthreads();            // the counts and bits of the unit before are read and cleared
      count(u, h);
      row.invert();
      request_history(behind(u), h);
      __syncthreads();
    }
    O* out = (O*)d.out + r * d.ldo + v0;
    const float* bias = d.bias ? d.bias + r * d.bias_rs + v0 : nullptr;
    const unsigned shift = N == 8 ? 0 : (tid & 1) * 4;       // of this thread's bits in their byte
    // A column as it leaves, with its penalties, bias and mask
    const auto leave = [&](int at, float x, bool penalised) {
      if (penalised) x = row(x, counts[at]);
      if (bias) x += __ldg(bias + at);
      if (d.allowed && !((unsigned)d.allowed[r * d.allowed_rs + ((v0 + at) >> 5)] >> (at & 31) & 1u)) x = -INFINITY;
      store1(out + at, x);
    };
    // The bits of N columns that have a history; they and the counts are cleared by forget()
    const auto bits_of = [&](int at) -> unsigned {
      if (!HISTORY) return 0;
      return reinterpret_cast<const unsigned char*>(seen)[at >> 3] >> (N == 8 ? 0 : at & 4) & ((1u << N) - 1);
    };
    const auto forget = [&](int at) {
      counts.template clear<N>(at);
      if (N == 8) reinterpret_cast<unsigned char*>(seen)[at >> 3] = 0;
      else atomicAnd(&seen[at >> 5], ~(15u << (at & 31)));      // the other half of the byte is a neighbour's
    };
    // a vector of columns, all of them there
    const auto vector = [&](int at, const uint4& x, unsigned bits) {
      float y[N];
      floats<T>(x, y);
      const unsigned k = bits_of(at);
      if (k) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float v = row(y[e], counts[at + e]);
          y[e] = k >> e & 1u ? v : y[e];
        }
        forget(at);
      }
      if (bias) {
        if (cut.bias16) {
#pragma unroll
          for (int e = 0; e < N; e += 4) {
            const float4 p = __ldg(reinterpret_cast<const float4*>(bias + at + e));
            y[e] += p.x, y[e + 1] += p.y, y[e + 2] += p.z, y[e + 3] += p.w;
          }
        } else {
#pragma unroll
          for (int e = 0; e < N; ++e) y[e] += __ldg(bias + at + e);
        }
      }
      if (d.allowed) {
        bits >>= shift;
#pragma unroll
        for (int e = 0; e < N; ++e) y[e] = bits >> e & 1u ? y[e] : -INFINITY;
      }
      write<N>(out + at, y);
    };
    const auto few = [&](int from) {      // up to N columns, one by one
      const unsigned k = bits_of(from);
      for (int e = 0; e < N && from + e < n; ++e) leave(from + e, load1((const T*)d.logits + r * d.ld + v0 + from + e), k >> e & 1u);
      if (k) forget(from);
    };
    for (int t0 = 0; t0 < n; t0 += tile) {
      const int at = t0 + tid * N;
      if (VEC) {
        const Tile x = next;
        request(next);
        if (t0 + tile <= n) {
          vector(at, x.x[0], x.bits[0]);
          vector(at + step, x.x[1], x.bits[1]);
        } else {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int from = at + i * step;
            if (from + N <= n) vector(from, x.x[i], x.bits[i]);
            else if (from < n) few(from);      // the vocabulary's last columns
          }
        }
      } else {
        for (int from = at; from < min(n, t0 + tile); from += step) few(from);
      }
    }
  }
}

template <typename T, typename O, bool HISTORY, bool VEC, bool WIDE>
static int launch(const FtkLogitsDesc& d, cudaStream_t s) {
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const long long row = (d.V + LG_BLOCK - 1) / LG_BLOCK;
  const long long ctas = max(1ll, min((long long)sms, row * d.R * LG_BLOCK / 2048));      // 2048 columns at least
  const long long run = (row * d.R + ctas - 1) / ctas * LG_BLOCK;
  const int columns = (int)min((long long)Counts<WIDE>::COLUMNS, min(run, row * LG_BLOCK));
  const LogitsCut cut = {row, columns, ((uintptr_t)d.bias | (uintptr_t)(d.bias_rs * 4)) % 16 == 0};
  // threads for the columns of a short run, or for a long history
  const long long vectors = max((columns + 2 * LgCols<T>::value - 1) / (2ll * LgCols<T>::value), HISTORY ? d.L / LG_TOKENS : 0ll);
  const int threads = (int)min((long long)LG_THREADS, max(128ll, (vectors + 31) / 32 * 32));
  const auto kernel = logits_kernel<T, O, HISTORY, VEC, WIDE>;
  const auto bytes = [](int n, int threads) { return HISTORY ? n * (WIDE ? 4 : 2) + n / 8 + LG_TOKENS * threads * 8 : 0; };
  int rc = (int)cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes(Counts<WIDE>::COLUMNS, LG_THREADS));
  if (rc) return rc;
  return launch_pdl(kernel, dim3((unsigned)ctas), dim3(threads), bytes(columns, threads), s, d, cut, ftk_status_word());
}
template <typename T, typename O, bool VEC>
static int launch(const FtkLogitsDesc& d, cudaStream_t s) {
  if (!d.tokens || d.L == 0) return launch<T, O, false, VEC, false>(d, s);
  return d.L < 0x8000 ? launch<T, O, true, VEC, false>(d, s) : launch<T, O, true, VEC, true>(d, s);
}
template <typename T, typename O>
static int launch(const FtkLogitsDesc& d, cudaStream_t s) {
  const bool vec = ((uintptr_t)d.logits | (uintptr_t)(d.R > 1 ? d.ld * sizeof(T) : 0)) % 16 == 0 &&
                   ((uintptr_t)d.out | (uintptr_t)(d.R > 1 ? d.ldo * sizeof(O) : 0)) % 16 == 0;
  return vec ? launch<T, O, true>(d, s) : launch<T, O, false>(d, s);
}

}  // namespace ftk
using namespace ftk;

extern "C" int ftk_logits(const FtkLogitsDesc* d, void* stream) {
  if (!d || !d->logits || !d->out || d->L < 0 || d->L > (1 << 30) || d->R <= 0 || d->R > 0x7fffffff || d->V <= 0 || d->V > 0x7fffffff - (1 << 20) ||
      d->R * ((d->V + 63) / 64) > (1ll << 38))
    return -2;
  cudaStream_t s = (cudaStream_t)stream;
  if (d->type == FTK_T_FP32 && d->out_type == FTK_T_FP32) return launch<float, float>(*d, s);
  if (d->type == FTK_T_BF16 && d->out_type == FTK_T_FP32) return launch<__nv_bfloat16, float>(*d, s);
  if (d->type == FTK_T_FP16 && d->out_type == FTK_T_FP32) return launch<__half, float>(*d, s);
  if (d->type == FTK_T_BF16 && d->out_type == FTK_T_BF16) return launch<__nv_bfloat16, __nv_bfloat16>(*d, s);
  if (d->type == FTK_T_FP16 && d->out_type == FTK_T_FP16) return launch<__half, __half>(*d, s);
  return -2;
}
