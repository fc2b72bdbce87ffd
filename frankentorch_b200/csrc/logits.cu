// Logits of a step on their way to a choice: penalties for repeated tokens, biases, a grammar's mask.
//
// Mathematics.  x = logit; where the token occurred in the row's history x = x / r if positive, else x r; x -= f n + p [n > 0] with n
// its count among the generated tokens; x += bias; -inf where the mask says no.  fp32, one rounding on the way out.
//
// What bounds it: each logit is read once and written once, a few operations in between; the copy bandwidth, and for a row or two
// the latency of three dependent reads and two barriers.
//
// Work.  A row belongs to a cluster of up to eight CTAs, each with a slice of the vocabulary: its columns in registers (requested
// before anything else) and a count per column in shared memory - occurrences among the generated tokens in the low 31 bits,
// "occurred in the prompt" in bit 31; whole numbers, so the order of additions does not matter.  Each CTA reads its share of the
// history once and counts into the slice of whichever CTA of the cluster has the token, so the history is read once per row
// rather than once per slice.  Rows without a history have no counts and no clusters.
#include <math.h>

#include "ft_sm100.cuh"
#include "half_types.cuh"
#include "launch.cuh"
#include "ftk_api.h"

extern "C" int* ftk_status_word(void);

namespace ftk {

constexpr int LG_THREADS = 512, LG_COLS = 8, LG_VECS = 4;            // columns of a vector, vectors a thread holds
constexpr int LG_SLICE = LG_THREADS * LG_COLS * LG_VECS;             // columns that a CTA holds at a time
constexpr int LG_CLUSTER = 8;

template <typename T> struct Row8 {      // eight columns as they are in memory
  uint4 v[sizeof(T) * LG_COLS / 16];
};
template <typename T> __device__ __forceinline__ Row8<T> read8(const T* p) {
  Row8<T> r;
#pragma unroll
  for (int i = 0; i < (int)(sizeof(r) / 16); ++i) r.v[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
  return r;
}
__device__ __forceinline__ void floats(const Row8<float>& r, float* f) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    f[4 * i] = __uint_as_float(r.v[i].x), f[4 * i + 1] = __uint_as_float(r.v[i].y);
    f[4 * i + 2] = __uint_as_float(r.v[i].z), f[4 * i + 3] = __uint_as_float(r.v[i].w);
  }
}
template <typename T> __device__ __forceinline__ void floats(const Row8<T>& r, float* f) { up8<T>(r.v[0], f); }
__device__ __forceinline__ void write8(float* p, const float* f) {
  reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
}
template <typename T> __device__ __forceinline__ void write8(T* p, const float* f) { *reinterpret_cast<uint4*>(p) = down8<T>(f); }
__device__ __forceinline__ float load1(const float* p) { return *p; }
template <typename T> __device__ __forceinline__ float load1(const T* p) { return Half16<T>::one(*p); }
__device__ __forceinline__ void store1(float* p, float x) { *p = x; }
template <typename T> __device__ __forceinline__ void store1(T* p, float x) { *p = Half16<T>::round(x); }

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// One more occurrence (or the prompt's bit) in the counts of CTA `rank` of the cluster.
__device__ __forceinline__ void count_at(uint32_t own, int rank, bool prompt) {
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(own), "r"(rank));
  if (prompt) asm volatile("red.relaxed.cluster.shared::cluster.or.b32 [%0], %1;" ::"r"(at), "r"(0x80000000u) : "memory");
  else asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], %1;" ::"r"(at), "r"(1u) : "memory");
}

struct Penalties {
  float rep, freq, pres;
  __device__ __forceinline__ float operator()(float x, unsigned c) const {
    if (c) {
      x = x > 0.f ? x / rep : x * rep;
      const unsigned n = c & 0x7fffffffu;
      if (n) x = x - freq * (float)n - pres;
    }
    return x;
  }
};

// VEC: rows of logits and results start on 16 bytes (of the bias too where BIAS16).
template <typename T, typename O, bool HISTORY, bool VEC>
__global__ void __launch_bounds__(LG_THREADS, 2) logits_kernel(const __grid_constant__ FtkLogitsDesc d, int slice, int ctas, bool bias16, int* status) {
  extern __shared__ __align__(16) unsigned counts[];
  pdl_wait();
  pdl_trigger();
  const long long r = blockIdx.x / ctas;
  const int rank = blockIdx.x % ctas;
  const T* in = (const T*)d.logits + r * d.ld;
  O* out = (O*)d.out + r * d.ldo;
  const float* bias = d.bias ? d.bias + r * d.bias_rs : nullptr;
  const int* allowed = d.allowed ? d.allowed + r * d.allowed_rs : nullptr;
  Penalties pen = {1.f, 0.f, 0.f};
  long long len = 0, prompt = 0;
  if (HISTORY) {
    pen.rep = d.rep_rows ? d.rep_rows[r] : (float)d.rep;
    pen.freq = d.freq_rows ? d.freq_rows[r] : (float)d.freq;
    pen.pres = d.pres_rows ? d.pres_rows[r] : (float)d.pres;
    len = d.L;
    if (d.lengths) {
      len = d.lengths[r];
      if (len < 0 || len > d.L) ft_index_ok(-1, 1, status);
      len = len < 0 ? 0 : (len > d.L ? d.L : len);
    }
    if (d.prompts) prompt = d.prompts[r];
  }
  // one round for vocabularies of up to ctas * LG_SLICE columns
  for (long long from = 0; from < d.V; from += (long long)slice * ctas) {
    const long long v0 = from + (long long)rank * slice;
    const int n = (int)max(0ll, min((long long)slice, d.V - v0));
    Row8<T> x[LG_VECS];
    if (VEC) {
#pragma unroll
      for (int i = 0; i < LG_VECS; ++i) {
        const int c = (i * LG_THREADS + threadIdx.x) * LG_COLS;
        if (c + LG_COLS <= n) x[i] = read8(in + v0 + c);
      }
    }
    if (HISTORY) {
      for (int i = threadIdx.x; i < slice / 4; i += LG_THREADS) reinterpret_cast<uint4*>(counts)[i] = make_uint4(0, 0, 0, 0);
      if (ctas > 1) cluster_barrier();
      else __syncthreads();
      for (long long j = (long long)rank * LG_THREADS + threadIdx.x; j < len; j += (long long)ctas * LG_THREADS) {
        const long long id = d.tokens[r * d.ldt + j];
        if (!ft_index_ok(id, d.V, status)) continue;
        if (id < from || id >= from + (long long)slice * ctas) continue;
        const int at = (int)(id - from), owner = at / slice;
        if (ctas > 1) count_at(smem_u32(counts + (at - owner * slice)), owner, j < prompt);
        else if (j < prompt) atomicOr(&counts[at], 0x80000000u);
        else atomicAdd(&counts[at], 1u);
      }
      if (ctas > 1) cluster_barrier();
      else __syncthreads();
    }
    const auto column = [&](int c) {
      float y = load1(in + v0 + c);
      if (HISTORY) y = pen(y, counts[c]);
      if (bias) y += bias[v0 + c];
      if (allowed && !((unsigned)allowed[(v0 + c) >> 5] >> ((v0 + c) & 31) & 1u)) y = -INFINITY;
      store1(out + v0 + c, y);
    };
    if (VEC) {
#pragma unroll
      for (int i = 0; i < LG_VECS; ++i) {
        const int c = (i * LG_THREADS + threadIdx.x) * LG_COLS;
        if (c + LG_COLS > n) {
          for (int e = c; e < n; ++e) column(e);
          break;
        }
        float y[LG_COLS];
        floats(x[i], y);
        if (HISTORY) {
          const uint4 a = *reinterpret_cast<const uint4*>(counts + c), b = *reinterpret_cast<const uint4*>(counts + c + 4);
          if (a.x | a.y | a.z | a.w | b.x | b.y | b.z | b.w) {
            y[0] = pen(y[0], a.x), y[1] = pen(y[1], a.y), y[2] = pen(y[2], a.z), y[3] = pen(y[3], a.w);
            y[4] = pen(y[4], b.x), y[5] = pen(y[5], b.y), y[6] = pen(y[6], b.z), y[7] = pen(y[7], b.w);
          }
        }
        if (bias) {
          if (bias16) {
            const float4 a = __ldg(reinterpret_cast<const float4*>(bias + v0 + c)), b = __ldg(reinterpret_cast<const float4*>(bias + v0 + c) + 1);
            y[0] += a.x, y[1] += a.y, y[2] += a.z, y[3] += a.w, y[4] += b.x, y[5] += b.y, y[6] += b.z, y[7] += b.w;
          } else {
#pragma unroll
            for (int e = 0; e < LG_COLS; ++e) y[e] += __ldg(bias + v0 + c + e);
          }
        }
        if (allowed) {
          const unsigned bits = reinterpret_cast<const unsigned char*>(allowed)[(v0 + c) >> 3];
#pragma unroll
          for (int e = 0; e < LG_COLS; ++e) y[e] = bits >> e & 1u ? y[e] : -INFINITY;
        }
        write8(out + v0 + c, y);
      }
    } else {
      for (int c = threadIdx.x; c < n; c += LG_THREADS) column(c);
    }
    if (HISTORY && from + (long long)slice * ctas < d.V) {      // the counts are read before another CTA's next round could write them
      if (ctas > 1) cluster_barrier();
      else __syncthreads();
    }
  }
}

template <typename T, typename O, bool HISTORY, bool VEC>
static int launch(const FtkLogitsDesc& d, cudaStream_t s) {
  // As few CTAs per row as hold it, or so many that some hundreds are at work, with no less than 2048 columns each
  const long long fit = (d.V + LG_SLICE - 1) / LG_SLICE, wide = (d.V + 2047) / 2048, idle = 444 / d.R;
  const long long ctas = min((long long)LG_CLUSTER, max(fit, min(wide, max(1ll, idle))));
  const int slice = (int)min((long long)LG_SLICE, ((d.V + ctas - 1) / ctas + 63) / 64 * 64);
  const size_t smem = HISTORY ? (size_t)slice * 4 : 0;
  const bool bias16 = ((uintptr_t)d.bias | (uintptr_t)(d.bias_rs * 4)) % 16 == 0;
  const auto kernel = logits_kernel<T, O, HISTORY, VEC>;
  int rc = (int)cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, LG_SLICE * 4);
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(ctas * d.R));
  cfg.blockDim = dim3(LG_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)ctas;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = HISTORY && ctas > 1 ? 2 : 1;
  return (int)cudaLaunchKernelEx(&cfg, kernel, d, slice, (int)ctas, bias16, ftk_status_word());
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
  if (!d || d->R <= 0 || d->R > (1 << 27) || d->V <= 0 || d->V > 0x7fffffff || !d->logits || !d->out) return -2;
  cudaStream_t s = (cudaStream_t)stream;
  if (d->type == FTK_T_FP32 && d->out_type == FTK_T_FP32) return launch<float, float>(*d, s);
  if (d->type == FTK_T_BF16 && d->out_type == FTK_T_FP32) return launch<__nv_bfloat16, float>(*d, s);
  if (d->type == FTK_T_FP16 && d->out_type == FTK_T_FP32) return launch<__half, float>(*d, s);
  if (d->type == FTK_T_BF16 && d->out_type == FTK_T_BF16) return launch<__nv_bfloat16, __nv_bfloat16>(*d, s);
  if (d->type == FTK_T_FP16 && d->out_type == FTK_T_FP16) return launch<__half, __half>(*d, s);
  return -2;
}
