// The choice of a token from the logits of a step: temperature, top-k, top-p, min-p, and a given random number.
//
// Mathematics.  Weights are whole numbers, w_i = 2^43 exp((x_i - max x) / T) rounded, so their sums (63 bits for up to 2^20 tokens) are
// exact whatever their order, and a row's choice is a function of its logits, settings and random number alone.  With tokens in the
// order of their logits (equal ones by their ids): the first k; of those the ones before which less than p of the sum lies; of those the
// ones of at least min_p of the largest; then the first by id whose running sum passes u times the sum.
//
// What bounds it: each logit is read once.  A weight takes 10 operations in 64 bits, at half the rate of fp32, so where all are needed they are
// next: with what is around them 6 to 7 cycles of an SM for 32.
//
// Work.  A cluster of CTAs has a row, each an equal run of its columns, which it keeps in shared memory (rows of more than that are read
// again from L2): everything behind the first pass works there.  The CTAs read one another's sums, histograms and lists over
// distributed shared memory, a warp of each for all of it, and come to the same conclusions.
//   * The k largest of a small k are among the elements that reach the k-th largest of 256 maxima, of as many parts of the row: hardly more
//     than k.  They become a list, ordered by counting, and the rest is done on it by one CTA.
//   * Else the border of top-k and of top-p is looked for in two steps: counts of 2048 equal steps of the logits' range say between which
//     two logits it is, and the elements between them are set aside.  For top-p the same pass has the sum of all weights and of those
//     above, the only time that all weights are formed.  What is set aside is divided further until it is one value, whose elements are
//     taken by their ids, or a short list.
//   * The choice: sums per warp in the order of the ids, the warp with the target, the 32 vectors, the lane.
// The random sums of shared memory's counters take 10 cycles of an SM for 32 elements; collectives of a cluster 1500 cycles each.
//
// Measured: 256 rows of 50257 fp32, 51 MB in 22 us with the largest alone, 36 with k = 50 and p, 84 with k = 200, 74 - 93 with p = 0.9, 46
// with the whole distribution, 66 with settings that change from row to row; 512 rows of 128003 bf16 with p = 0.9 268; one
// row of 50257 with k = 50 and p 8, 64 with the whole distribution 15 a call.  Reading is a small part of it.  Of the 66 us the SMs issue in 43 % of
// the cycles, of the 268 in 53 %, with 64-bit arithmetic in 9 and 13 %: barriers, the CTA's own and the cluster's, are the largest stall
// (3.6 and 4.1 of 8 and 11 cycles of a warp per instruction).
//
// Registers are bounded for four CTAs to an SM, 64 each, which leaves 8 to 204 bytes of spills.  Bounded for three, where nothing spills, and five:
// the 66 us become 65.4 and 69.7, the 268 302 and 279, the 15.3 of 64 whole distributions 19.1 and 15.6, the 84 of k = 200 82.8 and 84.9.
#include <math.h>

#include <type_traits>

#include "ft_sm100.cuh"
#include "half_types.cuh"
#include "launch.cuh"
#include "ftk_api.h"

namespace ftk {

typedef unsigned long long u64;
#define SA_INLINE __attribute__((always_inline))      // left out of line, a lambda keeps what it captures in local memory
constexpr int SA_LOG = 8, SA_THREADS = 1 << SA_LOG, SA_WARPS = SA_THREADS / 32;
constexpr int SA_BINS = 8 * SA_THREADS;      // steps of a histogram of counts
constexpr int SA_FINE = 2 * SA_THREADS;      // steps among the elements set aside
constexpr int SA_ASIDE = 512;          // elements that a CTA can set aside
constexpr int SA_LIST = SA_THREADS;    // elements of a list: one per thread
constexpr int SA_CLUSTER = 8;          // CTAs of a row at most
constexpr int SA_STEPS = 128;          // vectors of a lane at most
constexpr int SA_SHARE = 176 * 1024;   // bytes of a row that a CTA keeps at most
static_assert(SA_WARPS == 8, "a lane for each of four sums of the warps");

template <typename T> __device__ __forceinline__ void logits_of(const uint4& v, float (&x)[8]) { up8<T>(v, x); }
template <typename T> __device__ __forceinline__ void logits_of(const uint4& v, float (&x)[4]) {
  x[0] = __uint_as_float(v.x), x[1] = __uint_as_float(v.y), x[2] = __uint_as_float(v.z), x[3] = __uint_as_float(v.w);
}
__device__ __forceinline__ float logit_of(const float* p) { return *p; }
template <typename T> __device__ __forceinline__ float logit_of(const T* p) { return Half16<T>::one(*p); }
template <typename T> __device__ __forceinline__ uint32_t minus_infinity();      // as many as 32 bits hold
template <> __device__ __forceinline__ uint32_t minus_infinity<float>() { return 0xff800000u; }
template <> __device__ __forceinline__ uint32_t minus_infinity<__nv_bfloat16>() { return 0xff80ff80u; }
template <> __device__ __forceinline__ uint32_t minus_infinity<__half>() { return 0xfc00fc00u; }
// Whole numbers in the order of the logits (0 and -0 are equal), and back
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float ordered(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }
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
// All threads of the row's CTAs have come here, and what they wrote to shared memory is seen by all: one fence for a CTA's threads, which
// its own barrier has put in front of it (a fence of each warp takes three times as long)
__device__ __forceinline__ void cluster_sync() {
  __syncthreads();
  if (threadIdx.x == 0) asm volatile("fence.acq_rel.cluster;" ::: "memory");
  __syncwarp();
  asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// In two halves, for the end of a kernel: nobody leaves while its words are read
__device__ __forceinline__ void leave_arrive() {
  __syncthreads();
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
}
__device__ __forceinline__ void leave_wait() {
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t there(const void* mine, int rank) {      // the same place of another CTA's shared memory
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(mine)), "r"(rank));
  return r;
}
__device__ __forceinline__ u64 peek(const u64* p, int rank) {
  u64 v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(there(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t peek(const uint32_t* p, int rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(there(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <typename V> __device__ __forceinline__ V warp_upto(V v) {      // running sum over the lanes
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V w = __shfl_up_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) >= o) v += w;
  }
  return v;
}
__device__ __forceinline__ float max_or_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

struct SampleShared {
  u64 aside[SA_ASIDE];                 // order and inverted id, as in a list
  union {
    u64 mass[SA_FINE];                 // published: sums of weights per step
    struct {
      u64 sorted[SA_LIST], value[SA_LIST];
    };
  };
  u64 list[SA_LIST];                   // published
  double table[256];                   // 2^(i / 256)
  u64 steps[SA_STEPS];
  u64 sums[2][SA_WARPS];               // published: per warp, in the order of the ids
  u64 words[2][4];                     // published: of the CTA
  u64 record[2][2];                    // published: what the CTA with it has found
  u64 part[SA_WARPS][4];               // of the CTA's warps
  u64 got[8];                          // what all threads learn
  uint32_t hist[SA_BINS];              // published: counts per step
  uint32_t maxima[SA_THREADS];         // published: of parts of the row
  uint32_t n_list, n_aside;
};
constexpr int SA_OWN = (sizeof(SampleShared) + 15) / 16 * 16;      // bytes of a CTA beside its part of the row
constexpr int SA_THREE = (228 * 1024 / 3 - 1024 - SA_OWN) / (SA_THREADS * 16);      // steps up to which three CTAs share an SM's memory
static_assert(SA_THREE == 13, "the sizes measured at the launcher are on either side of it");
static_assert(SA_OWN <= 48 * 1024 && SA_OWN + SA_SHARE <= 227 * 1024, "a CTA's shared memory, where it keeps none of the row and where it keeps the most");

// A row's settings.  2^43 exp((x - top) / T): 2^(k / 256) out of the table, the rest by four terms of the exponential series, up to
// (ln(2) / 512)^4 / 24 (the next one is 2^-54), and by adding 2^9 a number of up to 1 is rounded to units of 2^-43.  What is rounded is within
// 2^-8 of the exact number of units: z exp(-z) 2^43, 0.37 2^43 at most, times the 2^-52 by which z = (top - x) / T is off, and some
// roundings of the result.
struct Weigh {
  const double* table;
  double top, by;                      // 256 log2(e) / T
  float floor;                         // what is below weighs less than half a unit
  __device__ __forceinline__ u64 operator()(float x) const {      // x >= floor
    constexpr double MAGIC = 6755399441055744.0;      // 1.5 2^52
    const double d = (double)x - top, kd = fma(d, by, MAGIC), r = fma(d, by, MAGIC - kd);
    const int k = __double2loint(kd);
    constexpr double C = 0.0027076061740622863;       // ln(2) / 256
    const double p = r * fma(r, fma(r, fma(r, C * C * C * C / 24, C * C * C / 6), C * C / 2), C), t = table[k & 255];
    double v = fma(t, p, t);
    v = __hiloint2double(__double2hiint(v) + (int)((uint32_t)(k & ~255) << 12), __double2loint(v)) + 512.0;
    return (u64)(uint32_t)(__double2hiint(v) - 0x40800000) << 32 | (uint32_t)__double2loint(v);
  }
};

template <typename T, bool RES, bool VEC>
__global__ void __launch_bounds__(SA_THREADS, 4) sample_kernel(const __grid_constant__ FtkSampleDesc d, const int its) {
  constexpr int N = 16 / (int)sizeof(T), STEP = 32 * N;      // elements of a vector, of a warp's step
  extern __shared__ __align__(16) unsigned char smem[];
  SampleShared& s = *reinterpret_cast<SampleShared*>(smem);
  uint4* kept_row = reinterpret_cast<uint4*>(smem + SA_OWN);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, V = (int)d.V;
  const int rank = (int)cluster_rank(), lc = (int)d.cluster, C = 1 << lc;
  const long long r = blockIdx.x >> lc;
  const int begin = (rank * SA_WARPS + warp) * its * STEP;      // this warp's run of columns
  const int mine = max(0, min(its, (V - begin + STEP - 1) / STEP));
  if (tid < 256) s.table[tid] = exp2(tid * (1.0 / 256));
  for (int i = tid; i < SA_BINS; i += SA_THREADS) s.hist[i] = 0;
  if (tid == 0) s.n_list = s.n_aside = 0;
  pdl_wait();
  pdl_trigger();
  const T* row = (const T*)d.logits + r * d.ld;
  const float t = d.temp_rows ? d.temp_rows[r] : (float)d.temp, p = d.p_rows ? d.p_rows[r] : (float)d.p, least = d.min_rows ? d.min_rows[r] : (float)d.min_p;
  const float u = d.uniform[r];
  const long long k0 = d.k_rows ? d.k_rows[r] : d.k;

  const auto fetch = [&](int first) {      // a vector of the row, -inf behind its end
    if (VEC && first + N <= V) return __ldg(reinterpret_cast<const uint4*>(row + first));
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = minus_infinity<T>();
    T* e = reinterpret_cast<T*>(w);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (first + i < V) e[i] = row[first + i];
    return make_uint4(w[0], w[1], w[2], w[3]);
  };
  // ---- the row comes in: its largest element, and about its smallest finite one
  float most = -INFINITY, fewest = INFINITY;
  const auto take = [&](const uint4& v) {
    float x[N];
    logits_of<T>(v, x);
#pragma unroll
    for (int e = 0; e < N; ++e) most = max_or_nan(most, x[e]);
    fewest = x[0] > -INFINITY ? fminf(fewest, x[0]) : fewest;
  };
  if (RES && VEC) {      // all of a thread's vectors are on their way at once
    for (int it = 0; it < mine; ++it) {
      uint4* to = kept_row + (warp * its + it) * 32 + lane;
      const int from = begin + (it * 32 + lane) * N;
      if (from + N <= V) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(row + from) : "memory");
      else *to = fetch(from);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    for (int it = 0; it < mine; ++it) take(kept_row[(warp * its + it) * 32 + lane]);
  } else {
    int it0 = 0;
    for (; it0 + 4 <= mine; it0 += 4) {
      uint4 v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = fetch(begin + ((it0 + j) * 32 + lane) * N);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (RES) kept_row[(warp * its + it0 + j) * 32 + lane] = v[j];
        take(v[j]);
      }
    }
    for (; it0 < mine; ++it0) {
      const uint4 v = fetch(begin + (it0 * 32 + lane) * N);
      if (RES) kept_row[(warp * its + it0) * 32 + lane] = v;
      take(v);
    }
  }
  bool odd = most != most || !(t >= 0.f) || p != p || least != least || u != u;

  // ---- what all CTAs of the row agree on.  Published words take turns: between two uses of a set lies a barrier of the cluster.
  int turn = 0;
  // The 256 parts of the row are C neighbouring lanes each; a thread learns one of their maxima (as `order`, 0 for none)
  uint32_t best = most > -INFINITY ? order_of(most) : 0;
  for (int o = 1; o < C; o <<= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  if ((tid & (C - 1)) == 0) s.maxima[tid >> lc] = best;
  {
    const uint32_t lo = __reduce_min_sync(0xffffffffu, order_of(fewest)), flag = __any_sync(0xffffffffu, odd);
    if (lane == 0) s.part[warp][0] = lo, s.part[warp][1] = flag;
    __syncthreads();
    if (warp == 0) {
      const uint32_t a = __reduce_min_sync(0xffffffffu, (uint32_t)s.part[lane & 7][0]), b = __any_sync(0xffffffffu, s.part[lane & 7][1] != 0);
      if (lane == 0) s.words[0][0] = a, s.words[0][1] = b;
    }
  }
  cluster_sync();
  const uint32_t part_max = peek(&s.maxima[tid & ((SA_THREADS >> lc) - 1)], tid >> (SA_LOG - lc));
  {
    const u64 own = lane < 2 * C ? peek(&s.words[0][lane & 1], lane >> 1) : (lane & 1 ? 0 : 0xffffffffu);
    const uint32_t hi = __reduce_max_sync(0xffffffffu, part_max), lo = __reduce_min_sync(0xffffffffu, part_max ? part_max : 0xffffffffu);
    if (lane == 0) s.part[warp][2] = hi, s.part[warp][3] = lo;
    if (warp == 0) {
      const uint32_t all = __reduce_min_sync(0xffffffffu, lane & 1 ? 0xffffffffu : (uint32_t)own), any = __reduce_or_sync(0xffffffffu, lane & 1 ? (uint32_t)own : 0);
      if (lane == 0) s.got[0] = all, s.got[1] = any;
    }
    __syncthreads();
  }
  turn = 1;
  uint32_t hi32 = (uint32_t)s.part[lane & 7][2], lo32 = (uint32_t)s.part[lane & 7][3];
  hi32 = __reduce_max_sync(0xffffffffu, hi32), lo32 = __reduce_min_sync(0xffffffffu, lo32);
  const float top = hi32 ? ordered(hi32) : -INFINITY, least_top = ordered(lo32), lowest = ordered((uint32_t)s.got[0]);
  odd = s.got[1] != 0;
  const auto leave = [&](long long token, float logprob) { d.token[r] = token, d.logprob[r] = logprob; };
  if (odd || top == -INFINITY) {
    if (rank == 0 && tid == 0) leave(-1, odd ? NAN : -INFINITY);
    cluster_sync();      // nobody leaves while its words are read
    return;
  }
  const double floor_d = t > 0.f ? (double)top - 31.0 * (double)t : (double)top;      // exp(-31) is below 2^-44
  const Weigh weigh = {s.table, (double)top, t > 0.f ? 369.32993046757463 / (double)t : 0.0, __double2float_ru(fmax(floor_d, -3.4028234663852886e38))};

  const auto each = [&](const auto& fn) {      // over this thread's elements: fn(id, logit), in the order of the ids per warp
    for (int it = 0; it < mine; ++it) {
      float x[N];
      logits_of<T>(RES ? kept_row[(warp * its + it) * 32 + lane] : fetch(begin + (it * 32 + lane) * N), x);
#pragma unroll
      for (int e = 0; e < N; ++e) fn(begin + (it * 32 + lane) * N + e, x[e]);
    }
  };
  // Sums of up to four numbers over the row
  const auto all_of = [&](u64 (&v)[4]) SA_INLINE {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = warp_sum(v[j]);
      if (lane == 0) s.part[warp][j] = v[j];
    }
    __syncthreads();
    if (warp == 0) {
      u64 a = s.part[lane & 7][lane >> 3];
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
      if ((lane & 7) == 0) s.words[turn][lane >> 3] = a;
    }
    cluster_sync();
    if (warp == 0) {
      u64 a = lane < 4 * C ? peek(&s.words[turn][lane & 3], lane >> 2) : 0;
#pragma unroll
      for (int o = 4; o < 4 * SA_CLUSTER; o <<= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
      if (lane < 4) s.got[lane] = a;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = s.got[j];
    turn ^= 1;
  };
  // The first element by id whose running sum of value(id, logit) passes aim(sum of all); what aim() leaves there is what the answer's weight is
  // a share of
  struct Place {
    int id, owner;                     // id; warp of the row
    u64 front, target;                 // sum in front of that warp's run, and what was looked for
  };
  // `leaves`: the answer of the row, written by who finds it; the CTAs end with it
  const auto locate_from = [&](u64 warps_sum, bool leaves, const auto& value, const auto& aim) SA_INLINE -> Place {
    u64* w = s.sums[turn];
    if (lane == 0) w[warp] = warps_sum;
    cluster_sync();
    if (warp == 0) {      // two warps' sums of the row per lane
      u64 v[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int at = lane * 2 + j;
        v[j] = at < C * SA_WARPS ? peek(&w[at % SA_WARPS], at / SA_WARPS) : 0;
      }
      u64 total = __shfl_sync(0xffffffffu, warp_upto(v[0] + v[1]), 31);
      const u64 upto = warp_upto(v[0] + v[1]), most = total, target = aim(total), front = upto - v[0] - v[1];
      const bool here = front <= target && target < upto, second = target >= front + v[0];
      if (here || (lane == 0 && target >= most))
        s.got[2] = lane * 2 + second, s.got[3] = second ? front + v[0] : front, s.got[4] = target, s.got[5] = total;
    }
    if (leaves) leave_arrive();
    else __syncthreads();
    const int owner = (int)s.got[2];
    const u64 target = s.got[4], total = s.got[5];
    if (owner / SA_WARPS == rank) {      // its CTA: the steps of that warp's run, then the lanes of one step
      const int wo = owner % SA_WARPS, first = (rank * SA_WARPS + wo) * its * STEP, n = max(0, min(its, (V - first + STEP - 1) / STEP));
      const auto lane_of = [&](int it, u64 (&y)[N]) {
        float x[N];
        logits_of<T>(RES ? kept_row[(wo * its + it) * 32 + lane] : fetch(first + (it * 32 + lane) * N), x);
        u64 q = 0;
#pragma unroll
        for (int e = 0; e < N; ++e) y[e] = value(first + (it * 32 + lane) * N + e, x[e]), q += y[e];
        return q;
      };
      u64 y[N];
      for (int it = warp; it < n; it += SA_WARPS) {
        const u64 q = warp_sum(lane_of(it, y));
        if (lane == 0) s.steps[it] = q;
      }
      __syncthreads();
      if (warp == 0) {
        int it = 0;
        u64 front = s.got[3];
        for (int i0 = 0; i0 < n; i0 += 32) {
          const u64 q = i0 + lane < n ? s.steps[i0 + lane] : 0, up = warp_upto(q);
          const unsigned hit = __ballot_sync(0xffffffffu, front + up > target);
          if (hit) {
            it = i0 + __ffs(hit) - 1;
            front += __shfl_sync(0xffffffffu, up - q, __ffs(hit) - 1);
            break;
          }
          front += __shfl_sync(0xffffffffu, up, 31);
        }
        const u64 q = lane_of(it, y), up = warp_upto(q);
        u64 at = front + up - q;
        bool done = !(at <= target && target < front + up);
#pragma unroll
        for (int e = 0; e < N; ++e) {
          if (!done && target < at + y[e]) {
            const int id = first + (it * 32 + lane) * N + e;
            if (leaves) d.token[r] = id, d.logprob[r] = (float)log((double)y[e] / (double)total);
            else s.record[turn][0] = (u64)id;
            done = true;
          }
          at += y[e];
        }
      }
    }
    Place got = {0, owner, s.got[3], target};
    if (leaves) {
      leave_wait();
      return got;
    }
    cluster_sync();
    if (tid == 0) s.got[6] = peek(&s.record[turn][0], owner / SA_WARPS);
    __syncthreads();
    got.id = (int)s.got[6];
    turn ^= 1;
    return got;
  };
  const auto sum_of = [&](const auto& value) SA_INLINE {      // of this warp's elements
    decltype(value(0, 0.f)) sum = 0;
    each([&](int i, float x) { sum += value(i, x); });
    return (u64)warp_sum(sum);
  };
  const auto at_random = [&](u64 total) { return u >= 1.f ? total - 1 : min(share_of<false>(total, u), total - 1); };

  const long long k = t == 0.f ? 1 : (k0 <= 0 || k0 > V ? V : k0);
  const u64 low = least >= 1.f ? 1ull << 43 : (u64)ceil(fmax((double)least, 0.0) * 0x1p43);
  if (k == 1 || top == INFINITY) {      // of the largest the first, or the first few: they weigh the same
    const auto largest = [&](int, float x) -> uint32_t { return x == top; };
    locate_from(sum_of(largest), true, largest, [&](u64& total) {
      total = min(total, (u64)k);
      if (p < 1.f) total = max((share_of<true>(total << 43, p) + (1ull << 43) - 1) >> 43, 1ull);
      return at_random(total << 43) >> 43;
    });
    return;
  }

  // ---- lists: `order` and inverted id of elements, the largest first: sorted[] of the CTAs that sort.  Returns how many there are.
  // Elements have been put into list[], n_list of them by this CTA (more than SA_LIST: not all).
  const auto sort_list = [&](bool here, bool seen) SA_INLINE {      // seen: the lists have been published
    if (!seen) cluster_sync();
    if (warp == 0) {
      const uint32_t n = lane < C ? min(peek(&s.n_list, lane), 1u << 21) : 0, upto = warp_upto(n);
      if (lane < SA_CLUSTER) s.part[lane][0] = upto;      // (behind the last CTA: all)
    }
    __syncthreads();
    const int n = (int)s.part[SA_CLUSTER - 1][0];
    if (here && n <= SA_LIST) {
      u64 v = 0;
      if (tid < n) {
        int c = 0, before = 0;
        while (tid >= (int)s.part[c][0]) before = (int)s.part[c++][0];
        v = peek(&s.list[tid - before], c);
        s.value[tid] = v;
      }
      __syncthreads();
      if (tid < n) {
        int above = 0;
        for (int j = 0; j < n; ++j) above += s.value[j] > v;
        s.sorted[above] = v;
      }
      __syncthreads();
    }
    return n;
  };
  const auto to_list = [&](int i, float x) SA_INLINE {
    const uint32_t at = atomicAdd(&s.n_list, 1);
    if (at < SA_LIST) s.list[at] = (u64)order_of(x) << 32 | (uint32_t)~i;
  };
  // Running sum of a number per thread, and the sum of all
  const auto run = [&](u64 v, u64& all) SA_INLINE {
    const u64 up = warp_upto(v);
    if (lane == 31) s.part[warp][1] = up;
    __syncthreads();
    u64 front = up;
    all = 0;
    for (int w = 0; w < SA_WARPS; ++w) {
      const u64 q = s.part[w][1];
      if (w < warp) front += q;
      all += q;
    }
    __syncthreads();
    return front;
  };
  // The choice among the elements of a list, of which a thread has `key` with the weight `stays`
  const auto from_list = [&](int n, u64 key, u64 stays) SA_INLINE {
    u64 sum;
    run(stays, sum);
    const u64 target = at_random(sum);
    s.value[tid] = stays;
    __syncthreads();
    if (stays) {      // the sum in front of it in the order of the ids, which are held inverted
      u64 front = 0;
      for (int j = 0; j < n; ++j)
        if ((uint32_t)s.sorted[j] > (uint32_t)key) front += s.value[j];
      if (front <= target && target < front + stays) leave((long long)(uint32_t)~(uint32_t)key, (float)log((double)stays / (double)sum));
    }
  };
  // Equal steps of the logits from the top down, to the nearest: no less for a smaller logit
  const auto step_of = [&](float x, float scale) {
    const float y = fminf(fmaf(top - x, scale, 12582912.f), 12582912.f + (SA_BINS - 1));      // 1.5 2^23
    return __float_as_int(y) - 0x4b400000;
  };
  const uint32_t hist_s = smem_u32(s.hist);
  const auto count_step = [&](float x, float scale, float from) {      // of x >= from
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ge.f32 p, %1, %2;\n\t@p red.shared.add.u32 [%0], 1;\n\t}" ::"r"(hist_s + (uint32_t)step_of(x, scale) * 4), "f"(x),
                 "f"(from) : "memory");
  };
  const auto scale_of = [&](float lo) {
    const float range = top - lo;
    const float per = (float)(SA_BINS - 1) / range;
    return range > 0.f && per < INFINITY ? per : 0.f;
  };

  // ---- a small k: the elements that reach the k-th largest of the parts' maxima
  if (k <= SA_LIST / 2) {
    const float scale = scale_of(least_top);
    const int bin = part_max ? step_of(ordered(part_max), scale) : SA_BINS;
    if (part_max) atomicAdd(&s.hist[bin], 1);
    __syncthreads();
    u64 all;
    constexpr int OWN = SA_BINS / SA_THREADS;
    uint32_t own = 0, v[OWN];
#pragma unroll
    for (int j = 0; j < OWN; ++j) v[j] = s.hist[tid * OWN + j], own += v[j];
    const u64 upto = run(own, all);
    if (tid == 0) s.got[0] = SA_BINS;
    __syncthreads();
    if (upto - own < (u64)k && (u64)k <= upto) {
      u64 at = upto - own;
#pragma unroll
      for (int j = 0; j < OWN; ++j) {
        if (at < (u64)k && (u64)k <= at + v[j]) s.got[0] = tid * OWN + j;
        at += v[j];
      }
    }
#pragma unroll
    for (int j = 0; j < OWN; ++j) s.hist[tid * OWN + j] = 0;
    __syncthreads();
    const int border = (int)s.got[0];
    const uint32_t low_max = __reduce_min_sync(0xffffffffu, part_max && bin <= border ? part_max : 0xffffffffu);
    if (lane == 0) s.part[warp][2] = low_max;
    __syncthreads();
    const uint32_t reach32 = __reduce_min_sync(0xffffffffu, (uint32_t)s.part[lane & 7][2]);
    const float reach = border == SA_BINS ? -3.402823466e38f : ordered(reach32);      // fewer maxima than k: all finite ones
    each([&](int i, float x) {
      if (x >= reach) to_list(i, x);
    });
    const int n = sort_list(rank == 0, false);
    if (n <= SA_LIST) {
      if (rank == 0) {
        const u64 key = tid < n ? s.sorted[tid] : 0;
        const float x = ordered((uint32_t)(key >> 32));
        const u64 w = tid < n && tid < k && x >= weigh.floor ? weigh(x) : 0;
        u64 total;
        const u64 before = run(w, total) - w;
        from_list(n, key, (tid == 0 || before < (p < 1.f ? share_of<true>(total, p) : ~0ull)) && w >= low ? w : 0);
      }
      cluster_sync();
      return;
    }
    cluster_sync();      // the lists have been looked at
    if (tid == 0) s.n_list = 0;
    __syncthreads();
  }

  // ---- borders: kept is what is larger than `edge`, and equal ones up to id `last`
  float edge = -INFINITY;
  int last = V;
  const auto kept = [&](int i, float x) { return x > edge || (x == edge && i <= last); };
  const auto clear_hist = [&]() SA_INLINE {
    for (int i = tid; i < SA_BINS; i += SA_THREADS) s.hist[i] = 0;
    __syncthreads();
  };
  // Two steps of a histogram of the row at which the running sum of value(step) per element reaches aim(sum of all, of squares, ..), in
  // fp32 (exact for counts) and a fixed order; each CTA adds up its part of the steps.  got[]: the steps in the upper halves, in the lower
  // how many elements are in front of the first and up to the second; ~0 where it is not reached.  Clears the histogram.
  const auto find = [&](const auto& value, const auto& aim) SA_INLINE {
    constexpr int MOST = SA_BINS / SA_THREADS;
    const int per = max(MOST >> lc, 1), b0 = (rank << SA_LOG) * per + tid * per;      // (eight CTAs have a step per thread)
    static_assert(SA_BINS == SA_THREADS * SA_CLUSTER, "a step per thread at least");
    cluster_sync();
    float v[MOST], own = 0.f, square = 0.f;      // square: of what one element of a step counts, over all
    uint32_t m[MOST], own_m = 0;
#pragma unroll
    for (int j = 0; j < MOST; ++j) {
      v[j] = 0.f, m[j] = 0;
      if (j < per) {
        uint32_t n = 0;
#pragma unroll
        for (int c = 0; c < SA_CLUSTER; ++c) n += c < C ? peek(&s.hist[b0 + j], c) : 0;
        const float one = n ? value(b0 + j) : 0.f;
        v[j] = (float)n * one, square += v[j] * one;
        own += v[j];
        m[j] = n, own_m += n;
      }
    }
    const float up = warp_upto(own);
    const uint32_t up_m = warp_upto(own_m);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) square += __shfl_xor_sync(0xffffffffu, square, o);
    float* part = reinterpret_cast<float*>(s.part);
    uint32_t* part_m = reinterpret_cast<uint32_t*>(part) + 2 * SA_WARPS;
    if (lane == 31) part[warp] = up, part[SA_WARPS + warp] = square, part_m[warp] = up_m;
    if (tid < 2) s.record[turn][tid] = ~0ull;
    __syncthreads();
    float front = up - own;
    uint32_t front_m = up_m - own_m;
#pragma unroll
    for (int w = 0; w < SA_WARPS; ++w) front += w < warp ? part[w] : 0.f, front_m += w < warp ? part_m[w] : 0;
    if (tid == 0) {
      float all = 0.f, squares = 0.f;
#pragma unroll
      for (int w = 0; w < SA_WARPS; ++w) all += part[w], squares += part[SA_WARPS + w];
      uint32_t all_m = 0;
#pragma unroll
      for (int w = 0; w < SA_WARPS; ++w) all_m += part_m[w];
      s.words[turn][0] = (u64)__float_as_uint(squares) << 32 | __float_as_uint(all), s.words[turn][1] = all_m;
    }
    cluster_sync();
    if (warp == 0) {
      const u64 q = lane < C ? peek(&s.words[turn][0], lane) : 0;
      const float upto = warp_upto(__uint_as_float((uint32_t)q)), squares = warp_upto(__uint_as_float((uint32_t)(q >> 32)));
      if (lane == 31) s.got[0] = __float_as_uint(upto), s.got[1] = __float_as_uint(squares);
      const uint32_t q_m = lane < C ? (uint32_t)peek(&s.words[turn][1], lane) : 0, upto_m = warp_upto(q_m);
      if (lane == rank) s.got[2] = (u64)(upto_m - q_m) << 32 | __float_as_uint(upto - __uint_as_float((uint32_t)q));
    }
    clear_hist();
    const float all = __uint_as_float((uint32_t)s.got[0]), squares = __uint_as_float((uint32_t)s.got[1]);
    front += __uint_as_float((uint32_t)s.got[2]), front_m += (uint32_t)(s.got[2] >> 32);
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      const float want = aim(all, squares, a);
      float at = front;
      uint32_t at_m = front_m;
#pragma unroll
      for (int j = 0; j < MOST; ++j) {
        if (v[j] > 0.f && at + v[j] >= want) {
          atomicMin(&s.record[turn][a], (u64)(b0 + j) << 32 | (at_m + (a ? m[j] : 0)));
          break;
        }
        at += v[j], at_m += m[j];
      }
    }
    cluster_sync();
    if (warp == 0) {
      u64 q = lane < 2 * C ? peek(&s.record[turn][lane & 1], lane >> 1) : ~0ull;
#pragma unroll
      for (int o = 2; o < 2 * SA_CLUSTER; o <<= 1) q = min(q, __shfl_xor_sync(0xffffffffu, q, o));
      if (lane < 2) s.got[lane] = q;
    }
    __syncthreads();
    turn ^= 1;
  };
  // The smallest logit (as `order`) of step `b` or one further up, found by all lanes of a warp
  const auto first_of = [&](int b, float scale) SA_INLINE {
    uint32_t lo = 0x00800000u, hi = order_of(top);      // the lowest finite number; step_of(top) = 0
    {      // about there
      const uint32_t at = order_of(fmaxf(top - ((float)b + 0.5f) / scale, -3.4e38f)) - 16 + lane;
      const unsigned yes = __ballot_sync(0xffffffffu, lo <= at && at <= hi && step_of(ordered(at), scale) <= b), in = __ballot_sync(0xffffffffu, lo <= at && at <= hi);
      if (in == 0xffffffffu && yes && !(yes & 1u)) return __shfl_sync(0xffffffffu, at, __ffs(yes) - 1);
    }
    while (lo < hi) {      // 31 points between them
      const u64 span = (u64)hi - lo;
      const uint32_t at = lo + (uint32_t)(span * (u64)lane >> 5);
      const unsigned yes = __ballot_sync(0xffffffffu, step_of(ordered(at), scale) <= b);
      const int f = yes ? __ffs(yes) - 1 : 32;
      const uint32_t new_hi = f < 32 ? lo + (uint32_t)(span * (u64)f >> 5) : hi;
      const uint32_t new_lo = f > 0 ? lo + (uint32_t)(span * (u64)(f - 1) >> 5) + 1 : lo;
      lo = min(new_lo, new_hi), hi = new_hi;
    }
    return lo;
  };
  // The logits of steps b1 to b2: got[0] the smallest, got[1] the largest (as `order`)
  const auto between = [&](int b1, int b2, float scale) SA_INLINE {
    if (warp < 2) {
      const int b = warp == 0 ? b2 : b1 - 1;
      const uint32_t o = b >= SA_BINS - 1 ? 0x00800000u : b < 0 ? order_of(top) + 1 : first_of(b, scale);
      if (lane == 0) s.got[warp] = warp == 0 ? o : o - 1;
    }
    __syncthreads();
  };
  const auto set_aside = [&](int i, float x) SA_INLINE {
    const uint32_t at = atomicAdd(&s.n_aside, 1);
    if (at < SA_ASIDE) s.aside[at] = (u64)order_of(x) << 32 | (uint32_t)~i;
  };
  constexpr int GRAIN = sizeof(T) == 4 ? 0 : (std::is_same<T, __half>::value ? 13 : 16);      // two logits are 2^GRAIN apart, at least
  const auto logit_below = [&](uint32_t o) {      // the largest logit up to `o`
    const uint32_t c = o & ~((1u << GRAIN) - 1);
    return c >= 0x80000000u ? c : ((o + 1) & ~((1u << GRAIN) - 1)) - 1;
  };
  // The border among the kept elements of one value, of which this warp has `many`: it has as many of them as are needed, by their ids.
  // Sets how many of the warp's own that are.  False where there are not so many.
  const auto among_equal = [&](uint32_t o, u64 one, u64 many, u64 need, u64& stay) SA_INLINE {
    const float value = ordered(o);
    const int until = value == edge ? last : V;
    const u64 take = (need + one - 1) / max(one, 1ull);
    __syncthreads();
    if (tid == 0) s.got[0] = 0;
    const Place at = locate_from(many, false, [&](int i, float x) -> uint32_t { return x == value && i <= until; }, [&](u64 total) {
      if (take > total) s.got[0] = 1;
      return min(take, total) - 1;
    });
    if (s.got[0]) return false;
    const int own = rank * SA_WARPS + warp;
    stay = own < at.owner ? many : own == at.owner ? at.target - at.front + 1 : 0;
    edge = value, last = at.id;
    return true;
  };
  // The border among n kept elements of logits lo .. hi (as `order`) is where the running count or sum of weights reaches `need`.  They have
  // been set aside, or where there was no room all look at the whole row for them.  False where they do not reach it.
  const auto inside = [&](uint32_t lo, uint32_t hi, u64 n, bool over, bool mass, u64 need) SA_INLINE {
    const float lo0 = ordered(lo), hi0 = ordered(hi);
    const int own = min((int)s.n_aside, SA_ASIDE);
    const auto members = [&](const auto& fn) {      // fn(order, inverted id)
      if (!over) {
        for (int j = tid; j < own; j += SA_THREADS) {
          const u64 v = s.aside[j];
          if (lo <= (uint32_t)(v >> 32) && (uint32_t)(v >> 32) <= hi) fn((uint32_t)(v >> 32), (uint32_t)v);
        }
      } else {
        each([&](int i, float x) {
          if (lo0 <= x && x <= hi0 && kept(i, x) && lo <= order_of(x) && order_of(x) <= hi) fn(order_of(x), (uint32_t)~i);
        });
      }
    };
    const auto weight_of = [&](uint32_t o) -> u64 { return mass ? (ordered(o) >= weigh.floor ? weigh(ordered(o)) : 0) : 1; };
    uint32_t* const mass32 = reinterpret_cast<uint32_t*>(s.mass);      // the low halves of all steps, then the high ones
    while (lo < hi && n > SA_LIST) {      // steps of the order itself
      int shift = GRAIN;
      while ((hi - lo) >> shift >= SA_FINE) ++shift;
      const bool one_value = shift == GRAIN;      // in each step: its sum of weights is a product
      const auto value_of = [&](int b) { return logit_below(hi - ((uint32_t)b << shift)); };
      for (int i = tid; i < SA_FINE; i += SA_THREADS) s.hist[i] = 0, s.mass[i] = 0;
      __syncthreads();
      members([&](uint32_t o, uint32_t) {
        const uint32_t b = (hi - o) >> shift;
        atomicAdd(&s.hist[b], 1);
        if (mass && !one_value) {      // (64 bits by two counters of 32)
          const u64 w = weight_of(o);
          const uint32_t was = atomicAdd(&mass32[b], (uint32_t)w);
          atomicAdd(&mass32[SA_FINE + b], (uint32_t)(w >> 32) + (was + (uint32_t)w < was));
        }
      });
      cluster_sync();
      // two steps per thread, all of them in each CTA
      u64 v[2];
      uint32_t m[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        v[j] = m[j] = 0;
#pragma unroll
        for (int c = 0; c < SA_CLUSTER; ++c) m[j] += c < C ? peek(&s.hist[tid * 2 + j], c) : 0;
        if (mass && !one_value) {
#pragma unroll
          for (int c = 0; c < SA_CLUSTER; ++c)
            if (c < C) v[j] += (u64)peek(&mass32[SA_FINE + tid * 2 + j], c) << 32 | peek(&mass32[tid * 2 + j], c);
        } else {
          v[j] = m[j] ? m[j] * weight_of(value_of(tid * 2 + j)) : 0;
        }
      }
      u64 sum;
      const u64 upto = run(v[0] + v[1], sum), front = upto - v[0] - v[1];
      if (front < need && need <= upto) {
        const int j = need > front + v[0] && v[1] ? 1 : 0;
        s.got[0] = tid * 2 + j, s.got[1] = j ? front + v[0] : front, s.got[2] = m[j];
      }
      cluster_sync();
      if (need > sum) {
        for (int i = tid; i < SA_FINE; i += SA_THREADS) s.hist[i] = 0;
        __syncthreads();
        return false;
      }
      const int bin = (int)s.got[0];
      need -= s.got[1], n = s.got[2];
      if (one_value) {
        lo = hi = value_of(bin);
      } else {
        const uint32_t start = hi - ((uint32_t)bin << shift);
        lo = max(lo, start - ((1u << shift) - 1)), hi = start;
      }
    }
    for (int i = tid; i < SA_FINE; i += SA_THREADS) s.hist[i] = 0;
    if (lo < hi) {
      members([&](uint32_t o, uint32_t inverted) { to_list((int)~inverted, ordered(o)); });
      const int m = sort_list(true, false);
      const u64 key = tid < m ? s.sorted[tid] : 0, w = tid < m ? weight_of((uint32_t)(key >> 32)) : 0;
      u64 sum;
      const u64 upto = run(w, sum);
      if (upto - w < need && need <= upto) s.got[0] = key;
      cluster_sync();      // the lists have been read
      if (need > sum) {
        if (tid == 0) s.n_list = 0;
        __syncthreads();
        return false;
      }
      edge = ordered((uint32_t)(s.got[0] >> 32)), last = (int)(uint32_t)~(uint32_t)s.got[0];
      if (tid == 0) s.n_list = 0;
    } else {
      const float value = ordered(lo);
      const int until = value == edge ? last : V;
      u64 stay;
      return among_equal(lo, weight_of(lo), sum_of([&](int i, float x) -> uint32_t { return x == value && i <= until; }), need, stay);
    }
    return true;
  };
  // The kept elements of logits lo .. hi are set aside; of 16-bit logits there are few values in between, of many elements each
  constexpr bool ASIDE = sizeof(T) == 4;
  const auto put_aside = [&](float lo_x, float hi_x) SA_INLINE {
    each([&](int i, float x) {
      if (lo_x <= x && x <= hi_x && kept(i, x)) set_aside(i, x);
    });
    __syncthreads();
  };
  if (k < V) {
    const float scale = scale_of(fmaxf(lowest, top - 48.f));
    each([&](int, float x) {
      count_step(x, scale, -3.402823466e38f);
    });
    find([](int) { return 1.f; }, [&](float, float, int) { return (float)k; });
    const u64 got = s.got[0];
    __syncthreads();
    if (got != ~0ull) {      // else there are not so many
      between((int)(got >> 32), (int)(got >> 32), scale);
      const uint32_t lo = (uint32_t)s.got[0], hi = (uint32_t)s.got[1];
      u64 v[4] = {0, 0, 0, 0};
      if (ASIDE) put_aside(ordered(lo), ordered(hi));
      v[0] = tid == 0 ? s.n_aside : 0, v[1] = tid == 0 && s.n_aside > SA_ASIDE;
      all_of(v);
      __syncthreads();
      inside(lo, hi, ASIDE ? v[0] : SA_LIST + 1, !ASIDE || v[1], false, (u64)k - (uint32_t)got);
      if (tid == 0) s.n_aside = 0;
      __syncthreads();
    }
  }
  // What counts of each element: from what on it weighs anything, and whether it is kept
  const auto final = [&](int i, float x) -> u64 {
    u64 w = weigh(x);
    w = x >= weigh.floor && x >= edge ? w : 0;
    if (last < V) w = x == edge && i > last ? 0 : w;
    if (low) w = w >= low ? w : 0;
    return w;
  };
  if (p < 1.f) {
    const float from = fmaxf(weigh.floor, edge), scale = scale_of(fmaxf(lowest, from));
    const bool ties = edge >= from;
    each([&](int, float x) { count_step(x, scale, from); });
    // A step's elements by the weight of its middle: each is off by up to half a step's factor, 1/sqrt(12) of a step on average and either
    // way, so that the border is between the two steps where their sums pass p of it all less and more four times that in the square mean
    const float per_bin = scale > 0.f ? 1.f / (scale * t) : 0.f;
    find([&](int b) { return exp2f(-1.4426950f * (float)b * per_bin); }, [&](float all, float squares, int a) {
      const float off = 1.2f * fminf(per_bin, 1.f) * sqrtf(squares) + 1e-5f * all;
      return p * all + (a ? off : -off);
    });
    const bool listed = s.got[1] != ~0ull && (uint32_t)s.got[1] <= SA_LIST;      // all down to the second step fit a list
    const int b1 = s.got[0] == ~0ull ? 0 : (int)(s.got[0] >> 32), b2 = s.got[1] == ~0ull ? SA_BINS - 1 : (int)(s.got[1] >> 32);
    __syncthreads();
    between(b1, b2, scale);
    uint32_t lo = (uint32_t)s.got[0], hi = (uint32_t)s.got[1];
    const float lo_x = fmaxf(ordered(lo), from), hi_x = ordered(hi);
    // up to four values between: their elements are only counted
    float value[4];
    int values = 0;
    {
      uint32_t o = logit_below(hi);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        value[j] = ordered(o);
        if (o >= lo && value[j] >= from && values == j) ++values;
        o = logit_below(o - 1);
      }
      if (o >= lo && ordered(o) >= from) values = 0;
    }
    u64 all = 0, above = 0;
    if (listed) {
      each([&](int i, float x) {
        const u64 w = weigh(x);
        if (x >= from) all += w;
        if (x >= lo_x && kept(i, x)) to_list(i, x);
      });
    } else {
      each([&](int, float x) {
        const u64 w = weigh(x);
        if (x >= from) all += w;
        if (x > hi_x) above += w;
      });
    }
    if (ties) {      // equal ones that top-k has not kept
      uint32_t out = 0;
      each([&](int i, float x) { out += x == edge && i > last; });
      all -= out * weigh(edge);
    }
    u64 limit, kept_sum = 0;             // kept_sum: of this warp
    bool guessed = false, over = false;
    int own = 0;
    if (listed) {
      u64 v[4] = {all, 0, 0, 0}, sum;
      all_of(v);
      limit = max(share_of<true>(v[0], p), 1ull);
      const int n = sort_list(true, true);
      if (n <= SA_LIST) {
        const u64 key = tid < n ? s.sorted[tid] : 0;
        const u64 w = tid < n ? weigh(ordered((uint32_t)(key >> 32))) : 0, upto = run(w, sum);
        if (sum >= limit) {
          if (rank == 0) from_list(n, key, upto - w < limit && w >= low ? w : 0);
          cluster_sync();      // nobody leaves while its words are read
          return;
        }
      }
      cluster_sync();      // the border is further down
      if (tid == 0) s.n_list = 0;
      __syncthreads();
    } else {
      u64 v[4] = {all, above, 0, 0};
      uint32_t many[4] = {0, 0, 0, 0};
      if (values) {
        if (values <= 2) {
          each([&](int, float x) { many[0] += x == value[0], many[1] += x == value[1]; });
        } else {
          each([&](int, float x) {
#pragma unroll
            for (int j = 0; j < 4; ++j) many[j] += x == value[j];
          });
        }
        if (ties) {
          each([&](int i, float x) {
#pragma unroll
            for (int j = 0; j < 4; ++j) many[j] -= x == value[j] && x == edge && i > last;
          });
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (j >= values) many[j] = 0;
          many[j] = __reduce_add_sync(0xffffffffu, many[j]);      // of the warp
        }
        v[2] = lane == 0 ? (u64)many[0] << 32 | many[1] : 0, v[3] = lane == 0 ? (u64)many[2] << 32 | many[3] : 0;
      } else if (ASIDE) {
        put_aside(lo_x, hi_x);
        v[2] = tid == 0 ? s.n_aside : 0, v[3] = tid == 0 && s.n_aside > SA_ASIDE;
      }
      own = min((int)s.n_aside, SA_ASIDE);
      kept_sum = warp_sum(above);
      all_of(v);
      __syncthreads();
      limit = max(share_of<true>(v[0], p), 1ull);
      over = !ASIDE || v[3];
      guessed = v[1] < limit;
      if (guessed && values) {
        u64 need = limit - v[1];
        bool found = false;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const u64 n = j & 1 ? (uint32_t)v[2 + (j >> 1)] : v[2 + (j >> 1)] >> 32, one = j < values ? weigh(value[j]) : 0;
          if (found || j >= values) continue;
          if (n * one >= need) {
            u64 stay;
            found = among_equal(order_of(value[j]), one, many[j], need, stay);
            kept_sum += stay * one;
          } else {
            need -= n * one, kept_sum += many[j] * one;
          }
        }
        guessed = found;
      } else if (guessed) {
        guessed = inside(max(lo, order_of(from)), hi, over ? SA_LIST + 1 : v[2], over, true, limit - v[1]);
      }
    }
    if (!guessed) inside(order_of(from), order_of(top), V, true, true, limit);      // not between those two: among all
    if (low == 0 && guessed) {      // the warps' sums: what was above, and the kept ones between the two
      if (lane == 0) s.sums[turn][warp] = kept_sum;
      __syncthreads();
      if (values) {
      } else if (!over) {
        for (int j = tid; j < own; j += SA_THREADS) {
          const u64 e = s.aside[j];
          const int i = (int)(uint32_t)~(uint32_t)e;
          const float x = ordered((uint32_t)(e >> 32));
          if (kept(i, x)) atomicAdd(&s.sums[turn][i / (its * STEP) % SA_WARPS], weigh(x));
        }
      } else {
        u64 rest = 0;
        each([&](int i, float x) {
          if (lo_x <= x && x <= hi_x && kept(i, x)) rest += weigh(x);
        });
        rest = warp_sum(rest);
        if (lane == 0) s.sums[turn][warp] += rest;
      }
      __syncthreads();
      const u64 sum = s.sums[turn][warp];
      __syncthreads();
      locate_from(sum, true, final, at_random);
      return;
    }
  }
  locate_from(sum_of(final), true, final, at_random);
}

template <typename T, bool RES, bool VEC>
static int launch(const FtkSampleDesc& d, int its, cudaStream_t s) {
  const auto kernel = sample_kernel<T, RES, VEC>;
  const size_t bytes = SA_OWN + (RES ? (size_t)its * SA_THREADS * 16 : 0);
  if (RES) {      // the most for any row: the limit is the function's, and calls of other sizes may be on their way to their launch
    const int rc = (int)cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SA_OWN + SA_SHARE);
    if (rc) return rc;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(d.R << d.cluster));
  cfg.blockDim = dim3(SA_THREADS);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = 1u << d.cluster, at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  return (int)cudaLaunchKernelEx(&cfg, kernel, d, its);
}

template <typename T> static int launch(FtkSampleDesc d, cudaStream_t s) {
  constexpr int STEP = SA_THREADS * 16 / (int)sizeof(T);      // columns of a step of a CTA
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const auto its_of = [&](int c) { return (int)((d.V + (long long)STEP * c - 1) / ((long long)STEP * c)); };
  // As many CTAs for a row as fill the SMs four times, with two steps each at least, and as many as it takes for three to share an SM, so
  // that one works while others wait.  With 13 steps, the most for that: 256 rows of 50257 fp32, settings by row, 65.8 us, and 74.7 in clusters twice
  // as large.  With 14, in clusters twice as large as against two CTAs to an SM: 256 rows of 55000 with settings by row 77.7 and 81.3, k = 50
  // 43.5 and 46.6, the whole distribution 51.9 and 54.3, p = 0.9 116.1 and 110.9; 640 of 14000, p = 0.9, 68.2 and 74.8; 512 of 110000 in bf16 the same
  int c = 1;
  while (c < SA_CLUSTER && its_of(c) > 1 && ((d.R * c < 4ll * sms && its_of(c) > 2) || its_of(c) > SA_THREE)) c *= 2;
  int lc = 0;
  while ((1 << lc) < c) ++lc;
  d.cluster = lc;
  const int its = its_of(c);
  if (its > SA_STEPS || d.R * c > 0x7fffffff) return -2;
  const bool res = its * SA_THREADS * 16 <= SA_SHARE;
  const bool vec = ((uintptr_t)d.logits | (uintptr_t)(d.R > 1 ? d.ld * sizeof(T) : 0)) % 16 == 0;
  if (res) return vec ? launch<T, true, true>(d, its, s) : launch<T, true, false>(d, its, s);
  return vec ? launch<T, false, true>(d, its, s) : launch<T, false, false>(d, its, s);
}

}  // namespace ftk
using namespace ftk;

extern "C" int ftk_sample(const FtkSampleDesc* d, void* stream) {
  if (!d || !d->logits || !d->uniform || !d->token || !d->logprob || d->R <= 0 || d->R > 0x7fffffff || d->V <= 0 || d->V > (1 << 20)) return -2;
  cudaStream_t s = (cudaStream_t)stream;
  if (d->type == FTK_T_FP32) return launch<float>(*d, s);
  if (d->type == FTK_T_BF16) return launch<__nv_bfloat16>(*d, s);
  if (d->type == FTK_T_FP16) return launch<__half>(*d, s);
  return -2;
}
