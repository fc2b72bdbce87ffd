// The choice of a token from the logits of a step: temperature, top-k, top-p, min-p, and a given random number.
//
// Mathematics.  Weights are whole numbers, w_i = 2^43 exp((x_i - max x) / T) to a unit, so their sums (63 bits for up to 2^20 tokens) are
// exact whatever their order, and a row's choice is a function of its logits, settings and random number alone.  With tokens in the
// order of their logits (equal ones by their ids): the first k; of those the ones before which less than p of the sum lies; of those the
// ones of at least min_p of the largest; then the first by id whose running sum passes u times the sum.
//
// What bounds it: each logit is read once.  Weights take 9 operations in 64 bits, half the rate of fp32.
//
// Work.  A cluster of CTAs has a row, each an equal run of its columns, which it keeps in shared memory (rows of more than that are read
// again from L2): everything behind the first pass works there.  Sums, histograms and lists of the CTAs are read by all of them over
// distributed shared memory, and all come to the same conclusions.
//   * The k largest of a small k are among the elements that reach the k-th largest of the threads' own maxima: hardly more than k.
//     They become a list, ordered by counting, and the rest is done on it.
//   * Else the border of top-k and of top-p is found by counts of 2048 equal steps of the logits' range: the step with the border is
//     looked into, with the sums of weights in it and above it, until it is one value or a short list.  Its equal elements are taken by id.
//   * The choice: sums per warp in the order of the ids, the warp with the target, the 32 vectors, the lane.
#include <math.h>

#include "ft_sm100.cuh"
#include "half_types.cuh"
#include "launch.cuh"
#include "ftk_api.h"

namespace ftk {

typedef unsigned long long u64;
constexpr int SA_THREADS = 512, SA_WARPS = SA_THREADS / 32;
constexpr int SA_BINS = 2048;          // steps of a histogram
constexpr int SA_LIST = 512;           // elements of a list
constexpr int SA_CLUSTER = 8;          // CTAs of a row at most
constexpr int SA_STEPS = 512;          // vectors of a lane at most
constexpr int SA_SHARE = 72 * 1024;    // bytes of a row that a CTA keeps at most: two CTAs share an SM

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
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
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

struct SampleShared {
  u64 sums[2][SA_WARPS + 8];           // per warp, published; then the CTA's
  u64 steps[SA_STEPS];
  double table[256];                   // 2^(i / 256)
  u64 list[SA_LIST], all[SA_LIST], sorted[SA_LIST], weights[SA_LIST];
  uint32_t hist[SA_BINS], total[SA_BINS];
  u64 found[4], mass[SA_WARPS];
  uint32_t words[2][4];                // published: minima and maxima of the CTA
  uint32_t part[SA_WARPS];
  uint32_t count[2];                   // of the list
};

// A row's settings.  2^43 exp((x - top) / T): 2^(k / 256) out of the table, the rest by three terms of the exponential series (relative
// error 2^-46), and by adding 2^9 a number of up to 1 is rounded to units of 2^-43.
struct Weigh {
  const double* table;
  double top, by;                      // 256 log2(e) / T
  float floor;                         // what is below weighs less than half a unit
  __device__ __forceinline__ u64 operator()(float x) const {
    constexpr double MAGIC = 6755399441055744.0;      // 1.5 2^52
    const double d = (double)x - top, kd = fma(d, by, MAGIC), r = fma(d, by, MAGIC - kd);
    const int k = __double2loint(kd);
    constexpr double C = 0.0027076061740622863;       // ln(2) / 256
    const double p = r * fma(r, fma(r, C * C * C / 6, C * C / 2), C), t = table[k & 255];
    double v = fma(t, p, t);
    v = __hiloint2double(__double2hiint(v) + (k >> 8) * (1 << 20), __double2loint(v));
    const u64 w = (u64)__double_as_longlong(v + 512.0) - 0x4080000000000000ull;
    return x >= floor ? w : 0;
  }
};

template <typename T, bool RES, bool VEC>
__global__ void __launch_bounds__(SA_THREADS, 2) sample_kernel(const __grid_constant__ FtkSampleDesc d, const int its) {
  constexpr int N = 16 / (int)sizeof(T), STEP = 32 * N;      // elements of a vector, of a warp's step
  extern __shared__ __align__(16) unsigned char smem[];
  SampleShared& s = *reinterpret_cast<SampleShared*>(smem);
  uint4* kept_row = reinterpret_cast<uint4*>(smem + (sizeof(SampleShared) + 15) / 16 * 16);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, V = (int)d.V;
  const int rank = (int)cluster_rank(), C = (int)d.cluster;
  const long long r = blockIdx.x / C;
  const int begin = (rank * SA_WARPS + warp) * its * STEP;      // this warp's run of columns
  const int mine = max(0, min(its, (V - begin + STEP - 1) / STEP));
  if (tid < 256) s.table[tid] = exp2(tid * (1.0 / 256));
  for (int i = tid; i < SA_BINS; i += SA_THREADS) s.hist[i] = 0;
  if (tid < 2) s.count[tid] = 0;
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
  // ---- the row comes in: largest and smallest finite elements
  float most = -INFINITY, fewest = INFINITY;
  bool odd = !(t >= 0.f) || p != p || least != least || u != u;
  const auto take = [&](const uint4& v, int it) {
    if (RES) kept_row[(warp * its + it) * 32 + lane] = v;
    float x[N];
    logits_of<T>(v, x);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      odd |= x[e] != x[e];
      most = fmaxf(most, x[e]);
      if (x[e] > -INFINITY) fewest = fminf(fewest, x[e]);
    }
  };
  int it0 = 0;
  for (; it0 + 4 <= mine; it0 += 4) {
    uint4 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = fetch(begin + ((it0 + j) * 32 + lane) * N);
#pragma unroll
    for (int j = 0; j < 4; ++j) take(v[j], it0 + j);
  }
  for (; it0 < mine; ++it0) take(fetch(begin + (it0 * 32 + lane) * N), it0);

  // ---- what all CTAs of the row agree on.  Two sets of published words take turns: between two uses of one lies a barrier of the cluster.
  int turn = 0;
  const auto extremes = [&](uint32_t lo, uint32_t hi, uint32_t lo2, uint32_t flag, uint32_t (&out)[4]) {      // smallest, largest, smallest, any
    lo = __reduce_min_sync(0xffffffffu, lo), hi = __reduce_max_sync(0xffffffffu, hi), lo2 = __reduce_min_sync(0xffffffffu, lo2);
    flag = __reduce_or_sync(0xffffffffu, flag);
    uint32_t* w = s.words[turn];
    if (tid == 0) w[0] = 0xffffffffu, w[1] = 0, w[2] = 0xffffffffu, w[3] = 0;
    __syncthreads();
    if (lane == 0) atomicMin(&w[0], lo), atomicMax(&w[1], hi), atomicMin(&w[2], lo2), atomicOr(&w[3], flag);
    __syncthreads();
    cluster_sync();
    out[0] = 0xffffffffu, out[1] = 0, out[2] = 0xffffffffu, out[3] = 0;
    for (int c = 0; c < C; ++c)
      out[0] = min(out[0], peek(&w[0], c)), out[1] = max(out[1], peek(&w[1], c)), out[2] = min(out[2], peek(&w[2], c)), out[3] |= peek(&w[3], c);
    turn ^= 1;
  };
  uint32_t e4[4];
  extremes(order_of(fewest), order_of(most), most > -INFINITY ? order_of(most) : 0xffffffffu, odd, e4);
  const float top = ordered(e4[1]), lowest = ordered(e4[0]), least_top = ordered(e4[2]);      // least_top: the smallest of the threads' maxima
  odd = e4[3] != 0;
  const auto leave = [&](long long token, float logprob) { d.token[r] = token, d.logprob[r] = logprob; };
  if (odd || top == -INFINITY) {
    if (rank == 0 && tid == 0) leave(-1, odd ? NAN : -INFINITY);
    cluster_sync();      // nobody leaves while its words are read
    return;
  }
  const double floor_d = t > 0.f ? (double)top - 31.0 * (double)t : (double)top;      // exp(-31) is below 2^-44
  const Weigh weigh = {s.table, (double)top, t > 0.f ? 369.32993046757463 / (double)t : 0.0,
                       top == INFINITY ? INFINITY : __double2float_ru(fmax(floor_d, -3.4028234663852886e38))};
  const auto weight = [&](float x) -> u64 { return x == top ? 1ull << 43 : weigh(x); };

  const auto each = [&](const auto& fn) {      // over this thread's elements: fn(id, logit), in the order of the ids per warp
    for (int it = 0; it < mine; ++it) {
      float x[N];
      logits_of<T>(RES ? kept_row[(warp * its + it) * 32 + lane] : fetch(begin + (it * 32 + lane) * N), x);
#pragma unroll
      for (int e = 0; e < N; ++e) fn(begin + (it * 32 + lane) * N + e, x[e]);
    }
  };
  const auto sums = [&](u64 a, u64 b, u64 c, u64 (&out)[3]) {      // of the whole row
    a = warp_sum(a), b = warp_sum(b), c = warp_sum(c);
    u64* w = s.sums[turn] + SA_WARPS;
    if (tid < 3) w[tid] = 0;
    __syncthreads();
    if (lane == 0) atomicAdd(&w[0], a), atomicAdd(&w[1], b), atomicAdd(&w[2], c);
    __syncthreads();
    cluster_sync();
    out[0] = out[1] = out[2] = 0;
    for (int q = 0; q < C; ++q) out[0] += peek(&w[0], q), out[1] += peek(&w[1], q), out[2] += peek(&w[2], q);
    turn ^= 1;
  };
  // The first element by id whose running sum of value(id, logit) passes aim(sum of all)
  struct Place {
    int id;
    u64 value, total;
  };
  const auto locate = [&](const auto& value, const auto& aim) -> Place {
    u64 sum = 0;
    each([&](int i, float x) { sum += value(i, x); });
    sum = warp_sum(sum);
    u64* w = s.sums[turn];
    if (lane == 0) w[warp] = sum;
    cluster_sync();
    // every warp for itself: four warps' sums of the row per lane
    u64 v[4], four = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int at = lane * 4 + j;
      v[j] = at < C * SA_WARPS ? peek(&w[at % SA_WARPS], at / SA_WARPS) : 0;
      four += v[j];
    }
    const u64 upto = warp_upto(four), total = __shfl_sync(0xffffffffu, upto, 31), target = aim(total);
    u64 front = upto - four;
    int owner = 0;
    const bool here = front <= target && target < upto;
#pragma unroll
    for (int j = 0; j < 3; ++j)
      if (owner == j && target >= front + v[j]) front += v[j], ++owner;
    const int who = __ffs(__ballot_sync(0xffffffffu, here)) - 1;
    owner = __shfl_sync(0xffffffffu, lane * 4 + owner, max(who, 0));
    front = __shfl_sync(0xffffffffu, front, max(who, 0));
    if (owner / SA_WARPS == rank) {      // its CTA: the steps of that warp's run, then the lanes of one step
      const int wo = owner % SA_WARPS, first = (rank * SA_WARPS + wo) * its * STEP, n = max(0, min(its, (V - first + STEP - 1) / STEP));
      const auto lane_of = [&](int it, float (&x)[N], u64 (&y)[N]) {
        logits_of<T>(RES ? kept_row[(wo * its + it) * 32 + lane] : fetch(first + (it * 32 + lane) * N), x);
        u64 q = 0;
#pragma unroll
        for (int e = 0; e < N; ++e) y[e] = value(first + (it * 32 + lane) * N + e, x[e]), q += y[e];
        return q;
      };
      float x[N];
      u64 y[N];
      for (int it = warp; it < n; it += SA_WARPS) {
        const u64 q = warp_sum(lane_of(it, x, y));
        if (lane == 0) s.steps[it] = q;
      }
      __syncthreads();
      if (warp == 0) {
        int it = 0;
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
        const u64 q = lane_of(it, x, y), up = warp_upto(q);
        u64 at = front + up - q;
        bool done = !(at <= target && target < front + up);
#pragma unroll
        for (int e = 0; e < N; ++e) {
          if (!done && target < at + y[e]) {
            s.found[0] = (u64)(first + (it * 32 + lane) * N + e), s.found[1] = y[e];
            done = true;
          }
          at += y[e];
        }
      }
    }
    cluster_sync();
    const Place got = {(int)peek(&s.found[0], owner / SA_WARPS), peek(&s.found[1], owner / SA_WARPS), total};
    turn ^= 1;
    return got;
  };
  const auto finish = [&](const Place& x) {
    if (rank == 0 && tid == 0) leave(x.id, (float)log((double)x.value / (double)x.total));
  };
  const auto at_random = [&](u64 total) { return u >= 1.f ? total - 1 : min(share_of<false>(total, u), total - 1); };

  const long long k = t == 0.f ? 1 : (k0 <= 0 || k0 > V ? V : k0);
  const u64 low = least >= 1.f ? 1ull << 43 : (u64)ceil(fmax((double)least, 0.0) * 0x1p43);
  if (k == 1) {
    finish(locate([&](int, float x) -> u64 { return x == top; }, [](u64) -> u64 { return 0; }));
    // (a sum of one for each of the largest: what is drawn is certain)
    if (rank == 0 && tid == 0) d.logprob[r] = 0.f;
    cluster_sync();
    return;
  }

  // ---- lists: `order` (32 bits) and id of elements, the same in all CTAs, the largest first.  Returns how many, or more than SA_LIST.
  const auto collect = [&](const auto& belongs) {
    each([&](int i, float x) {
      if (belongs(i, x)) {
        const uint32_t at = atomicAdd(&s.count[0], 1);
        if (at < SA_LIST) s.list[at] = (u64)order_of(x) << 32 | (uint32_t)~i;
      }
    });
    cluster_sync();
    int n = 0, before[SA_CLUSTER + 1];
#pragma unroll
    for (int c = 0; c < SA_CLUSTER; ++c) {
      before[c] = n;
      if (c < C) n += (int)min(peek(&s.count[0], c), 1u << 21);
    }
    before[SA_CLUSTER] = n;
    if (n <= SA_LIST) {
      u64 v = 0;
      if (tid < n) {
#pragma unroll
        for (int c = 0; c < SA_CLUSTER; ++c)
          if (before[c] <= tid && tid < before[c + 1]) v = peek(&s.list[tid - before[c]], c);
        s.all[tid] = v;
      }
      __syncthreads();
      if (tid < n) {
        int above = 0;
        for (int j = 0; j < n; ++j) above += s.all[j] > v;
        s.sorted[above] = v;
      }
    }
    cluster_sync();      // the counts have been read
    if (tid == 0) s.count[0] = 0;
    __syncthreads();
    return n;
  };
  // Running sums of a value per element of the sorted list, into weights[]; returns the sum
  const auto run = [&](int n, u64 v) {
    const u64 up = warp_upto(tid < n ? v : 0);
    if (lane == 31) s.mass[warp] = up;
    __syncthreads();
    u64 front = 0, all = 0;
    for (int w = 0; w < SA_WARPS; ++w) {
      if (w < warp) front += s.mass[w];
      all += s.mass[w];
    }
    if (tid < n) s.weights[tid] = front + up;
    __syncthreads();
    return all;
  };
  const auto step_of = [&](float x, float scale) { return (int)fminf((top - x) * scale, (float)(SA_BINS - 1)); };
  const auto scale_of = [&](float lo) {
    const float range = top - lo;
    return range > 0.f && range < INFINITY ? (float)(SA_BINS - 1) / range : 0.f;
  };
  // Adds the CTAs' histograms up and clears them; every thread has four neighbouring bins, from the largest elements on
  const auto add_up = [&]() {
    cluster_sync();
    for (int i = tid; i < SA_BINS; i += SA_THREADS) {
      uint32_t n = 0;
      for (int c = 0; c < C; ++c) n += peek(&s.hist[i], c);
      s.total[i] = n;
    }
    cluster_sync();
    for (int i = tid; i < SA_BINS; i += SA_THREADS) s.hist[i] = 0;
    __syncthreads();
  };
  // The first bin at which the running sum of value(bin) reaches `limit` (the last one if none does), and the sum in front of it
  const auto crossing = [&](const auto& value, auto limit, auto& front) {
    typedef decltype(limit) S;
    S v[SA_BINS / SA_THREADS], four = 0;
#pragma unroll
    for (int j = 0; j < SA_BINS / SA_THREADS; ++j) v[j] = value(tid * (SA_BINS / SA_THREADS) + j), four += v[j];
    const S up = warp_upto(four);
    S* part = reinterpret_cast<S*>(s.mass);
    if (lane == 31) part[warp] = up;
    if (tid == 0) s.found[2] = SA_BINS;
    __syncthreads();
    S at = up - four;
    for (int w = 0; w < warp; ++w) at += part[w];
    int hit = SA_BINS;
    S before = 0;
#pragma unroll
    for (int j = 0; j < SA_BINS / SA_THREADS; ++j) {
      if (hit == SA_BINS && at + v[j] >= limit) hit = tid * (SA_BINS / SA_THREADS) + j, before = at;
      at += v[j];
    }
    if (hit < SA_BINS) atomicMin(&s.found[2], (u64)hit);
    __syncthreads();
    const int bin = (int)s.found[2];
    if (hit == bin) *reinterpret_cast<S*>(&s.found[3]) = before;
    __syncthreads();
    front = bin == SA_BINS ? S(0) : *reinterpret_cast<S*>(&s.found[3]);
    __syncthreads();
    return bin == SA_BINS ? SA_BINS - 1 : bin;
  };

  // ---- a small k: the elements that reach the k-th largest of the threads' maxima
  if (k <= SA_LIST / 2) {
    float reach = -INFINITY;
    const float scale = scale_of(least_top);
    if (most > -INFINITY) atomicAdd(&s.hist[step_of(most, scale)], 1);
    add_up();
    uint32_t front;
    const int bin = crossing([&](int b) { return s.total[b]; }, (uint32_t)k, front);
    if (front + s.total[bin] >= (uint32_t)k) {
      uint32_t m4[4];
      extremes(most > -INFINITY && step_of(most, scale) <= bin ? order_of(most) : 0xffffffffu, 0, 0xffffffffu, 0, m4);
      reach = ordered(m4[0]);
    }
    const int n = collect([&](int, float x) { return x >= reach && x > -INFINITY; });
    if (n <= SA_LIST) {
      const u64 key = tid < n ? s.sorted[tid] : 0;
      const u64 w = tid < min((long long)n, k) ? weight(ordered((uint32_t)(key >> 32))) : 0;
      const u64 total = run(n, w);
      const u64 limit = p < 1.f ? share_of<true>(total, p) : ~0ull, front_w = tid < n ? s.weights[tid] - w : 0;
      const u64 stays = tid < n && tid < k && (tid == 0 || front_w < limit) && w >= low ? w : 0;
      const u64 sum = run(n, stays), target = at_random(sum);
      // what is kept by the order of the ids: the sum in front of each
      __syncthreads();
      if (tid < n) s.all[tid] = stays;
      __syncthreads();
      if (rank == 0 && stays) {
        u64 before = 0;
        for (int j = 0; j < n; ++j)
          if ((uint32_t)s.sorted[j] > (uint32_t)key) before += s.all[j];      // ids are held inverted
        if (before <= target && target < before + stays) leave((long long)(uint32_t)~(uint32_t)key, (float)log((double)stays / (double)sum));
      }
      cluster_sync();
      return;
    }
  }

  // ---- borders: kept is what is larger than `edge`, and equal ones up to id `last`
  float edge = -INFINITY;
  int last = V;
  const auto kept = [&](int i, float x) { return x > edge || (x == edge && i <= last); };
  // Inside the elements of `belongs`, of which there are n, the border is where the running count (or sum of weights) reaches `need`
  const auto inside = [&](const auto& belongs, uint32_t n, bool mass, u64 need) {
    uint32_t lo = 0xffffffffu, hi = 0, m4[4];
    each([&](int i, float x) {
      if (belongs(i, x)) lo = min(lo, order_of(x)), hi = max(hi, order_of(x));
    });
    extremes(lo, hi, 0xffffffffu, 0, m4);
    lo = m4[0], hi = m4[1];
    while (lo < hi && n > SA_LIST) {      // steps of the order itself
      int shift = 0;
      while ((hi - lo) >> shift >= SA_BINS) ++shift;
      uint32_t above = 0;
      u64 above_w = 0;
      each([&](int i, float x) {
        const uint32_t o = order_of(x);
        if (belongs(i, x) && lo <= o && o <= hi) atomicAdd(&s.hist[(hi - o) >> shift], 1);
      });
      add_up();
      int bin;
      if (!mass) {
        bin = crossing([&](int b) { return s.total[b]; }, (uint32_t)need, above);
        need -= above;
      } else {
        // sums of weights by halving: the first bin up to which they reach what is needed
        int b0 = 0, b1 = (int)((hi - lo) >> shift);
        while (b0 < b1) {
          const int mid = (b0 + b1) >> 1;
          u64 sum = 0, s3[3];
          each([&](int i, float x) {
            const uint32_t o = order_of(x);
            if (belongs(i, x) && lo <= o && o <= hi) {
              const int b = (int)((hi - o) >> shift);
              if (b0 <= b && b <= mid) sum += weight(x);
            }
          });
          sums(sum, 0, 0, s3);
          if (above_w + s3[0] >= need) b1 = mid;
          else above_w += s3[0], b0 = mid + 1;
        }
        bin = b0;
        need -= above_w;
      }
      const uint32_t start = hi - ((uint32_t)bin << shift);
      n = s.total[bin];
      lo = max(lo, shift ? start - ((1u << shift) - 1) : start);
      hi = start;
    }
    if (lo < hi) {
      const int m = collect([&](int i, float x) { return belongs(i, x) && lo <= order_of(x) && order_of(x) <= hi; });
      const u64 key = tid < m ? s.sorted[tid] : 0;
      const u64 w = tid < m ? (mass ? weight(ordered((uint32_t)(key >> 32))) : 1) : 0;
      run(m, w);
      if (tid == 0) s.found[2] = (u64)(m - 1);
      __syncthreads();
      if (tid < m && s.weights[tid] >= need) atomicMin(&s.found[2], (u64)tid);
      __syncthreads();
      const u64 border = s.sorted[s.found[2]];
      __syncthreads();
      edge = ordered((uint32_t)(border >> 32)), last = (int)(uint32_t)~(uint32_t)border;
      return;
    }
    // equal ones: as many as are needed, by their ids
    const float value = ordered(lo);
    const u64 one = mass ? weight(value) : 1, many = one ? (need + one - 1) / one : n;
    const Place at = locate([&](int i, float x) -> u64 { return x == value && belongs(i, x); }, [&](u64 total) { return min(max(many, 1ull), total) - 1; });
    edge = value, last = at.id;
  };
  if (k < V) {
    const float lo = fmaxf(lowest, top - 48.f), scale = scale_of(lo);
    each([&](int, float x) {
      if (x > -INFINITY) atomicAdd(&s.hist[step_of(x, scale)], 1);
    });
    add_up();
    uint32_t above;
    const int bin = crossing([&](int b) { return s.total[b]; }, (uint32_t)k, above);
    if (above + s.total[bin] >= (uint32_t)k)      // else there are not so many
      inside([&](int, float x) { return x > -INFINITY && step_of(x, scale) == bin; }, s.total[bin], false, (u64)k - above);
  }
  if (p < 1.f) {
    const float lo = fmaxf(fmaxf(lowest, weigh.floor), edge), scale = scale_of(lo);
    each([&](int i, float x) {
      if (x > -INFINITY && kept(i, x)) atomicAdd(&s.hist[step_of(x, scale)], 1);
    });
    add_up();
    // by counts and the weight at the middle of a bin, about where the border is
    const float per_bin = scale > 0.f && t > 0.f ? 1.4426950f / (scale * t) : 0.f;
    const auto about = [&](int b) { return (float)s.total[b] * exp2f(-((float)b + 0.5f) * per_bin); };
    float before;
    crossing(about, INFINITY, before);
    float sum = 0.f;
    for (int w = 0; w < SA_WARPS; ++w) sum += reinterpret_cast<float*>(s.mass)[w];
    __syncthreads();
    int bin = crossing(about, p * sum, before);
    while (bin > 0 && s.total[bin] == 0) --bin;
    u64 all = 0, above = 0, in = 0, s3[3];
    each([&](int i, float x) {
      if (x > -INFINITY && kept(i, x)) {
        const u64 w = weight(x);
        const int b = step_of(x, scale);
        all += w;
        if (b < bin) above += w;
        if (b == bin) in += w;
      }
    });
    sums(all, above, in, s3);
    const u64 limit = max(share_of<true>(s3[0], p), 1ull);
    above = s3[1], in = s3[2];
    while (above >= limit || above + in < limit) {      // a bin further up or down
      const bool down = above + in < limit;
      int next = bin;
      do next += down ? 1 : -1;
      while (next > 0 && next < SA_BINS - 1 && s.total[next] == 0);
      u64 got = 0;
      each([&](int i, float x) {
        if (x > -INFINITY && kept(i, x) && step_of(x, scale) == next) got += weight(x);
      });
      sums(got, 0, 0, s3);
      if (down) above += in;
      else above -= s3[0];
      in = s3[0], bin = next;
      if (next <= 0 || next >= SA_BINS - 1) break;
    }
    inside([&](int i, float x) { return x > -INFINITY && kept(i, x) && step_of(x, scale) == bin; }, s.total[bin], true, limit > above ? limit - above : 1);
  }
  finish(locate([&](int i, float x) -> u64 {
    if (!(x >= weigh.floor) || !kept(i, x)) return 0;
    const u64 w = weight(x);
    return w >= low ? w : 0;
  }, at_random));
  cluster_sync();
}

template <typename T, bool RES, bool VEC>
static int launch(const FtkSampleDesc& d, int its, cudaStream_t s) {
  const auto kernel = sample_kernel<T, RES, VEC>;
  const size_t bytes = (sizeof(SampleShared) + 15) / 16 * 16 + (RES ? (size_t)its * SA_THREADS * 16 : 0);
  int rc = (int)cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(d.R * d.cluster));
  cfg.blockDim = dim3(SA_THREADS);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)d.cluster, at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
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
  // As many CTAs for a row as fill the SMs twice, with two steps each at least, and as many as it takes to keep the row
  int c = 1;
  while (c < SA_CLUSTER && its_of(c) > 1 && ((d.R * c < 2ll * sms && its_of(c) > 2) || its_of(c) * SA_THREADS * 16 > SA_SHARE)) c *= 2;
  d.cluster = c;
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
