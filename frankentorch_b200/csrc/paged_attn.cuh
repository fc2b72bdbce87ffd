// What the decoding attentions over a paged cache share: copies and matrix instructions of a warp, the list of tiles and the join of
// parts (paged_attention.cu says how they work together).
#pragma once
#include <math.h>

#include "ft_sm100.cuh"
#include "half_types.cuh"
#include "launch.cuh"
#include "ftk_api.h"
#include "paged_cache.h"

namespace ftk {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int PA_HEADER = 8;                 // ints of a header

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ float exp2_of(float x) {      // within 2^-22; what is below the normal numbers is 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldm4(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldm4t(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
template <typename T> __device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma16<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma16<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

struct PagedAttn {
  FtkPagedAttnDesc d;
  int group, subs, sub_heads;      // query heads per head of the cache, parts of a group, heads of a part
  bool by_head;                    // a header per head rather than per CTA: there are fewer
  int* header;                     // [heads or CTAs][PA_HEADER]: the first CTA or -1, sequence, head, place of the part, last CTA
  float* parts;                    // [CTAs][2][PA_PART]: accumulators, then maxima and sums
};
template <int ROWS, int HD> constexpr int PA_PART = (ROWS * (HD + 2) + 3) / 4 * 4;      // floats of a part: the next one starts on 16 bytes

// A place in the list of tiles: tile `t` of `tiles` of unit head `h` (head of the cache times part of the group) of sequence `b`.
struct Place {
  int b, h, t, tiles, n;
};

// A CTA's piece of the list: its first unit of `total`, units of a piece, units left of it (none: nothing to do)
struct Piece {
  long long first, total, per;
  int left;
};
// Every warp for itself: tiles in front of each lane's share of the sequences, then the sequence in which the CTA's piece begins
template <int TILE, typename F>
__device__ __forceinline__ Place first_place(const int B, const int heads, const F& length, Piece& x) {
  const int lane = threadIdx.x & 31, each = (B + 31) / 32, b0 = min(B, lane * each), b1 = min(B, b0 + each);
  long long mine = 0;
#pragma unroll 4
  for (int b = b0; b < b1; ++b) mine += (length(b) + TILE - 1) / TILE;
  long long upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  x.total = __shfl_sync(0xffffffffu, upto, 31) * heads;
  x.per = max((x.total + gridDim.x - 1) / gridDim.x, 2ll);      // a part of less than two tiles costs more to join than it saves
  x.first = x.per * blockIdx.x;
  x.left = (int)min(x.per, x.total - x.first);
  Place p = {0, 0, 0, 0, 0};
  if (x.left <= 0) return p;
  long long front = (upto - mine) * heads;
  const bool here = front <= x.first && x.first < upto * heads;
  if (here) {
    for (int b = b0; b < b1; ++b) {
      const int n = length(b), tiles = (n + TILE - 1) / TILE;
      const long long in = x.first - front;
      if (in < (long long)tiles * heads) {
        p = {b, (int)(in / tiles), (int)(in % tiles), tiles, n};
        break;
      }
      front += (long long)tiles * heads;
    }
  }
  const int owner = __ffs(__ballot_sync(0xffffffffu, here)) - 1;
  p.b = __shfl_sync(0xffffffffu, p.b, owner), p.h = __shfl_sync(0xffffffffu, p.h, owner), p.t = __shfl_sync(0xffffffffu, p.t, owner);
  p.tiles = __shfl_sync(0xffffffffu, p.tiles, owner), p.n = __shfl_sync(0xffffffffu, p.n, owner);
  return p;
}

// A part's sum l, relative to its accumulators' reference m: the reference by the sum's own power of two, and what is left of it
__device__ __forceinline__ float2 own_power(float m, float l) {
  if (l == 0.f) return make_float2(-3.402823466e38f, 0.f);      // of no tokens
  const int e = min((int)(__float_as_uint(l) >> 23 & 255) - 127, 126);
  return make_float2(m + (float)e, l * __uint_as_float((uint32_t)(127 - e) << 23));
}
// Joins the parts of a head that several CTAs had, if header blockIdx.x is of one: `together` rows from together * blockIdx.y on, and
// where that leaves threads over, several of them share a row's parts.  Sums are in a fixed order.  And since sequences of no tokens are in
// nobody's piece, the blocks write them, a sequence each.  Sums and accumulators are carried times 2^SHIFT.  FAR: a part's sum may be
// any power of two away from its accumulators, so the sums are added up by their own largest.
template <typename T, int HD, int ROWS, int SHIFT, bool FAR, int THREADS>
__global__ void __launch_bounds__(THREADS) paged_attn_join_kernel(const __grid_constant__ PagedAttn a, const int together) {
  constexpr int PART = PA_PART<ROWS, HD>, LANES = HD / 4, SLOTS = THREADS / LANES;      // threads of a row, and how many times those
  constexpr int FIRST = 4;               // parts whose accumulators a thread requests along with the statistics
  extern __shared__ float2 part_ml[];    // [parts][together]: maximum and sum, then (factor, -)
  __shared__ float sums[SLOTS], tops[SLOTS], backs[SLOTS];
  __shared__ float4 shares[SLOTS][LANES];
  const FtkPagedAttnDesc& d = a.d;
  pdl_wait();
  pdl_trigger();
  const int* h = a.header + (long long)blockIdx.x * PA_HEADER;
  const int4 head4 = *reinterpret_cast<const int4*>(h);
  const int last = h[4], own = a.by_head ? d.lengths[blockIdx.x / (unsigned)(d.Hkv * a.subs)] : 1;
  const int c = own > 0 ? head4.x : -1;      // (nobody writes the header of a head without tokens)
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, slot_of = threadIdx.x / LANES, quad = threadIdx.x % LANES;
  if (c >= 0) {
    const int b = head4.y, head = head4.z, slot = head4.w, n = last - c + 1;
    const int rows = min(a.sub_heads, a.group - (head % a.subs) * a.sub_heads);
    const float* first = a.parts + ((long long)c * 2 + slot) * PART;
    const float* rest = a.parts + (long long)c * 2 * PART;      // part i > 0 is at rest + 2 i PART
    const auto part = [&](int i) { return i == 0 ? first : rest + (long long)i * 2 * PART; };
    const int r0 = blockIdx.y * together, some = min(together, rows - r0);
    const int j = slot_of % together, share = slot_of / together, sharing = SLOTS / together;
    const auto acc_of = [&](int i) { return *reinterpret_cast<const float4*>(part(i) + (r0 + j) * HD + quad * 4); };
    float4 x[FIRST];
#pragma unroll
    for (int k = 0; k < FIRST; ++k)
      if (j < some && share + k * sharing < n) x[k] = acc_of(share + k * sharing);
    for (int i = threadIdx.x; i < n * together; i += THREADS) {
      const int p = i / together, row = i % together;
      if (row < some) part_ml[i] = make_float2(part(p)[ROWS * HD + r0 + row], part(p)[ROWS * (HD + 1) + r0 + row]);
    }
    __syncthreads();
    // a warp per row: the largest maximum, every part's factor, the sum
    for (int row = warp; row < some; row += THREADS / 32) {
      float top = -INFINITY, most = -INFINITY;
      for (int i = lane; i < n; i += 32) {
        top = fmaxf(top, part_ml[i * together + row].x);
        if (FAR) most = fmaxf(most, own_power(part_ml[i * together + row].x, part_ml[i * together + row].y).x);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (FAR) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
      }
      const float base = top == -INFINITY ? 0.f : top;
      float sum = 0.f;
      for (int i = lane; i < n; i += 32) {
        float2& ml = part_ml[i * together + row];
        if (FAR) {
          const float2 x = own_power(ml.x, ml.y);
          sum += exp2_of(x.x - most) * x.y;
        }
        ml.x = exp2f(ml.x - base);
        if (!FAR) sum += ml.x * ml.y;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0) sums[row] = sum, tops[row] = FAR ? most : top, backs[row] = FAR ? exp2f(top - most) / sum : 1.f;
    }
    __syncthreads();
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    const auto add = [&](int i, const float4& y) {
      const float e = part_ml[i * together + j].x;
      v.x += e * y.x, v.y += e * y.y, v.z += e * y.z, v.w += e * y.w;
    };
    if (j < some) {
#pragma unroll
      for (int k = 0; k < FIRST; ++k)
        if (share + k * sharing < n) add(share + k * sharing, x[k]);
#pragma unroll 8
      for (int i = share + FIRST * sharing; i < n; i += sharing) add(i, acc_of(i));
    }
    shares[slot_of][quad] = v;
    __syncthreads();
    if (share == 0 && j < some) {
      for (int k = 1; k < sharing; ++k) {
        const float4 y = shares[k * together + j][quad];
        v.x += y.x, v.y += y.y, v.z += y.z, v.w += y.w;
      }
      const float sum = sums[j], by = sum == 0.f ? 0.f : FAR ? backs[j] : 1.f / sum;
      const int q = (head / a.subs) * a.group + (head % a.subs) * a.sub_heads + r0 + j;
      if (sum == 0.f) v = make_float4(0.f, 0.f, 0.f, 0.f);
      v.x *= by, v.y *= by, v.z *= by, v.w *= by;
      *reinterpret_cast<uint2*>((T*)d.o + b * d.o_bs + q * d.o_hs + quad * 4) = make_uint2(Half16<T>::down(v.x, v.y), Half16<T>::down(v.z, v.w));
      if (quad == 0) d.lse[(long long)b * d.Hq + q] = sum == 0.f ? -INFINITY : (tops[j] + log2f(sum) - (float)SHIFT) * LN2;
    }
  }
  for (int b = blockIdx.x; b < (int)d.B; b += gridDim.x) {
    if (d.lengths[b] > 0) continue;
    for (int i = blockIdx.y * THREADS + threadIdx.x; i < (int)d.Hq * LANES; i += gridDim.y * THREADS)
      *reinterpret_cast<uint2*>((T*)d.o + b * d.o_bs + (i / LANES) * d.o_hs + (i % LANES) * 4) = make_uint2(0, 0);
    for (int i = blockIdx.y * THREADS + threadIdx.x; i < (int)d.Hq; i += gridDim.y * THREADS) d.lse[(long long)b * d.Hq + i] = -INFINITY;
  }
}

// The launch of the join: few heads have many parts each: a row per block, its parts shared by the block's threads.  Else the rows of a
// head, as far as shared memory goes.
template <typename T, int HD, int ROWS, int SHIFT, bool FAR = false, int THREADS = 256>
static int launch_join(const PagedAttn& a, long long heads, long long ctas, long long headers, cudaStream_t s) {
  constexpr int slots = THREADS / (HD / 4);
  int together = 1;
  while (heads > 32 && together < a.sub_heads && together < slots && ctas * together * 2 * sizeof(float2) <= 40 * 1024)
    together *= 2;
  return launch_pdl(paged_attn_join_kernel<T, HD, ROWS, SHIFT, FAR, THREADS>, dim3((unsigned)headers, (unsigned)((a.sub_heads + together - 1) / together)), dim3(THREADS),
                    (size_t)ctas * together * sizeof(float2), s, a, together);
}

}  // namespace ftk
