// Attention of one new token per sequence over a paged key-value cache.
//
// Mathematics.  With scores x_t = scale q . k_t the running maximum m, the sum l = sum_t exp(x_t - m) and the accumulator
// a = sum_t exp(x_t - m) v_t are carried over the tokens; a larger maximum rescales l and a by exp(m_old - m_new).  Two parts join
// the same way.  o = a / l, lse = m + log(l); a part of no tokens has m = -inf, l = 0.
//
// What bounds it: every key and value is read once, 1 to 16 flops a byte, so it is the copy bandwidth.
//
// Work.  A unit is a tile of 64 tokens of one head of the cache with the (up to 16) query heads that share it, so keys and values
// are read once for the group.  The units of all sequences and heads are one list, of which each of the CTAs (two or three per SM)
// takes an equal piece: ragged batches, few long sequences and many short ones all keep every SM busy to the end.  The list is made from
// the lengths on the device, so a captured launch follows them.  A CTA that has a whole head writes the output; pieces of one are
// left as (m, l, a) in the call's scratch and joined by a second kernel, always in the order of the tokens.  Where the table is so
// short that nothing is worth splitting a CTA takes one head and there is no second kernel; with an SM for each head it has 8 or 16
// warps instead of four, since one warp per scheduler needs 1400 cycles for 16 tokens (12 heads of 64, 500 tokens: 5.3 us, 8.1 with four).
//
// Inside a CTA each of the warps takes 16 tokens of the tile on its own, through a ring of stages in shared memory that it fills
// with 16-byte asynchronous copies several tiles (and heads, and sequences) ahead: no barrier but the warp's own until the end of a
// head.  Scores and the product with V are 16 x 8 x 16 matrix instructions of the warp (mma.sync): rows of a tile are the query
// heads of the group, of which there are too few for a tile of the tensor memory's 128 rows, and a quarter of the warp
// instructions' rate is enough to keep up with the memory.  Probabilities are needed in 16 bits there; rounding them once would
// cost as much accuracy as the rounding of the output, so each is split into two 16-bit halves, p = hi + lo with an error of
// 2^-17: for groups of up to 8 heads the lo halves are the rows 8 to 15 of the same instruction, which are idle otherwise.  A lo of
// 0 makes NaN of an infinite value, so elements that end as NaN are added up again with undivided probabilities (pa_infinite()).
#include <math.h>

#include "ft_sm100.cuh"
#include "half_types.cuh"
#include "launch.cuh"
#include "ftk_api.h"
#include "paged_cache.h"

extern "C" int* ftk_status_word(void);

namespace ftk {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int PA_WARPS = 4, PA_TILE = 16 * PA_WARPS;      // of a CTA that shares its SM
// Tiles of 64 tokens, by the width of the table, up to which a head is left whole: a second launch and the join cost 3 - 4 us, so few heads
// are cut late, and heads for all SMs fill the time among themselves.  Whole and cut (us) with all positions in use, an SM for each head:
// 12 heads of 64, 16 tiles 8.1 and 8.6, 32 tiles 13.7 and 9.2; 32 heads of 128, up to 17 tiles 13.1 and 10.7; 128 heads of 128, up to 17
// 13.7 and 16.4, up to 33 22.4 and 25.0; with several heads per SM, 256 of 128, up to 17 21.7 and 26.4, up to 33 38.0 and 36.9.  A straight
// line below these borders: for a dozen heads it cuts from 12 tiles on where 17 would do, and the width stands for lengths that only the
// device knows, so few tokens under a wide table are cut too (12 heads of 64, 301 tokens: 4.8 us under 5 tiles, 8.9 under 16).
__host__ inline long long pa_whole(long long heads, long long sms) { return heads <= sms ? 9 + 28 * heads / sms : 20; }
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
// fp16 has five bits of exponent: probabilities are carried times 2^15, so that what underflows is 2^-39 of the largest.
template <typename T> struct PaShift { static constexpr float value = 0.f; };
template <> struct PaShift<__half> { static constexpr float value = 15.f; };

struct PagedAttn {
  FtkPagedAttnDesc d;
  int group, subs, sub_heads;      // query heads per head of the cache, parts of a group, heads of a part
  bool by_head;                    // a header per head rather than per CTA: there are fewer
  int* header;                     // [heads or CTAs][PA_HEADER]: the first CTA or -1, sequence, head, place of the part, last CTA
  float* parts;                    // [CTAs][2][rows][hd + 2]: accumulators, then maxima and sums
};

// A place in the list of tiles: tile `t` of `tiles` of unit head `h` (head of the cache times part of the group) of sequence `b`.
struct Place {
  int b, h, t, tiles, n;
};

// W warps of a CTA: CTAs of an SM, bytes of a warp's ring (three to six stages of 16 tokens)
template <int ROWS, int HD, int W> struct PaSmem {
  static constexpr int CTAS = W > PA_WARPS ? 1 : (HD == 64 && ROWS == 8 ? 3 : 2);
  static constexpr int RING = W == 16 ? 12 * 1024 : (CTAS == 3 ? 16 * 1024 : 24 * 1024);
  static constexpr int STAGE = 16 * HD * 4, STAGES = RING / STAGE;
  static constexpr int MERGE = W * ROWS * 64 * 4;             // accumulators of 64 columns of all warps
  static constexpr bool OWN = W <= PA_WARPS;                  // in memory of their own, or in the rings of a head that is through
  static constexpr int BYTES = W * RING + (OWN ? MERGE : 0) + 2 * W * ROWS * 4 + W * STAGES * 4;
  static_assert(OWN || MERGE <= W * RING, "the accumulators fit the rings");
  static_assert(CTAS * (BYTES + 1024) <= 228 * 1024, "the CTAs of an SM share its memory");
};
// Warps of a CTA that has its SM and one head for itself: as many as registers and rings allow
template <int ROWS, int HD> constexpr int PA_ALONE = HD == 64 && ROWS == 8 ? 16 : 8;

// An element of the output whose column has infinities or NaN among the values of tokens [t, end), as a sum of those alone with their
// whole probabilities: exp2(x - base), positive for every score that fp32 can tell from the maximum.  `was` where there are none: NaN
// came from elsewhere.  `q`: the query; `k`, `v`: the head's first row of the cache, `v` from the element's column on.  Nobody comes here
// but with NaN.
template <typename T, int HD>
__device__ __forceinline__ float pa_infinite(const FtkPagedAttnDesc& d, const int b, const T* q, const T* k, const T* v, const int t, const int end,
                                          const float base, const float was) {
  constexpr int AT_ONCE = 8;
  const PagedTable table = {d.table, d.table_stride, d.table_cols, d.n_pages, (int)d.page_shift};
  const float sc = (float)d.scale * LOG2E;
  float sum = 0.f;
  bool some = false;
#pragma unroll 1
  for (int from = t; from < end; from += AT_ONCE) {
    unsigned odd = 0;
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      const long long page = from + i < end ? paged_page(table, b, from + i) : -1;
      const float y = page < 0 ? 0.f : Half16<T>::one(v[page * d.vp_ps + paged_row(table, from + i) * d.vp_rs]);
      odd |= isfinite(y) ? 0u : 1u << i;
    }
#pragma unroll 1
    for (; odd; odd &= odd - 1) {
      const int at = from + __ffs(odd) - 1;
      const long long page = paged_page(table, b, at), row = paged_row(table, at);
      const T* key = k + page * d.kp_ps + row * d.kp_rs;
      float x = 0.f;
#pragma unroll 1
      for (int e = 0; e < HD; ++e) x += Half16<T>::one(q[e]) * Half16<T>::one(key[e]);
      sum += exp2f(x * sc - base + PaShift<T>::value) * Half16<T>::one(v[page * d.vp_ps + row * d.vp_rs]);
      some = true;
    }
  }
  return some ? sum : was;
}

template <typename T, int HD, int ROWS, bool SPLIT, int W>
__global__ void __launch_bounds__(W * 32, PaSmem<ROWS, HD, W>::CTAS) paged_attn_kernel(const __grid_constant__ PagedAttn a, int* status) {
  typedef PaSmem<ROWS, HD, W> SM;
  static_assert(!SPLIT || SM::OWN, "a piece goes on while the parts are joined");
  constexpr int TILE = 16 * W;
  constexpr int STAGES = SM::STAGES, STAGE = SM::STAGE, CH = HD / 8, NT = HD / 8, KS = HD / 16;
  constexpr int RR = ROWS / 8;
  constexpr float SHIFT = PaShift<T>::value;
  extern __shared__ __align__(256) unsigned char smem[];      // rows of 256 bytes are addressed by exclusive or
  const FtkPagedAttnDesc& d = a.d;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, heads = (int)d.Hkv * a.subs;
  unsigned char* ring = smem + warp * SM::RING;
  float* merge = reinterpret_cast<float*>(smem + (SM::OWN ? W * SM::RING : 0));
  float* stat = reinterpret_cast<float*>(smem + W * SM::RING + (SM::OWN ? SM::MERGE : 0));                                     // [2][warps][ROWS]
  unsigned* there = reinterpret_cast<unsigned*>(stat + 2 * W * ROWS) + warp * STAGES;
  const PagedTable table = {d.table, d.table_stride, d.table_cols, d.n_pages, (int)d.page_shift};
  const auto length = [&](int b) {
    bool bad;
    const long long n = paged_length(table, d.lengths[b], bad);
    if (bad) ft_index_ok(-1, 1, status);
    return (int)n;
  };
  const auto row0 = [&](int h) { return (h / a.subs) * a.group + (h % a.subs) * a.sub_heads; };      // first query head
  const auto rows_of = [&](int h) { return min(a.sub_heads, a.group - (h % a.subs) * a.sub_heads); };
  pdl_wait();
  pdl_trigger();

  constexpr int AHEAD = STAGES - 1;     // tiles whose pages are known before they are asked for
  const bool one_page = table.shift >= 4;
  const int tok_of = warp * 16 + (one_page ? 0 : lane & 15);      // of a tile: the token whose page this lane looks up

  // ---- this CTA's piece of the list
  Place p;
  int left;                             // tiles of the piece (counters of 64 bits took 5 % more for heads of 64)
  long long first_unit = 0, total = 0, per = 0;
  int entry[AHEAD];
  if (!SPLIT) {
    p.b = blockIdx.x / heads, p.h = blockIdx.x % heads, p.t = 0;
    // the first entries of the table along with the length that says whether they count
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const long long col = (i * TILE + tok_of) >> table.shift;
      entry[i] = col < table.cols ? table.table[p.b * table.stride + col] : -1;
    }
    p.n = length(p.b), p.tiles = (p.n + TILE - 1) / TILE;
    left = p.tiles;
  } else {
    // Every warp for itself: tiles in front of each lane's share of the sequences, then the sequence in which the piece begins
    const int each = ((int)d.B + 31) / 32, b0 = min((int)d.B, lane * each), b1 = min((int)d.B, b0 + each);
    long long mine = 0;
#pragma unroll 4
    for (int b = b0; b < b1; ++b) mine += (length(b) + TILE - 1) / TILE;
    long long upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    total = __shfl_sync(0xffffffffu, upto, 31) * heads;
    per = max((total + gridDim.x - 1) / gridDim.x, 2ll);      // a part of less than two tiles costs more to join than it saves
    first_unit = per * blockIdx.x;
    left = (int)min(per, total - first_unit);
    if (!a.by_head && threadIdx.x == 0) a.header[(long long)blockIdx.x * PA_HEADER] = -1;
    if (left <= 0) return;
    long long front = (upto - mine) * heads;
    p = {0, 0, 0, 0, 0};
    const bool here = front <= first_unit && first_unit < upto * heads;
    if (here) {
      for (int b = b0; b < b1; ++b) {
        const int n = length(b), tiles = (n + TILE - 1) / TILE;
        const long long in = first_unit - front;
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
  }

  // ---- loads: the ring is filled from a place of its own, which runs ahead over heads and sequences, and the table is read from
  // another one as far ahead of that
  const auto advance = [&](Place& x, int& more) {
    --more;
    if (++x.t == x.tiles) {
      x.t = 0;
      if (++x.h == heads) {
        x.h = 0;
        x.tiles = 0;
        while (more > 0 && x.tiles == 0 && x.b + 1 < (int)d.B) x.n = length(++x.b), x.tiles = (x.n + TILE - 1) / TILE;
      }
    }
  };
  Place f = p, g = p;
  int to_load = left, to_look = left;
  // Pages of the next tiles.  A page of 16 rows or more holds all of a warp's part of a tile; of smaller ones lane j < 16 has token j's.
  int page_of[AHEAD] = {};
  const auto look = [&]() {
    int page = -1;
    if (to_look > 0) {
      const int tok = g.t * TILE + tok_of;
      if (tok < g.n) {
        page = (int)paged_page(table, g.b, tok);
        if (page < 0) ft_index_ok(-1, 1, status);
      }
      advance(g, to_look);
    }
    return page;
  };
  const uint32_t ring_s = smem_u32(ring);
  const int lrow = lane / CH, lchunk = lane % CH;
  constexpr int RSTEP = 32 / CH, COPIES = 16 / RSTEP;      // rows of a copy of the warp, copies of 16 rows
  const uint32_t lane_at = lrow * (HD * 2), lane_sw = lchunk << 4;
  const long long k_lane = lrow * d.kp_rs + lchunk * 8, v_lane = lrow * d.vp_rs + lchunk * 8;
  const auto load = [&](int stage) {
    const int pages = page_of[0];
#pragma unroll
    for (int i = 0; i + 1 < AHEAD; ++i) page_of[i] = page_of[i + 1];
    page_of[AHEAD - 1] = look();
    if (to_load > 0) {
      const int head = f.h / a.subs, tok0 = f.t * TILE + warp * 16;
      const T* kb = (const T*)d.k_pages + head * d.kp_hs;
      const T* vb = (const T*)d.v_pages + head * d.vp_hs;
      const uint32_t dst = ring_s + stage * STAGE + lane_at;
      unsigned ok;
      if (one_page) {
        const int n = pages < 0 ? 0 : min(16, f.n - tok0);      // rows that are there
        const long long page = pages < 0 ? 0 : pages, in = paged_row(table, tok0);
        ok = (1u << n) - 1;
        const T* k = kb + page * d.kp_ps + in * d.kp_rs + k_lane;
        const T* v = vb + page * d.vp_ps + in * d.vp_rs + v_lane;
        const long long k_step = RSTEP * d.kp_rs, v_step = RSTEP * d.vp_rs;
#pragma unroll
        for (int c = 0; c < COPIES; ++c) {
          const bool t = c * RSTEP + lrow < n;
          const uint32_t at = dst + c * RSTEP * HD * 2 + (lane_sw ^ (((c * RSTEP + lrow) & 7) << 4));
          copy16(at, t ? k : kb, t);
          copy16(at + 16 * HD * 2, t ? v : vb, t);
          k += k_step, v += v_step;
        }
      } else {
        ok = __ballot_sync(0xffffffffu, pages >= 0) & 0xffffu;
#pragma unroll
        for (int c = 0; c < COPIES; ++c) {
          const int row = c * RSTEP + lrow;
          const long long page = __shfl_sync(0xffffffffu, pages, row), in = paged_row(table, tok0 + row);
          const bool t = page >= 0;
          const uint32_t at = dst + c * RSTEP * HD * 2 + (lane_sw ^ ((row & 7) << 4));
          copy16(at, t ? kb + page * d.kp_ps + in * d.kp_rs + lchunk * 8 : kb, t);
          copy16(at + 16 * HD * 2, t ? vb + page * d.vp_ps + in * d.vp_rs + lchunk * 8 : vb, t);
        }
      }
      if (lane == 0) there[stage] = ok;
      advance(f, to_load);
    }
    copy_commit();
  };
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) {
    if (SPLIT) {
      page_of[i] = look();
    } else {
      page_of[i] = to_look > 0 && g.t * TILE + tok_of < g.n && ft_index_ok(entry[i], table.n_pages, status) ? entry[i] : -1;
      if (to_look > 0) advance(g, to_look);
    }
  }
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) load(s);

  // ---- tiles
  const float sc = (float)d.scale * LOG2E;
  uint32_t q[KS][ROWS == 16 ? 4 : 2];
  float acc[NT][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  const int r0 = lane >> 2, c0 = (lane & 3) * 2;
  const auto begin = [&]() {            // queries of the head at `p`; rows beyond the group are zero
    const int first = row0(p.h), rows = rows_of(p.h);
    const T* base = (const T*)d.q + p.b * d.q_bs;
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int i = 0; i < (ROWS == 16 ? 4 : 2); ++i) {
        const int row = r0 + (ROWS == 16 && (i & 1) ? 8 : 0), col = k * 16 + c0 + ((ROWS == 16 ? i >> 1 : i) ? 8 : 0);
        q[k][i] = row < rows ? *reinterpret_cast<const uint32_t*>(base + (first + row) * d.q_hs + col) : 0u;
      }
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = 0.f;
  };
  bool begun = p.t == 0;                // the piece has the beginning of the head at `p`
  int parts = 0;
  begin();
  // this lane's rows for ldmatrix: chunk c of row r is at c ^ (r & 7), so the chunks of a step differ by an exclusive or
  const int k_row = ((lane >> 4) << 3) + (lane & 7), v_row = (((lane >> 3) & 1) << 3) + (lane & 7);
  const uint32_t k_at = k_row * (HD * 2) + ((((lane >> 3) & 1) ^ (k_row & 7)) << 4);
  const uint32_t v_at = 16 * HD * 2 + v_row * (HD * 2) + (((lane >> 4) ^ (v_row & 7)) << 4);
  int stage = 0;
  for (bool more = true; more; more = left > 0) {
    if (left > 0) {
      copy_wait<STAGES - 2>();
      __syncwarp();
      const uint32_t ks = ring_s + stage * STAGE + k_at, vs = ring_s + stage * STAGE + v_at;
      const unsigned ok = there[stage];
      const int refill = stage == 0 ? STAGES - 1 : stage - 1;
      float s[2][4] = {};
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        uint32_t b[4];
        ldm4(ks ^ (k << 5), b);
        const uint32_t qa[4] = {q[k][0], ROWS == 16 ? q[k][1] : 0u, ROWS == 16 ? q[k][ROWS == 16 ? 2 : 0] : q[k][1],
                                ROWS == 16 ? q[k][ROWS == 16 ? 3 : 0] : 0u};
        mma16<T>(s[0], qa, b[0], b[1]);
        mma16<T>(s[1], qa, b[2], b[3]);
      }
      load(refill);                     // the stage that the tile before left: its reads are behind the warp's barrier
      // masked scores, and the larger maximum of the row's sixteen tokens and what was there
      uint32_t hi[4] = {}, lo[4] = {};
      float grow[2];
      bool moved = false;
#pragma unroll
      for (int r = 0; r < RR; ++r) {
        float x[4], top = m[r];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = s[i >> 1][2 * r + (i & 1)] * sc;
        if (ok != 0xffffu) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (!(ok >> ((i >> 1) * 8 + c0 + (i & 1)) & 1u)) x[i] = -INFINITY;
        }
        top = fmaxf(fmaxf(top, fmaxf(x[0], x[1])), fmaxf(x[2], x[3]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float base = top == -INFINITY ? 0.f : top;
        moved |= top != m[r];
        grow[r] = exp2_of(m[r] - base);
        m[r] = top;
        float e[4], h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = exp2_of(x[i] - base + SHIFT);
        l[r] = l[r] * grow[r] + ((e[0] + e[1]) + (e[2] + e[3]));
        hi[r] = Half16<T>::down(e[0], e[1]), hi[2 + r] = Half16<T>::down(e[2], e[3]);
        const float2 u = Half16<T>::up(hi[r]), w = Half16<T>::up(hi[2 + r]);
        h[0] = u.x, h[1] = u.y, h[2] = w.x, h[3] = w.y;
        lo[r] = Half16<T>::down(e[0] - h[0], e[1] - h[1]), lo[2 + r] = Half16<T>::down(e[2] - h[2], e[3] - h[3]);
      }
      if (__any_sync(0xffffffffu, moved)) {
        const float g0 = grow[0], g1 = ROWS == 16 ? grow[ROWS == 16 ? 1 : 0] : grow[0];
#pragma unroll
        for (int i = 0; i < NT; ++i) acc[i][0] *= g0, acc[i][1] *= g0, acc[i][2] *= g1, acc[i][3] *= g1;
      }
      if (ROWS != 16) hi[1] = lo[0], hi[3] = lo[2];
#pragma unroll
      for (int i = 0; i < NT; i += 2) {
        uint32_t b[4];
        ldm4t(vs ^ (i << 4), b);
        mma16<T>(acc[i], hi, b[0], b[1]);
        mma16<T>(acc[i + 1], hi, b[2], b[3]);
        if (ROWS == 16) {
          mma16<T>(acc[i], lo, b[0], b[1]);
          mma16<T>(acc[i + 1], lo, b[2], b[3]);
        }
      }
      stage = stage + 1 == STAGES ? 0 : stage + 1;
      --left;
      ++p.t;
    }
    if (left > 0 && p.t < p.tiles) continue;

    // ---- the end of a head, or of the piece: the warps' parts become one, over 64 columns at a time
#pragma unroll
    for (int r = 0; r < RR; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      if ((lane & 3) == 0) {
        stat[warp * ROWS + r * 8 + r0] = m[r];
        stat[(W + warp) * ROWS + r * 8 + r0] = l[r];
      }
    }
    const bool whole = begun && p.t == p.tiles;
    const int first = row0(p.h), rows = rows_of(p.h);
    float* part = SPLIT ? a.parts + ((long long)blockIdx.x * 2 + parts) * ROWS * (HD + 2) : nullptr;
    __syncthreads();
    float scale[RR];                    // of the warp's part: to the maximum of all
#pragma unroll
    for (int r = 0; r < RR; ++r) {
      float top = m[r];
#pragma unroll
      for (int w = 0; w < W; ++w) top = fmaxf(top, stat[w * ROWS + r * 8 + r0]);
      scale[r] = exp2f(m[r] - (top == -INFINITY ? 0.f : top));
    }
    // all columns of a few rows at once, else 64 of all rows
    const int cols = rows * HD <= ROWS * 64 ? HD : 64;
    for (int from = 0; from < HD; from += cols) {
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        if (i * 8 < from || i * 8 >= from + cols) continue;
        float* to = merge + (warp * rows + r0) * cols + i * 8 - from + c0;
        const float* c = acc[i];
        if (ROWS == 16) {
          if (r0 < rows) *reinterpret_cast<float2*>(to) = make_float2(c[0] * scale[0], c[1] * scale[0]);
          if (r0 + 8 < rows) *reinterpret_cast<float2*>(to + 8 * cols) = make_float2(c[2] * scale[RR - 1], c[3] * scale[RR - 1]);
        } else {
          if (r0 < rows) *reinterpret_cast<float2*>(to) = make_float2((c[0] + c[2]) * scale[0], (c[1] + c[3]) * scale[0]);
        }
      }
      __syncthreads();
      for (int i = threadIdx.x; i < rows * cols / 2; i += W * 32) {
        const int row = i / (cols / 2), in = (i % (cols / 2)) * 2, col = from + in;
        float2 v = make_float2(0.f, 0.f);
        float top = stat[row], sum = 0.f;
#pragma unroll
        for (int w = 1; w < W; ++w) top = fmaxf(top, stat[w * ROWS + row]);
        const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const float2 x = *reinterpret_cast<const float2*>(merge + (w * rows + row) * cols + in);
          v.x += x.x, v.y += x.y;
          sum += exp2f(stat[w * ROWS + row] - base) * stat[(W + w) * ROWS + row];
        }
        if (sum == sum && (v.x != v.x || v.y != v.y)) {
          const int kv = p.h / a.subs, start = begun ? 0 : p.t - ((int)min(per, total - first_unit) - left);      // the piece's first tile
          const T* qr = (const T*)d.q + p.b * d.q_bs + (first + row) * d.q_hs;
          const T* kr = (const T*)d.k_pages + kv * d.kp_hs;
          const T* vr = (const T*)d.v_pages + kv * d.vp_hs + col;
          const int end = min(p.n, p.t * TILE);
          if (v.x != v.x) v.x = pa_infinite<T, HD>(d, p.b, qr, kr, vr, start * TILE, end, base, v.x);
          if (v.y != v.y) v.y = pa_infinite<T, HD>(d, p.b, qr, kr, vr + 1, start * TILE, end, base, v.y);
        }
        if (!SPLIT || whole) {
          const float by = sum == 0.f ? 0.f : 1.f / sum;
          T* o = (T*)d.o + p.b * d.o_bs + (first + row) * d.o_hs + col;
          *reinterpret_cast<uint32_t*>(o) = Half16<T>::down(sum == 0.f ? 0.f : v.x * by, sum == 0.f ? 0.f : v.y * by);
          if (col == 0) d.lse[(long long)p.b * d.Hq + first + row] = sum == 0.f ? -INFINITY : (top + log2f(sum) - SHIFT) * LN2;
        } else {
          *reinterpret_cast<float2*>(part + row * HD + col) = v;
          if (col == 0) part[ROWS * HD + row] = top, part[ROWS * (HD + 1) + row] = sum;
        }
      }
      __syncthreads();
    }
    if (!SPLIT) return;
    // the part that has the beginning of its head says who has the rest, up to the CTA of the head's last tile
    if (begun && threadIdx.x == 0 && (a.by_head || !whole)) {
      const long long behind = first_unit + min(per, total - first_unit);
      int* h = a.header + (a.by_head ? (long long)p.b * heads + p.h : (long long)blockIdx.x) * PA_HEADER;
      h[0] = whole ? -1 : (int)blockIdx.x;
      h[1] = p.b, h[2] = p.h, h[3] = parts, h[4] = (int)((behind + (p.tiles - p.t) - 1) / per);
    }
    parts = 1;
    if (left <= 0) return;
    // the next head
    begun = true;
    p.t = 0;
    if (++p.h == heads) {
      p.h = 0;
      p.tiles = 0;
      while (p.tiles == 0 && p.b + 1 < (int)d.B) p.n = length(++p.b), p.tiles = (p.n + TILE - 1) / TILE;
    }
    begin();
  }
}

// Joins the parts of a head that several CTAs had, if header blockIdx.x is of one: `together` rows from together * blockIdx.y on, and
// where that leaves threads over, several of them share a row's parts.  Sums are in a fixed order.  And since sequences of no tokens are in
// nobody's piece, the blocks write them, a sequence each.
template <typename T, int HD, int ROWS>
__global__ void __launch_bounds__(256) paged_attn_join_kernel(const __grid_constant__ PagedAttn a, const int together) {
  constexpr float SHIFT = PaShift<T>::value;
  constexpr int PART = ROWS * (HD + 2), LANES = HD / 4, SLOTS = 256 / LANES;      // threads of a row, and how many times those
  constexpr int FIRST = 4;               // parts whose accumulators a thread requests along with the statistics
  extern __shared__ float2 part_ml[];    // [parts][together]: maximum and sum, then (factor, -)
  __shared__ float sums[SLOTS], tops[SLOTS];
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
    for (int i = threadIdx.x; i < n * together; i += 256) {
      const int p = i / together, row = i % together;
      if (row < some) part_ml[i] = make_float2(part(p)[ROWS * HD + r0 + row], part(p)[ROWS * (HD + 1) + r0 + row]);
    }
    __syncthreads();
    // a warp per row: the largest maximum, every part's factor, the sum
    for (int row = warp; row < some; row += 8) {
      float top = -INFINITY;
      for (int i = lane; i < n; i += 32) top = fmaxf(top, part_ml[i * together + row].x);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float base = top == -INFINITY ? 0.f : top;
      float sum = 0.f;
      for (int i = lane; i < n; i += 32) {
        float2& ml = part_ml[i * together + row];
        ml.x = exp2f(ml.x - base);
        sum += ml.x * ml.y;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0) sums[row] = sum, tops[row] = top;
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
      const float sum = sums[j], by = sum == 0.f ? 0.f : 1.f / sum;
      const int q = (head / a.subs) * a.group + (head % a.subs) * a.sub_heads + r0 + j;
      if (sum == 0.f) v = make_float4(0.f, 0.f, 0.f, 0.f);
      *reinterpret_cast<uint2*>((T*)d.o + b * d.o_bs + q * d.o_hs + quad * 4) = make_uint2(Half16<T>::down(v.x * by, v.y * by), Half16<T>::down(v.z * by, v.w * by));
      if (quad == 0) d.lse[(long long)b * d.Hq + q] = sum == 0.f ? -INFINITY : (tops[j] + log2f(sum) - SHIFT) * LN2;
    }
  }
  for (int b = blockIdx.x; b < (int)d.B; b += gridDim.x) {
    if (d.lengths[b] > 0) continue;
    for (int i = blockIdx.y * 256 + threadIdx.x; i < (int)d.Hq * LANES; i += gridDim.y * 256)
      *reinterpret_cast<uint2*>((T*)d.o + b * d.o_bs + (i / LANES) * d.o_hs + (i % LANES) * 4) = make_uint2(0, 0);
    for (int i = blockIdx.y * 256 + threadIdx.x; i < (int)d.Hq; i += gridDim.y * 256) d.lse[(long long)b * d.Hq + i] = -INFINITY;
  }
}

struct Plan {
  int subs, sub_heads, rows;
  bool split, alone;               // heads cut into pieces; a CTA per SM, for few heads
  long long ctas, heads, headers, bytes;      // heads: of all sequences, a part of a group counting as one
};
static Plan plan_of(const FtkPagedAttnDesc& d) {
  Plan p;
  const long long group = d.Hq / d.Hkv;
  p.subs = (int)((group + 15) / 16);
  p.sub_heads = (int)((group + p.subs - 1) / p.subs);
  p.rows = p.sub_heads <= 8 ? 8 : 16;
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  p.ctas = p.heads = d.B * d.Hkv * p.subs;
  p.headers = p.bytes = 0;
  const long long tiles = ((d.table_cols << d.page_shift) + PA_TILE - 1) / PA_TILE;
  p.alone = p.heads <= sms;
  p.split = tiles > pa_whole(p.heads, sms);
  if (p.split) {
    p.ctas = (d.hd == 64 && p.rows == 8 ? PaSmem<8, 64, PA_WARPS>::CTAS : 2ll) * sms;
    p.headers = p.heads < p.ctas ? p.heads : p.ctas;
    p.bytes = p.headers * PA_HEADER * 4 + p.ctas * 2 * p.rows * (d.hd + 2) * 4;
  }
  return p;
}

template <typename T, int HD, int ROWS>
static int launch(const FtkPagedAttnDesc& d, const Plan& p, void* scratch, cudaStream_t s) {
  PagedAttn a = {d, (int)(d.Hq / d.Hkv), p.subs, p.sub_heads, p.heads < p.ctas, (int*)scratch, nullptr};
  a.parts = (float*)((char*)scratch + p.headers * PA_HEADER * 4);
  int* status = ftk_status_word();
  if (!p.split && p.alone) {
    constexpr int W = PA_ALONE<ROWS, HD>, bytes = PaSmem<ROWS, HD, W>::BYTES;
    const auto kernel = paged_attn_kernel<T, HD, ROWS, false, W>;
    const int rc = (int)cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    return rc ? rc : launch_pdl(kernel, dim3((unsigned)p.ctas), dim3(W * 32), bytes, s, a, status);
  }
  constexpr int bytes = PaSmem<ROWS, HD, PA_WARPS>::BYTES;
  const auto whole = paged_attn_kernel<T, HD, ROWS, false, PA_WARPS>, split = paged_attn_kernel<T, HD, ROWS, true, PA_WARPS>;
  const auto kernel = p.split ? split : whole;
  int rc = (int)cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (rc) return rc;
  rc = launch_pdl(kernel, dim3((unsigned)p.ctas), dim3(PA_WARPS * 32), bytes, s, a, status);
  if (rc || !p.split) return rc;
  // Few heads have many parts each: a row per block, its parts shared by the block's threads.  Else the rows of a head, as far as
  // shared memory goes.
  constexpr int slots = 256 / (HD / 4);
  int together = 1;
  while (p.heads > 32 && together < p.sub_heads && together < slots && p.ctas * together * 2 * sizeof(float2) <= 40 * 1024)
    together *= 2;
  return launch_pdl(paged_attn_join_kernel<T, HD, ROWS>, dim3((unsigned)p.headers, (unsigned)((p.sub_heads + together - 1) / together)), dim3(256),
                    (size_t)p.ctas * together * sizeof(float2), s, a, together);
}

static bool refused(const FtkPagedAttnDesc* d) {
  return !d || d->B <= 0 || d->B > (1 << 30) || d->Hkv <= 0 || d->Hq <= 0 || d->Hq % d->Hkv || d->Hq > (1 << 20) || (d->hd != 64 && d->hd != 128) ||
         (d->type != FTK_T_BF16 && d->type != FTK_T_FP16) || d->page_shift < 0 || d->page_shift > 30 || d->table_cols <= 0 ||
         d->table_cols > (0x7fffff00ll >> d->page_shift) || d->n_pages <= 0 || d->n_pages > 0x7fffffff || d->B * d->Hq > 0x7fffffff ||
         d->B * d->Hq * (((d->table_cols << d->page_shift) >> 6) + 1) > (1ll << 38);      // a CTA counts its tiles in 32 bits
}

}  // namespace ftk
using namespace ftk;

extern "C" long long ftk_paged_attn_scratch(const FtkPagedAttnDesc* d) { return refused(d) ? -2 : plan_of(*d).bytes; }

extern "C" int ftk_paged_attn(const FtkPagedAttnDesc* d, void* scratch, void* stream) {
  if (refused(d) || !d->q || !d->o || !d->lse || !d->k_pages || !d->v_pages || !d->table || !d->lengths) return -2;
  const Plan p = plan_of(*d);
  if (p.split && !scratch) return -2;
  cudaStream_t s = (cudaStream_t)stream;
  const bool bf = d->type == FTK_T_BF16;
  if (p.rows == 8) {
    if (d->hd == 64) return bf ? launch<__nv_bfloat16, 64, 8>(*d, p, scratch, s) : launch<__half, 64, 8>(*d, p, scratch, s);
    return bf ? launch<__nv_bfloat16, 128, 8>(*d, p, scratch, s) : launch<__half, 128, 8>(*d, p, scratch, s);
  }
  if (d->hd == 64) return bf ? launch<__nv_bfloat16, 64, 16>(*d, p, scratch, s) : launch<__half, 64, 16>(*d, p, scratch, s);
  return bf ? launch<__nv_bfloat16, 128, 16>(*d, p, scratch, s) : launch<__half, 128, 16>(*d, p, scratch, s);
}
