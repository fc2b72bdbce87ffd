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
#include "paged_attn.cuh"

extern "C" int* ftk_status_word(void);

namespace ftk {

constexpr int PA_WARPS = 4, PA_TILE = 16 * PA_WARPS;      // of a CTA that shares its SM
// Tiles of 64 tokens, by the width of the table, up to which a head is left whole: a second launch and the join cost 3 - 4 us, so few heads
// are cut late, and heads for all SMs fill the time among themselves.  Whole and cut (us) with all positions in use, an SM for each head:
// 12 heads of 64, 16 tiles 8.1 and 8.6, 32 tiles 13.7 and 9.2; 32 heads of 128, up to 17 tiles 13.1 and 10.7; 128 heads of 128, up to 17
// 13.7 and 16.4, up to 33 22.4 and 25.0; with several heads per SM, 256 of 128, up to 17 21.7 and 26.4, up to 33 38.0 and 36.9.  A straight
// line below these borders: for a dozen heads it cuts from 12 tiles on where 17 would do, and the width stands for lengths that only the
// device knows, so few tokens under a wide table are cut too (12 heads of 64, 301 tokens: 4.8 us under 5 tiles, 8.9 under 16).
__host__ inline long long pa_whole(long long heads, long long sms) { return heads <= sms ? 9 + 28 * heads / sms : 20; }

// fp16 has five bits of exponent: probabilities are carried times 2^15, so that what underflows is 2^-39 of the largest.
template <typename T> struct PaShift { static constexpr int value = 0; };
template <> struct PaShift<__half> { static constexpr int value = 15; };

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
    Piece piece;
    p = first_place<TILE>((int)d.B, heads, length, piece);
    total = piece.total, per = piece.per, first_unit = piece.first, left = piece.left;
    if (!a.by_head && threadIdx.x == 0) a.header[(long long)blockIdx.x * PA_HEADER] = -1;
    if (left <= 0) return;
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
    float* part = SPLIT ? a.parts + ((long long)blockIdx.x * 2 + parts) * PA_PART<ROWS, HD> : nullptr;
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
  return launch_join<T, HD, ROWS, PaShift<T>::value>(a, p.heads, p.ctas, p.headers, s);
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
