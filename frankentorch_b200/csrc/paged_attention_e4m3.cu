// Attention of one new token per sequence over a paged key-value cache held in 8 bits (e4m3) with a scale per block of rows and head.
//
// Mathematics.  With ks and vs the scales of token t's key and value, x_t = scale ks_t (q . k_t), o = sum_t softmax_t(x) vs_t v_t and
// lse = log sum_t exp(x_t).  Terms of the output have size 2^(x_t) vs_t, terms of the sum 2^(x_t), so each has a reference of its own, a whole
// number of base 2: the accumulators are sum_t 2^(y_t - m) (vs_t / 2^e_t) v_t with e_t the power of two in vs_t, y_t = x_t + e_t and m the largest
// y_t, rounded up; l = sum_t 2^(x_t - n) with n the largest x_t.  One reference for both takes tokens out of the sum that weigh as much as
// others, where scales are 2^126 apart.  Whole numbers leave x_t - (m - e_t) as exact as x_t.  As long as a head's scales are within 2^40 of
// its first ones, n = m - e of those serves, and a weight is its term of l times a power of two and the scale; from the first tile on
// where they are not, n is each lane's own and weights have an exponential of their own (32 heads over 8 of 128, 16 x 2048 tokens: 20.0 us that
// way throughout, 18.9 this way); with one head to a head of the cache, a token per lane, that costs nothing and is always so.  Parts are
// given on as m and l 2^(n - m), which |n - m| <= 129 keeps in fp32; where parts meet, sums are compared by their own powers of two.  The
// list of tiles, the pieces, the rings and the join are paged_attention.cu's.
//
// What is lost: weights are held in two halves of fp16, the largest as 2^13 or more, each to 2^-25: what adds less than 2^-38 of the largest weight
// (value scale and all) times 448 to an element of the output does not count.
//
// What bounds it: every key and value is read once, in 8 bits; the copy bandwidth, with twice the arithmetic per byte of a 16-bit cache.
// 128 sequences of 700 to 4096, 16 heads of 128: 211 - 230 us in calls one after another, by the power that is left, 5.7 - 6.2 TB/s, and 203 - 205
// in a captured burst of them (16-bit cache 388 - 410); 32 of up to 2048 31.8 (51); two of up to 65537, 32 heads over 4, 36.2 (51); one of 301
// tokens, 12 heads of 64, 5.4.  A warp's 32 tokens of 128 bytes are 620 instructions, of which 64 convert; the SMs issue in 45 - 47 % of the
// cycles, so few heads are bound by the first tiles' way and by the join.
//
// A warp takes 32 tokens of a tile at a time.  fp16 holds every e4m3 value, so keys and values go into the matrix instructions as they
// are, converted in registers, and the scales are applied to scores and probabilities, which are few.  The queries are in fp16 too, a
// row at a time times the power of two, up to 2^127, that brings its largest element to 2^14 .. 2^15: what that loses is below 2^-39 of it.
// Matrix products of the 8-bit values as they are, with queries and probabilities in several parts, took 284 us where these took 276.
//
// Scores are formed with the tokens as rows and the heads as columns: of 16 x 8 results none is wasted for up to eight heads, where heads as
// rows would fill half.  The elements of a product's inner dimension may come in any order that both operands share, so a thread's four
// neighbouring bytes of a key are two operand registers as they are.  For the output the heads are rows; a register's transposition in the warp
// turns the probabilities, and of a value column one byte permutation brings the bytes of two tokens together, even columns in one
// product and odd ones in another.  Probabilities times scales are split into two halves of fp16, carried times 2^14: 22 bits of them count.
// With one head to a head of the cache three of four lanes would hold nothing, so its scores go through shared memory to a token per
// lane, and the two halves of its probabilities are two rows of one product: 118 us and 123, 128 sequences of 16 heads of 64.
//
// Two warps and six CTAs to an SM, two tiles in flight: 218 us; four warps and three CTAs 231 (heads of 128, the largest batch above).
#include "e4m3.cuh"
#include "paged_attn.cuh"

extern "C" int* ftk_status_word(void);

namespace ftk {

constexpr int A8_WARPS = 2, A8_TOKENS = 32;      // of a CTA that shares its SM; tokens that a warp takes at a time
constexpr float A8_NONE = -3.402823466e38f;      // the reference where there is no token yet
// Scales within 2^40 of one another: x - (m - unit) is 40 at most, and what it loses to fp32 below 2^-126 is below 2^-46 of l and of the accumulator
constexpr float A8_NEAR = 40.f;
// Tiles of 64 tokens, by the width of the table, up to which a head is left whole: a second launch and the join cost 4 - 6 us.  Whole and cut
// (us), all positions in use, 64 to a tile: 12 heads of 64, 16 tiles 7.5 and 10.1, 24 tiles 9.5 and 10.3, 32 tiles 11.4 and 10.2; 32 heads of
// 128, 16 tiles 9.9 and 11.4, 32 tiles 15.9 and 13.1; 128 heads of 128, 16 tiles 10.7 and 16.3, 40 tiles 19.7 and 24.2.  With several heads
// per SM, which fill the time among themselves: 256 of 128, 16 tiles 22.0 and 21.8, 32 tiles 39.4 and 32.0; 768 of 64, 16 tiles 30.5 and
// 33.1, 32 tiles 55.4 and 49.4; 1024 of 128, 16 tiles 61.6 and 54.4, 24 tiles 87.6 and 72.1.  A straight line below these borders up to a
// head per SM, and one border above.
__host__ inline long long a8_whole(long long heads, long long sms) { return heads <= sms ? 18 + 32 * heads / sms : 16; }

// ROWS query heads of a head of the cache: 1, up to 8 or up to 16
template <int ROWS, int HD, int W> struct A8Smem {
  static constexpr bool ONE = ROWS == 1, OWN = W <= A8_WARPS;      // OWN: what is joined in memory of its own, or in the rings of a head that is through
  static constexpr int CTAS = !OWN ? 1 : (HD == 64 ? (ROWS == 16 ? 6 : 8) : (ROWS == 16 ? 4 : 6));
  static constexpr int DATA = A8_TOKENS * HD * 2, STAGE = DATA + A8_TOKENS * 8;      // keys, values, scales
  static constexpr int STAGES = OWN ? 2 : 3;
  static constexpr int WEIGHT_ROW = 80, TURN = ONE ? A8_TOKENS * 4 + 16 * WEIGHT_ROW : A8_TOKENS * 16;      // of a warp, for what goes from lane to lane
  static constexpr int RING = STAGES * STAGE;
  static constexpr int COLS = ONE ? HD : (HD == 128 ? 32 : 64);      // columns of the accumulators of all warps that are joined at a time
  static constexpr int MERGE = W * ROWS * COLS * 4;
  static constexpr int BYTES = W * (RING + TURN) + (OWN ? MERGE : 0) + (3 * W + 1) * ROWS * 4 + W * STAGES * 4;
  static_assert(OWN || MERGE <= W * RING, "the accumulators fit the rings");
  static_assert(STAGE % 128 == 0, "chunks of a row are exchanged by address bits");
  static_assert(CTAS * (BYTES + 1024) <= 228 * 1024 && BYTES <= 227 * 1024, "the CTAs of an SM share its memory");
};
template <int ROWS, int HD> constexpr int A8_ALONE = HD == 64 && ROWS <= 8 ? 16 : 8;

__device__ __forceinline__ uint32_t transposed(uint32_t pair) {      // of 8 x 8 values of 16 bits, two of row lane / 4 in each lane
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(pair));
  return r;
}
constexpr int A8_SHIFT = 14;      // weights are carried times 2^14
__device__ __forceinline__ float power(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }      // 2^e of -126 to 127
// v / 2^e, times 2^14
__device__ __forceinline__ float unscaled(float v, float e) { return v * power(A8_SHIFT - (int)e); }
__device__ __forceinline__ float max_of(float x) {      // over the warp; NaN is not counted
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(there ? 4 : 0) : "memory");
}

// What the loads of a tile take, in 32 bits: with 64 bits of everything and a division for the head they were 100 instructions more
struct Strides8 {
  unsigned k_page, k_head, k_row, v_page, v_head, v_row;      // of pages, in 16 bytes
  unsigned ks_page, ks_head, vs_page, vs_head;                // of scales
  unsigned n_pages, cols, table_row;
  int page_shift, block_shift;
};

template <typename T, int HD, int ROWS, bool SPLIT, int W>
__global__ void __launch_bounds__(W * 32, A8Smem<ROWS, HD, W>::CTAS) paged_attn_e4m3_kernel(const __grid_constant__ PagedAttn a, const __grid_constant__ Strides8 by, int* status) {
  typedef A8Smem<ROWS, HD, W> SM;
  static_assert(!SPLIT || SM::OWN, "a piece goes on while the parts are joined");
  constexpr int N = A8_TOKENS, TILE = N * W;
  constexpr int STAGES = SM::STAGES, STAGE = SM::STAGE, CH = HD / 16, NT = HD / 8;      // CH: 16-byte chunks of a row
  constexpr int RR = ROWS == 16 ? 2 : 1;      // eights of query heads
  constexpr bool ONE = SM::ONE;
  extern __shared__ __align__(256) unsigned char smem[];
  const FtkPagedAttnDesc& d = a.d;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, heads = (int)d.Hkv * a.subs;
  unsigned char* ring = smem + warp * SM::RING;
  unsigned char* turn = smem + W * SM::RING + warp * SM::TURN;      // ONE: scores, then 16 rows of weights; else the scales of each token
  float* merge = reinterpret_cast<float*>(smem + (SM::OWN ? W * (SM::RING + SM::TURN) : 0));
  // [3][warps][ROWS]: m, then the sum as own_power has it; [ROWS]: what the output is multiplied by
  float* stat = reinterpret_cast<float*>(smem + W * (SM::RING + SM::TURN) + (SM::OWN ? SM::MERGE : 0));
  unsigned* there = reinterpret_cast<unsigned*>(stat + (3 * W + 1) * ROWS) + warp * STAGES;
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
  const bool one_page = table.shift >= 5;
  const int tok_of = warp * N + (one_page ? 0 : lane);      // of a tile: the token whose page this lane looks up

  // ---- this CTA's piece of the list
  Place p;
  Piece piece = {0, 0, 0, 0};
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
    piece.left = p.tiles;
  } else {
    p = first_place<TILE>((int)d.B, heads, length, piece);
    if (!a.by_head && threadIdx.x == 0) a.header[(long long)blockIdx.x * PA_HEADER] = -1;
    if (piece.left <= 0) return;
  }
  int left = piece.left;

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
  // Pages of the next tiles.  A page of 32 rows or more holds all of a warp's part of a tile; of smaller ones lane j has token j's.
  int page_of[AHEAD] = {};
  const auto look = [&]() {
    int page = -1;
    if (to_look > 0) {
      const int tok = g.t * TILE + tok_of;
      if (tok < g.n) {
        const unsigned col = (unsigned)tok >> by.page_shift;
        page = col < by.cols ? d.table[(unsigned long long)(unsigned)g.b * by.table_row + col] : -1;
        if ((unsigned)page >= by.n_pages) page = -1, ft_index_ok(-1, 1, status);
      }
      advance(g, to_look);
    }
    return page;
  };
  const uint32_t ring_s = smem_u32(ring);
  // Chunk c of row r is at c ^ swizzle(r), so that eight rows' chunks of a matrix are in different banks
  const auto swizzle = [](int r) { return HD == 128 ? r & 7 : (r >> 1) & 3; };
  const int lrow = lane / CH, lchunk = lane % CH;
  constexpr int RSTEP = 32 / CH, COPIES = N / RSTEP;      // rows of a copy of the warp, copies of 32 rows
  const uint32_t lane_at = lrow * HD, lane_sw = lchunk << 4;
  const bool packed = by.k_row == HD / 16 && by.v_row == HD / 16;
  const auto offset = [](unsigned page, unsigned s_page, unsigned head, unsigned s_head, unsigned row, unsigned s_row) {
    return (unsigned long long)page * s_page + (unsigned long long)head * s_head + (unsigned long long)row * s_row;
  };
  const auto load = [&](int stage) {
    const int pages = page_of[0];
#pragma unroll
    for (int i = 0; i + 1 < AHEAD; ++i) page_of[i] = page_of[i + 1];
    page_of[AHEAD - 1] = look();
    if (to_load > 0) {
      const int tok0 = f.t * TILE + warp * N;
      const unsigned f_kv = a.subs == 1 ? f.h : f.h / a.subs;      // head of the cache
      const uint4 *const keys = (const uint4*)d.k_pages + lchunk, *const values = (const uint4*)d.v_pages + lchunk;
      const unsigned in_page = (1u << by.page_shift) - 1;
      const uint32_t dst = ring_s + stage * STAGE + lane_at, sdst = ring_s + stage * STAGE + SM::DATA + lane * 4;
      unsigned ok, own_row;             // this lane's own token: its row in its page, its page
      int own_page;
      if (one_page) {
        const int n = pages < 0 ? 0 : min(N, f.n - tok0);      // rows that are there
        const unsigned page = pages < 0 ? 0u : (unsigned)pages, in = (unsigned)tok0 & in_page;
        ok = n >= N ? 0xffffffffu : (1u << max(n, 0)) - 1;
        const uint4* k = keys + offset(page, by.k_page, f_kv, by.k_head, in + lrow, by.k_row);
        const uint4* v = values + offset(page, by.v_page, f_kv, by.v_head, in + lrow, by.v_row);
        if (packed && n >= N) {         // one run of bytes, all of it there
#pragma unroll
          for (int c = 0; c < COPIES; ++c) {
            const uint32_t at = dst + c * RSTEP * HD + (lane_sw ^ (swizzle(c * RSTEP + lrow) << 4));
            copy16(at, k + c * 32, true);
            copy16(at + N * HD, v + c * 32, true);
          }
        } else {
#pragma unroll
          for (int c = 0; c < COPIES; ++c) {
            const bool t = c * RSTEP + lrow < n;
            const uint32_t at = dst + c * RSTEP * HD + (lane_sw ^ (swizzle(c * RSTEP + lrow) << 4));
            copy16(at, t ? k + (unsigned long long)(c * RSTEP) * by.k_row : keys, t);
            copy16(at + N * HD, t ? v + (unsigned long long)(c * RSTEP) * by.v_row : values, t);
          }
        }
        own_page = lane < n ? (int)page : -1, own_row = in + lane;
      } else {
        ok = __ballot_sync(0xffffffffu, pages >= 0);
#pragma unroll
        for (int c = 0; c < COPIES; ++c) {
          const int row = c * RSTEP + lrow, page = __shfl_sync(0xffffffffu, pages, row);
          const unsigned in = (unsigned)(tok0 + row) & in_page;
          const bool t = page >= 0;
          const uint32_t at = dst + c * RSTEP * HD + (lane_sw ^ (swizzle(row) << 4));
          copy16(at, t ? keys + offset(page, by.k_page, f_kv, by.k_head, in, by.k_row) : keys, t);
          copy16(at + N * HD, t ? values + offset(page, by.v_page, f_kv, by.v_head, in, by.v_row) : values, t);
        }
        own_page = pages, own_row = (unsigned)(tok0 + lane) & in_page;
      }
      const bool t = own_page >= 0;
      copy4(sdst, t ? d.k_scales + offset(own_page, by.ks_page, f_kv, by.ks_head, own_row >> by.block_shift, 1) : d.k_scales, t);
      copy4(sdst + N * 4, t ? d.v_scales + offset(own_page, by.vs_page, f_kv, by.vs_head, own_row >> by.block_shift, 1) : d.v_scales, t);
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
  uint32_t q[CH][2 * RR];               // of chunk c: elements 2 c0 .. + 3 of head r0, then of head r0 + 8
  // of heads c0, c0 + 1, c0 + 8, c0 + 9; ONE: [0].  m of the accumulators, of all lanes; n and l of this lane's tokens
  float acc[NT][4], m[2 * RR], n[2 * RR], l[2 * RR], sc[2 * RR];
  float k_by;                           // what keys' scales are multiplied by
  float unit;                           // power of two of the first tokens' value scales
  bool near;                            // all so far are within A8_NEAR powers of it: then n = m - unit, and a weight is taken from its term of l
  const int r0 = lane >> 2, c0 = (lane & 3) * 2;
  const auto begin = [&]() {            // queries of the head at `p`; rows beyond the group are zero
    const int first = row0(p.h), rows = rows_of(p.h);
    int e[RR];
#pragma unroll
    for (int r = 0; r < RR; ++r) {
      const int row = r * 8 + r0;
      const T* base = (const T*)d.q + p.b * d.q_bs + (first + row) * d.q_hs + c0 * 2;
      uint2 u[CH];
      float most = 0.f;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        u[c] = row < rows ? *reinterpret_cast<const uint2*>(base + c * 16) : make_uint2(0, 0);
        const float2 x = Half16<T>::up(u[c].x), y = Half16<T>::up(u[c].y);
        most = fmaxf(fmaxf(fmaxf(most, fabsf(x.x)), fmaxf(fabsf(x.y), fabsf(y.x))), fabsf(y.y));
      }
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
      e[r] = min(max((int)(__float_as_uint(most) >> 23) - 127, -113), 127);
      const float by = power(14 - e[r]);
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const float2 x = Half16<T>::up(u[c].x), y = Half16<T>::up(u[c].y);
        q[c][2 * r] = Half16<__half>::down(x.x * by, x.y * by), q[c][2 * r + 1] = Half16<__half>::down(y.x * by, y.y * by);
      }
    }
    // What a score is multiplied by beside its key's scale, scale log2(e) 2^(e - 14): the power of two of the row that has the largest goes
    // to the keys' scales, so that neither of the two is beyond fp32 where their product is not
    const float factor = (float)d.scale * LOG2E;
    const int of_factor = min(max((int)(__float_as_uint(factor) >> 23 & 255) - 127, -126), 126);
    if (ONE) e[0] = __shfl_sync(0xffffffffu, e[0], 0);
    const int largest = ONE ? e[0] : __reduce_max_sync(0xffffffffu, max(e[0], e[RR - 1]));
    const int with_key = min(max(largest - 14 + of_factor, -126), 127);
    k_by = power(with_key);
#pragma unroll
    for (int r = 0; r < RR; ++r) {
      const int rest = e[r] - 14 + of_factor - with_key;      // -240 to 112: rows may be that far apart
      const float own = factor * power(-of_factor) * power(rest >> 1) * power(rest - (rest >> 1));
      sc[2 * r] = ONE ? own : __shfl_sync(0xffffffffu, own, c0 * 4);
      if (!ONE) sc[2 * r + 1] = __shfl_sync(0xffffffffu, own, c0 * 4 + 4);
    }
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
#pragma unroll
    for (int r = 0; r < 2 * RR; ++r) m[r] = n[r] = A8_NONE, l[r] = 0.f;
    unit = A8_NONE, near = true;
  };
  bool begun = p.t == 0;                // the piece has the beginning of the head at `p`
  int parts = 0;
  begin();
  // this lane's row for ldmatrix: of four groups of eight tokens at one chunk
  const uint32_t l_at = lane * HD + (swizzle(lane) << 4);
  // ONE: the row of weights that this lane addresses, of 16 rows at the first eight tokens and 16 at the next; all but two rows stay 0
  const uint32_t weights_at = smem_u32(turn) + N * 4 + (lane & 15) * SM::WEIGHT_ROW + (lane >> 4) * 16;
  if (ONE) {
    for (int i = lane; i < SM::TURN / 4; i += 32) reinterpret_cast<uint32_t*>(turn)[i] = 0;
  }
  int stage = 0;
  for (bool more = true; more; more = left > 0) {
    if (left > 0) {
      copy_wait<STAGES - 2>();
      __syncwarp();
      const uint32_t ks = ring_s + stage * STAGE + l_at, vs = ks + N * HD;
      const unsigned ok = there[stage];
      load(stage == 0 ? STAGES - 1 : stage - 1);      // the stage that the tile before left: its reads are behind the warp's barrier
      const float* scales = reinterpret_cast<const float*>(ring + stage * STAGE + SM::DATA);      // keys', values'
      const float k_scale = scales[lane] * k_by, v_scale = scales[N + lane], v_exp = (float)max((int)(__float_as_uint(v_scale) >> 23 & 255) - 127, -100);
      // Scores with the tokens as rows: s[2 r + t] of tokens 16 t and on, the r-th eight heads
      float s[2 * RR][4] = {};
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        uint32_t b[4], lower[4], upper[4];
        ldm4(ks ^ (c << 4), b);
#pragma unroll
        for (int j = 0; j < 4; ++j) lower[j] = e4m3_up(b[j] & 0xffffu), upper[j] = e4m3_up(b[j] >> 16);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint32_t k[4] = {lower[2 * u], lower[2 * u + 1], upper[2 * u], upper[2 * u + 1]};
#pragma unroll
          for (int r = 0; r < RR; ++r) mma16<__half>(s[2 * r + u], k, q[c][2 * r], q[c][2 * r + 1]);
        }
      }
      uint32_t hi[2][4] = {}, lo[2][4] = {};      // weights of two steps of 16 tokens
      if constexpr (ONE) {
        // the one head's scores, in every fourth lane, go to a token per lane, their weights to the rows 0 (hi) and 8 (lo) of an operand
        float* score = reinterpret_cast<float*>(turn);
        unsigned short* weight = reinterpret_cast<unsigned short*>(turn + N * 4);
        if (c0 == 0) {
#pragma unroll
          for (int u = 0; u < 2; ++u) score[16 * u + r0] = s[u][0], score[16 * u + 8 + r0] = s[u][2];
        }
        __syncwarp();
        const float x = ok >> lane & 1u ? score[lane] * (k_scale * sc[0]) : -INFINITY;
        const float top = fmaxf(m[0], ceilf(max_of(x + v_exp))), own = fmaxf(n[0], ceilf(x));
        const float w = exp2_of(x - (top - v_exp)) * unscaled(v_scale, v_exp);
        if (top != m[0]) {
          const float grow = exp2_of(m[0] - top);
#pragma unroll
          for (int i = 0; i < NT; ++i) acc[i][0] *= grow, acc[i][1] *= grow, acc[i][2] *= grow, acc[i][3] *= grow;
          m[0] = top;
        }
        l[0] = fmaf(l[0], exp2_of(n[0] - own), exp2_of(x - own));
        n[0] = own;
        const __half h = __float2half_rn(w);
        weight[lane] = __half_as_ushort(h);
        weight[8 * (SM::WEIGHT_ROW / 2) + lane] = __half_as_ushort(__float2half_rn(w - __half2float(h)));
        __syncwarp();
        ldm4(weights_at, hi[0]);
        ldm4(weights_at + 32, hi[1]);
      } else {
        // masked scores of heads c0, c0 + 1 at tokens r0, r0 + 8 .., and the larger references of the head's tokens and what was there
        const bool own_there = ok >> lane & 1u;
        if (unit == A8_NONE) unit = max_of(own_there ? v_exp : A8_NONE);
        near = near && !__any_sync(0xffffffffu, own_there && fabsf(v_exp - unit) > A8_NEAR);
        reinterpret_cast<float4*>(turn)[lane] = make_float4(k_scale, v_exp, own_there ? unscaled(v_scale, near ? unit : v_exp) : 0.f, 0.f);
        __syncwarp();
        float grow[2 * RR], v14[4], v_of[4];
        bool moved = false;
#pragma unroll
        for (int r = 0; r < RR; ++r) {
          float x[4][2], top[2] = {m[2 * r], m[2 * r + 1]};
#pragma unroll
          for (int i = 0; i < 4; ++i) {        // token 8 i + r0: key's scale, exponent of the value's, the rest of that
            const float4 f = reinterpret_cast<const float4*>(turn)[8 * i + r0];
            v_of[i] = f.y, v14[i] = f.z;
            const bool there = ok >> (8 * i + r0) & 1u;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              x[i][e] = there ? s[2 * r + (i >> 1)][(i & 1) * 2 + e] * (f.x * sc[2 * r + e]) : -INFINITY;
              top[e] = fmaxf(top[e], x[i][e] + f.y);
            }
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], o));
            top[e] = ceilf(top[e]);
            moved |= top[e] != m[2 * r + e];
            grow[2 * r + e] = exp2_of(m[2 * r + e] - top[e]);
            m[2 * r + e] = top[e];
          }
          if (near) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float own = top[e] == A8_NONE ? A8_NONE : top[e] - unit;      // (a tile may have no token: pages that are none)
              l[2 * r + e] *= grow[2 * r + e];
              n[2 * r + e] = own;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                x[i][e] = exp2_of(x[i][e] - own);
                l[2 * r + e] += x[i][e];
              }
            }
          } else {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float own = fmaxf(n[2 * r + e], ceilf(fmaxf(fmaxf(x[0][e], x[1][e]), fmaxf(x[2][e], x[3][e]))));
              l[2 * r + e] *= exp2_of(n[2 * r + e] - own);
              n[2 * r + e] = own;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                l[2 * r + e] += exp2_of(x[i][e] - own);
                x[i][e] = exp2_of(x[i][e] - (top[e] - v_of[i]));
              }
            }
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {        // to rows of heads: step i / 2, its first or second eight tokens
            const float w0 = x[i][0] * v14[i], w1 = x[i][1] * v14[i];
            const uint32_t h = Half16<__half>::down(w0, w1);
            const float2 u = Half16<__half>::up(h);
            hi[i >> 1][(i & 1) * 2 + r] = transposed(h);
            lo[i >> 1][(i & 1) * 2 + r] = transposed(Half16<__half>::down(w0 - u.x, w1 - u.y));
          }
        }
        if (__any_sync(0xffffffffu, moved)) {
          float g[2];                          // of the accumulators' rows r0 and r0 + 8
#pragma unroll
          for (int r = 0; r < RR; ++r) {
            const float even = __shfl_sync(0xffffffffu, grow[2 * r], r0 >> 1), odd = __shfl_sync(0xffffffffu, grow[2 * r + 1], r0 >> 1);
            g[r] = r0 & 1 ? odd : even;
          }
          if (RR == 1) g[1] = g[0];
#pragma unroll
          for (int i = 0; i < NT; ++i) acc[i][0] *= g[0], acc[i][1] *= g[0], acc[i][2] *= g[1], acc[i][3] *= g[1];
        }
        if (RR == 1) {
#pragma unroll
          for (int u = 0; u < 2; ++u) hi[u][1] = lo[u][0], hi[u][3] = lo[u][2];
        }
      }
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        uint32_t b[4];
        ldm4t(vs ^ (c << 4), b);        // of tokens 8 i + c0, + 1: two columns of each
#pragma unroll
        for (int i = 0; i < 4; ++i) b[i] = __byte_perm(b[i], 0, 0x3120);      // the first column's, the second's
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const uint32_t e0 = e4m3_up(b[2 * t] & 0xffffu), e1 = e4m3_up(b[2 * t + 1] & 0xffffu), o0 = e4m3_up(b[2 * t] >> 16), o1 = e4m3_up(b[2 * t + 1] >> 16);
          mma16<__half>(acc[2 * c], hi[t], e0, e1);
          mma16<__half>(acc[2 * c + 1], hi[t], o0, o1);
          if (ROWS == 16) {
            mma16<__half>(acc[2 * c], lo[t], e0, e1);
            mma16<__half>(acc[2 * c + 1], lo[t], o0, o1);
          }
        }
      }
      stage = stage + 1 == STAGES ? 0 : stage + 1;
      --left;
      ++p.t;
    }
    if (left > 0 && p.t < p.tiles) continue;

    // ---- the end of a head, or of the piece: the warps' parts become one
#pragma unroll
    for (int r = 0; r < (ONE ? 1 : 2 * RR); ++r) {
      float most = n[r];
      if (ONE) most = max_of(most);
      if (!ONE && !near) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
      }
      if (ONE || !near) l[r] *= exp2_of(n[r] - most);
#pragma unroll
      for (int o = ONE ? 1 : 4; o < 32; o <<= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], o);
      if (r0 == 0 && (!ONE || c0 == 0)) {
        const int head = ONE ? 0 : (r >> 1) * 8 + c0 + (r & 1);
        stat[warp * ROWS + head] = m[r];
        const float2 x = own_power(most, l[r]);
        stat[(W + warp) * ROWS + head] = x.x;
        stat[(2 * W + warp) * ROWS + head] = x.y;
      }
    }
    const bool whole = begun && p.t == p.tiles;
    const int first = row0(p.h), rows = rows_of(p.h);
    float* part = SPLIT ? a.parts + ((long long)blockIdx.x * 2 + parts) * PA_PART<ROWS, HD> : nullptr;
    __syncthreads();
    float scale[RR];                    // of the warp's part: to the maximum of all, without the 2^14
#pragma unroll
    for (int r = 0; r < RR; ++r) {
      const int head = ONE ? 0 : r * 8 + r0;
      const float own = stat[warp * ROWS + head];
      float top = own;
#pragma unroll
      for (int w = 0; w < W; ++w) top = fmaxf(top, stat[w * ROWS + head]);
      scale[r] = exp2_of(own - top) * (1.f / (1 << A8_SHIFT));
      if (warp == 0 && c0 == 0 && head < rows && (!ONE || r0 == 0)) {      // the sum of all warps, and where it belongs
        float most = A8_NONE, sum = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) most = fmaxf(most, stat[(W + w) * ROWS + head]);
#pragma unroll
        for (int w = 0; w < W; ++w) sum += exp2_of(stat[(W + w) * ROWS + head] - most) * stat[(2 * W + w) * ROWS + head];
        if (!SPLIT || whole) {
          stat[3 * W * ROWS + head] = sum == 0.f ? 0.f : exp2f(top - most) / sum;
          d.lse[(long long)p.b * d.Hq + first + head] = sum == 0.f ? -INFINITY : (most + log2f(sum)) * LN2;
        } else {
          part[ROWS * HD + head] = top, part[ROWS * (HD + 1) + head] = sum * exp2f(most - top);
        }
      }
    }
    // all columns of a few rows at once, else some of all rows
    const int cols = rows * HD <= ROWS * SM::COLS ? HD : SM::COLS;
    for (int from = 0; from < HD; from += cols) {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        if (c * 16 < from || c * 16 >= from + cols) continue;
        float* to = merge + (warp * rows + r0) * cols + c * 16 - from + c0 * 2;
        const float *x = acc[2 * c], *y = acc[2 * c + 1];      // even and odd columns
        if (ROWS == 16) {
          const float s1 = scale[RR - 1];
          if (r0 < rows) *reinterpret_cast<float4*>(to) = make_float4(x[0] * scale[0], y[0] * scale[0], x[1] * scale[0], y[1] * scale[0]);
          if (r0 + 8 < rows) *reinterpret_cast<float4*>(to + 8 * cols) = make_float4(x[2] * s1, y[2] * s1, x[3] * s1, y[3] * s1);
        } else if (r0 < rows) {
          *reinterpret_cast<float4*>(to) = make_float4((x[0] + x[2]) * scale[0], (y[0] + y[2]) * scale[0], (x[1] + x[3]) * scale[0], (y[1] + y[3]) * scale[0]);
        }
      }
      __syncthreads();
      for (int i = threadIdx.x; i < rows * cols / 2; i += W * 32) {
        const int row = i / (cols / 2), in = (i % (cols / 2)) * 2, col = from + in;
        float2 v = make_float2(0.f, 0.f);
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const float2 x = *reinterpret_cast<const float2*>(merge + (w * rows + row) * cols + in);
          v.x += x.x, v.y += x.y;
        }
        if (!SPLIT || whole) {
          const float by = stat[3 * W * ROWS + row];
          T* o = (T*)d.o + p.b * d.o_bs + (first + row) * d.o_hs + col;
          *reinterpret_cast<uint32_t*>(o) = Half16<T>::down(by == 0.f ? 0.f : v.x * by, by == 0.f ? 0.f : v.y * by);
        } else {
          *reinterpret_cast<float2*>(part + row * HD + col) = v;
        }
      }
      __syncthreads();
    }
    if (!SPLIT) return;
    // the part that has the beginning of its head says who has the rest, up to the CTA of the head's last tile
    if (begun && threadIdx.x == 0 && (a.by_head || !whole)) {
      const long long behind = piece.first + min(piece.per, piece.total - piece.first);
      int* h = a.header + (a.by_head ? (long long)p.b * heads + p.h : (long long)blockIdx.x) * PA_HEADER;
      h[0] = whole ? -1 : (int)blockIdx.x;
      h[1] = p.b, h[2] = p.h, h[3] = parts, h[4] = (int)((behind + (p.tiles - p.t) - 1) / piece.per);
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

struct Plan8 {
  int subs, sub_heads, rows;
  bool split, alone, wide_join;    // heads cut into pieces; a CTA per SM, for few heads; 1024 threads for a row of the join
  long long ctas, heads, headers, bytes;      // heads: of all sequences, a part of a group counting as one
};
template <int ROWS, int HD> constexpr int A8_CTAS = A8Smem<ROWS, HD, A8_WARPS>::CTAS;
static Plan8 plan_of(const FtkPagedAttnDesc& d) {
  Plan8 p;
  const long long group = d.Hq / d.Hkv;
  p.subs = (int)((group + 15) / 16);
  p.sub_heads = (int)((group + p.subs - 1) / p.subs);
  p.rows = p.sub_heads == 1 ? 1 : (p.sub_heads <= 8 ? 8 : 16);
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  p.ctas = p.heads = d.B * d.Hkv * p.subs;
  p.headers = p.bytes = 0;
  const long long tiles = ((d.table_cols << d.page_shift) + 63) / 64;
  p.alone = p.heads <= sms;
  p.split = tiles > a8_whole(p.heads, sms);
  // Few heads have up to a hundred parts each, which 1024 threads join faster than 256, as long as the rows, a block each, have an SM each (us):
  // 8 heads of 8 queries, 2 x 65537, 36.1 and 38.7; 16 of 8 31.3 and 32.2; 32 of 1 22.3 and 22.1; 32 of 8 50.1 and 46.7; 32 of 16 72.0 and 62.7.
  // Many heads have a part or two: 464 heads 50.8 and 40.6, 48 42.6 and 42.2
  p.wide_join = p.heads <= 32 && p.heads * p.sub_heads <= sms;
  if (p.split) {
    p.ctas = (d.hd == 64 ? (p.rows == 1 ? A8_CTAS<1, 64> : p.rows == 8 ? A8_CTAS<8, 64> : A8_CTAS<16, 64>)
                         : (p.rows == 1 ? A8_CTAS<1, 128> : p.rows == 8 ? A8_CTAS<8, 128> : A8_CTAS<16, 128>)) * (long long)sms;
    p.headers = p.heads < p.ctas ? p.heads : p.ctas;
    p.bytes = p.headers * PA_HEADER * 4 + p.ctas * 2 * (p.rows * (d.hd + 2) + 2) * 4;
  }
  return p;
}

template <typename T, int HD, int ROWS>
static int launch(const FtkPagedAttnDesc& d, const Plan8& p, void* scratch, cudaStream_t s) {
  PagedAttn a = {d, (int)(d.Hq / d.Hkv), p.subs, p.sub_heads, p.heads < p.ctas, (int*)scratch, nullptr};
  a.parts = (float*)((char*)scratch + p.headers * PA_HEADER * 4);
  const Strides8 by = {(unsigned)(d.kp_ps >> 4), (unsigned)(d.kp_hs >> 4), (unsigned)(d.kp_rs >> 4), (unsigned)(d.vp_ps >> 4), (unsigned)(d.vp_hs >> 4),
                       (unsigned)(d.vp_rs >> 4), (unsigned)d.ks_ps, (unsigned)d.ks_hs, (unsigned)d.vs_ps, (unsigned)d.vs_hs, (unsigned)d.n_pages,
                       (unsigned)d.table_cols, (unsigned)d.table_stride, (int)d.page_shift, (int)d.block_shift};
  int* status = ftk_status_word();
  if (!p.split && p.alone) {
    constexpr int W = A8_ALONE<ROWS, HD>, bytes = A8Smem<ROWS, HD, W>::BYTES;
    const auto kernel = paged_attn_e4m3_kernel<T, HD, ROWS, false, W>;
    const int rc = (int)cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    return rc ? rc : launch_pdl(kernel, dim3((unsigned)p.ctas), dim3(W * 32), bytes, s, a, by, status);
  }
  constexpr int bytes = A8Smem<ROWS, HD, A8_WARPS>::BYTES;
  const auto whole = paged_attn_e4m3_kernel<T, HD, ROWS, false, A8_WARPS>, split = paged_attn_e4m3_kernel<T, HD, ROWS, true, A8_WARPS>;
  const auto kernel = p.split ? split : whole;
  int rc = (int)cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (rc) return rc;
  rc = launch_pdl(kernel, dim3((unsigned)p.ctas), dim3(A8_WARPS * 32), bytes, s, a, by, status);
  if (rc || !p.split) return rc;
  return p.wide_join ? launch_join<T, HD, ROWS, 0, true, 1024>(a, p.heads, p.ctas, p.headers, s) : launch_join<T, HD, ROWS, 0, true>(a, p.heads, p.ctas, p.headers, s);
}

// Strides of 64 GB and more are refused: offsets are 32 bits times 16 bytes (4 of scales and of the table) of each kind, added up in 64
static bool wide(const FtkPagedAttnDesc* d) {
  const long long most = 0xffffffffll;
  for (long long s : {d->kp_ps, d->kp_hs, d->kp_rs, d->vp_ps, d->vp_hs, d->vp_rs})
    if (s < 0 || s >> 4 > most) return true;
  for (long long s : {d->ks_ps, d->ks_hs, d->vs_ps, d->vs_hs, d->table_stride})
    if (s < 0 || s > most) return true;
  return false;
}
static bool refused(const FtkPagedAttnDesc* d) {
  return !d || wide(d) || d->B <= 0 || d->B > (1 << 30) || d->Hkv <= 0 || d->Hq <= 0 || d->Hq % d->Hkv || d->Hq > (1 << 20) || (d->hd != 64 && d->hd != 128) ||
         (d->type != FTK_T_BF16 && d->type != FTK_T_FP16) || d->page_shift < 0 || d->page_shift > 30 || d->table_cols <= 0 ||
         d->table_cols > (0x7fffff00ll >> d->page_shift) || d->n_pages <= 0 || d->n_pages > 0x7fffffff || d->B * d->Hq > 0x7fffffff ||
         d->B * d->Hq * (((d->table_cols << d->page_shift) >> 6) + 1) > (1ll << 38) ||      // a CTA counts its tiles in 32 bits
         d->block_shift < 0 || d->block_shift > 6 || d->block_shift > d->page_shift;
}

}  // namespace ftk
using namespace ftk;

extern "C" long long ftk_paged_attn_e4m3_scratch(const FtkPagedAttnDesc* d) { return refused(d) ? -2 : plan_of(*d).bytes; }

extern "C" int ftk_paged_attn_e4m3(const FtkPagedAttnDesc* d, void* scratch, void* stream) {
  if (refused(d) || !d->q || !d->o || !d->lse || !d->k_pages || !d->v_pages || !d->k_scales || !d->v_scales || !d->table || !d->lengths) return -2;
  const Plan8 p = plan_of(*d);
  if (p.split && !scratch) return -2;
  cudaStream_t s = (cudaStream_t)stream;
  const bool bf = d->type == FTK_T_BF16;
  if (p.rows == 1) {
    if (d->hd == 64) return bf ? launch<__nv_bfloat16, 64, 1>(*d, p, scratch, s) : launch<__half, 64, 1>(*d, p, scratch, s);
    return bf ? launch<__nv_bfloat16, 128, 1>(*d, p, scratch, s) : launch<__half, 128, 1>(*d, p, scratch, s);
  }
  if (p.rows == 8) {
    if (d->hd == 64) return bf ? launch<__nv_bfloat16, 64, 8>(*d, p, scratch, s) : launch<__half, 64, 8>(*d, p, scratch, s);
    return bf ? launch<__nv_bfloat16, 128, 8>(*d, p, scratch, s) : launch<__half, 128, 8>(*d, p, scratch, s);
  }
  if (d->hd == 64) return bf ? launch<__nv_bfloat16, 64, 16>(*d, p, scratch, s) : launch<__half, 64, 16>(*d, p, scratch, s);
  return bf ? launch<__nv_bfloat16, 128, 16>(*d, p, scratch, s) : launch<__half, 128, 16>(*d, p, scratch, s);
}
