// Attention of one new token per sequence over a paged key-value cache held in 8 bits (e4m3) with a scale per block of rows and head.
//
// Mathematics.  With ks and vs the scales of token t's key and value, x_t = scale ks_t (q . k_t), o = sum_t softmax_t(x) vs_t v_t and
// lse = log sum_t exp(x_t).  What is added up for the output are terms of size exp(x_t) vs_t, so the running maximum m is that of
// y_t = x_t + log2 vs_t (base 2; of vs_t its power of two): the accumulator is sum_t 2^(x_t - m) vs_t v_t, the sum l = sum_t 2^(x_t - m),
// which no scale from 2^-100 to 2^100 takes out of fp32.  Parts join as in paged_attention.cu, which this follows: the list of tiles,
// the pieces, the rings and the join are the same.
//
// What bounds it: every key and value is read once, in 8 bits; the copy bandwidth, with twice the arithmetic per byte of a 16-bit cache.
//
// A warp takes 32 tokens of a tile at a time.  fp16 holds every e4m3 value, so keys and values go into the matrix instructions as they
// are, converted in registers, and the scales are applied to scores and probabilities, which are few.  The queries are in fp16 too, a
// row at a time times the power of two that brings its largest element to 2^14 .. 2^15: what that loses is below 2^-39 of it.  The
// elements of a product's inner dimension may come in any order that both operands share: a thread's four neighbouring bytes of a key
// row are two operand registers as they are, and of a value column one byte permutation brings the bytes of two tokens together, with
// even columns in one product and odd ones in another.  Probabilities times scales are split into two halves of fp16, carried times 2^14.
#include "e4m3.cuh"
#include "paged_attn.cuh"

extern "C" int* ftk_status_word(void);

namespace ftk {

constexpr int A8_WARPS = 4, A8_TOKENS = 32;      // of a CTA that shares its SM; tokens that a warp takes at a time
constexpr float A8_SHIFT = 16384.f;
__host__ inline long long a8_whole(long long heads, long long sms) { return heads <= sms ? 9 + 28 * heads / sms : 20; }

template <int ROWS, int HD, int W> struct A8Smem {
  static constexpr int CTAS = W > A8_WARPS ? 1 : (HD == 64 ? 3 : 2);
  static constexpr int DATA = A8_TOKENS * HD * 2, STAGE = DATA + A8_TOKENS * 8;      // keys, values, scales
  static constexpr int STAGES = 3;
  static constexpr int RING = STAGES * STAGE;
  static constexpr int COLS = ROWS == 16 && HD == 128 ? 32 : 64;      // columns of the accumulators of all warps that are joined at a time
  static constexpr int MERGE = W * ROWS * COLS * 4;
  static constexpr bool OWN = W <= A8_WARPS;                  // in memory of their own, or in the rings of a head that is through
  static constexpr int BYTES = W * RING + (OWN ? MERGE : 0) + 2 * W * ROWS * 4 + W * STAGES * 4;
  static_assert(OWN || MERGE <= W * RING, "the accumulators fit the rings");
  static_assert(CTAS * (BYTES + 1024) <= 228 * 1024 && BYTES <= 227 * 1024, "the CTAs of an SM share its memory");
};
template <int ROWS, int HD> constexpr int A8_ALONE = HD == 64 && ROWS == 8 ? 16 : 8;

__device__ __forceinline__ void copy4(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(there ? 4 : 0) : "memory");
}

template <typename T, int HD, int ROWS, bool SPLIT, int W>
__global__ void __launch_bounds__(W * 32, A8Smem<ROWS, HD, W>::CTAS) paged_attn_e4m3_kernel(const __grid_constant__ PagedAttn a, int* status) {
  typedef A8Smem<ROWS, HD, W> SM;
  static_assert(!SPLIT || SM::OWN, "a piece goes on while the parts are joined");
  constexpr int N = A8_TOKENS, TILE = N * W;
  constexpr int STAGES = SM::STAGES, STAGE = SM::STAGE, CH = HD / 16, NT = HD / 8;      // CH: 16-byte chunks of a row
  constexpr int RR = ROWS / 8;
  extern __shared__ __align__(256) unsigned char smem[];
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
        page = (int)paged_page(table, g.b, tok);
        if (page < 0) ft_index_ok(-1, 1, status);
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
  const long long k_lane = lrow * d.kp_rs + lchunk * 16, v_lane = lrow * d.vp_rs + lchunk * 16;
  const auto load = [&](int stage) {
    const int pages = page_of[0];
#pragma unroll
    for (int i = 0; i + 1 < AHEAD; ++i) page_of[i] = page_of[i + 1];
    page_of[AHEAD - 1] = look();
    if (to_load > 0) {
      const int head = f.h / a.subs, tok0 = f.t * TILE + warp * N;
      const unsigned char* kb = (const unsigned char*)d.k_pages + head * d.kp_hs;
      const unsigned char* vb = (const unsigned char*)d.v_pages + head * d.vp_hs;
      const uint32_t dst = ring_s + stage * STAGE + lane_at, sdst = ring_s + stage * STAGE + SM::DATA + lane * 4;
      unsigned ok;
      if (one_page) {
        const int n = pages < 0 ? 0 : min(N, f.n - tok0);      // rows that are there
        const long long page = pages < 0 ? 0 : pages, in = paged_row(table, tok0);
        ok = n >= N ? 0xffffffffu : (1u << n) - 1;
        const unsigned char* k = kb + page * d.kp_ps + in * d.kp_rs + k_lane;
        const unsigned char* v = vb + page * d.vp_ps + in * d.vp_rs + v_lane;
        const long long k_step = RSTEP * d.kp_rs, v_step = RSTEP * d.vp_rs;
#pragma unroll
        for (int c = 0; c < COPIES; ++c) {
          const bool t = c * RSTEP + lrow < n;
          const uint32_t at = dst + c * RSTEP * HD + (lane_sw ^ (swizzle(c * RSTEP + lrow) << 4));
          copy16(at, t ? k : kb, t);
          copy16(at + N * HD, t ? v : vb, t);
          k += k_step, v += v_step;
        }
        const bool t = lane < n;
        const long long block = t ? (in + lane) >> d.block_shift : 0;
        copy4(sdst, d.k_scales + page * d.ks_ps + head * d.ks_hs + block, t);
        copy4(sdst + N * 4, d.v_scales + page * d.vs_ps + head * d.vs_hs + block, t);
      } else {
        ok = __ballot_sync(0xffffffffu, pages >= 0);
#pragma unroll
        for (int c = 0; c < COPIES; ++c) {
          const int row = c * RSTEP + lrow;
          const long long page = __shfl_sync(0xffffffffu, pages, row), in = paged_row(table, tok0 + row);
          const bool t = page >= 0;
          const uint32_t at = dst + c * RSTEP * HD + (lane_sw ^ (swizzle(row) << 4));
          copy16(at, t ? kb + page * d.kp_ps + in * d.kp_rs + lchunk * 16 : kb, t);
          copy16(at + N * HD, t ? vb + page * d.vp_ps + in * d.vp_rs + lchunk * 16 : vb, t);
        }
        const bool t = pages >= 0;
        const long long page = t ? pages : 0, block = t ? paged_row(table, tok0 + lane) >> d.block_shift : 0;
        copy4(sdst, d.k_scales + page * d.ks_ps + head * d.ks_hs + block, t);
        copy4(sdst + N * 4, d.v_scales + page * d.vs_ps + head * d.vs_hs + block, t);
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
  uint32_t q[CH][2 * RR];               // of chunk c: elements 4 c0' .. + 3 of row r0, then of row r0 + 8
  float acc[NT][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, sc[2] = {0.f, 0.f};
  const int r0 = lane >> 2, c0 = (lane & 3) * 2;
  const auto begin = [&]() {            // queries of the head at `p`; rows beyond the group are zero
    const int first = row0(p.h), rows = rows_of(p.h);
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
      const int e = min(max((int)(__float_as_uint(most) >> 23) - 127, -100), 127);
      const float by = __uint_as_float((uint32_t)(127 + 14 - e) << 23);
      sc[r] = (float)d.scale * LOG2E * __uint_as_float((uint32_t)(127 - 14 + e) << 23);
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const float2 x = Half16<T>::up(u[c].x), y = Half16<T>::up(u[c].y);
        q[c][2 * r] = Half16<__half>::down(x.x * by, x.y * by), q[c][2 * r + 1] = Half16<__half>::down(y.x * by, y.y * by);
      }
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
  // this lane's row for ldmatrix: of four groups of eight tokens at one chunk
  const uint32_t l_at = lane * HD + (swizzle(lane) << 4);
  int stage = 0;
  for (bool more = true; more; more = left > 0) {
    if (left > 0) {
      copy_wait<STAGES - 2>();
      __syncwarp();
      const uint32_t ks = ring_s + stage * STAGE + l_at, vs = ks + N * HD;
      const float* scales = reinterpret_cast<const float*>(ring + stage * STAGE + SM::DATA);
      const unsigned ok = there[stage];
      const int refill = stage == 0 ? STAGES - 1 : stage - 1;
      float s[4][4] = {};
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        uint32_t b[4];
        ldm4(ks ^ (c << 4), b);
        const uint32_t qa[4] = {q[c][0], ROWS == 16 ? q[c][2 * RR - 2] : 0u, q[c][1], ROWS == 16 ? q[c][2 * RR - 1] : 0u};
#pragma unroll
        for (int j = 0; j < 4; ++j) mma16<__half>(s[j], qa, e4m3_up(b[j] & 0xffffu), e4m3_up(b[j] >> 16));
      }
      load(refill);                     // the stage that the tile before left: its reads are behind the warp's barrier
      // masked scores, and the larger maximum of the row's tokens and what was there
      float kf[8], vf[8], lv[8];        // of this thread's tokens: 8 j + c0, + 1
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 x = *reinterpret_cast<const float2*>(scales + j * 8 + c0), y = *reinterpret_cast<const float2*>(scales + N + j * 8 + c0);
        kf[2 * j] = x.x, kf[2 * j + 1] = x.y, vf[2 * j] = y.x, vf[2 * j + 1] = y.y;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        lv[i] = (float)max((int)(__float_as_uint(vf[i]) >> 23 & 255) - 127, -100);
        vf[i] *= A8_SHIFT;
      }
      uint32_t hi[2][4] = {}, lo[2][4] = {};      // of two steps of 16 tokens
      float grow[2];
      bool moved = false;
#pragma unroll
      for (int r = 0; r < RR; ++r) {
        float x[8], top = m[r];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = s[i >> 1][2 * r + (i & 1)] * (kf[i] * sc[r]);
        if (ok != 0xffffffffu) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (!(ok >> ((i >> 1) * 8 + c0 + (i & 1)) & 1u)) x[i] = -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, x[i] + lv[i]);
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float base = top == -INFINITY ? 0.f : top;
        moved |= top != m[r];
        grow[r] = exp2_of(m[r] - base);
        m[r] = top;
        float e[8], sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          e[i] = exp2_of(x[i] - base), e[i + 1] = exp2_of(x[i + 1] - base);
          sum += e[i] + e[i + 1];
          e[i] *= vf[i], e[i + 1] *= vf[i + 1];
        }
        l[r] = l[r] * grow[r] + sum;
#pragma unroll
        for (int j = 0; j < 4; ++j) {      // tokens 8 j and on: step j / 2, its first or second half
          const uint32_t h = Half16<__half>::down(e[2 * j], e[2 * j + 1]);
          const float2 u = Half16<__half>::up(h);
          hi[j >> 1][(j & 1) * 2 + r] = h;
          lo[j >> 1][(j & 1) * 2 + r] = Half16<__half>::down(e[2 * j] - u.x, e[2 * j + 1] - u.y);
        }
      }
      if (__any_sync(0xffffffffu, moved)) {
        const float g0 = grow[0], g1 = ROWS == 16 ? grow[RR - 1] : grow[0];
#pragma unroll
        for (int i = 0; i < NT; ++i) acc[i][0] *= g0, acc[i][1] *= g0, acc[i][2] *= g1, acc[i][3] *= g1;
      }
      if (ROWS != 16) {
#pragma unroll
        for (int t = 0; t < 2; ++t) hi[t][1] = lo[t][0], hi[t][3] = lo[t][2];
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
    float scale[RR];                    // of the warp's part: to the maximum of all, without the 2^14
#pragma unroll
    for (int r = 0; r < RR; ++r) {
      float top = m[r];
#pragma unroll
      for (int w = 0; w < W; ++w) top = fmaxf(top, stat[w * ROWS + r * 8 + r0]);
      scale[r] = exp2f(m[r] - (top == -INFINITY ? 0.f : top)) * (1.f / A8_SHIFT);
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
        if (!SPLIT || whole) {
          const float by = sum == 0.f ? 0.f : 1.f / sum;
          T* o = (T*)d.o + p.b * d.o_bs + (first + row) * d.o_hs + col;
          *reinterpret_cast<uint32_t*>(o) = Half16<T>::down(sum == 0.f ? 0.f : v.x * by, sum == 0.f ? 0.f : v.y * by);
          if (col == 0) d.lse[(long long)p.b * d.Hq + first + row] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * LN2;
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
  bool split, alone;               // heads cut into pieces; a CTA per SM, for few heads
  long long ctas, heads, headers, bytes;      // heads: of all sequences, a part of a group counting as one
};
template <int ROWS, int HD> constexpr int A8_CTAS = A8Smem<ROWS, HD, A8_WARPS>::CTAS;
static Plan8 plan_of(const FtkPagedAttnDesc& d) {
  Plan8 p;
  const long long group = d.Hq / d.Hkv;
  p.subs = (int)((group + 15) / 16);
  p.sub_heads = (int)((group + p.subs - 1) / p.subs);
  p.rows = p.sub_heads <= 8 ? 8 : 16;
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  p.ctas = p.heads = d.B * d.Hkv * p.subs;
  p.headers = p.bytes = 0;
  const long long tiles = ((d.table_cols << d.page_shift) + 63) / 64;
  p.alone = p.heads <= sms;
  p.split = tiles > a8_whole(p.heads, sms);
  if (p.split) {
    p.ctas = (d.hd == 64 ? (p.rows == 8 ? A8_CTAS<8, 64> : A8_CTAS<16, 64>) : (p.rows == 8 ? A8_CTAS<8, 128> : A8_CTAS<16, 128>)) * (long long)sms;
    p.headers = p.heads < p.ctas ? p.heads : p.ctas;
    p.bytes = p.headers * PA_HEADER * 4 + p.ctas * 2 * p.rows * (d.hd + 2) * 4;
  }
  return p;
}

template <typename T, int HD, int ROWS>
static int launch(const FtkPagedAttnDesc& d, const Plan8& p, void* scratch, cudaStream_t s) {
  PagedAttn a = {d, (int)(d.Hq / d.Hkv), p.subs, p.sub_heads, p.heads < p.ctas, (int*)scratch, nullptr};
  a.parts = (float*)((char*)scratch + p.headers * PA_HEADER * 4);
  int* status = ftk_status_word();
  if (!p.split && p.alone) {
    constexpr int W = A8_ALONE<ROWS, HD>, bytes = A8Smem<ROWS, HD, W>::BYTES;
    const auto kernel = paged_attn_e4m3_kernel<T, HD, ROWS, false, W>;
    const int rc = (int)cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    return rc ? rc : launch_pdl(kernel, dim3((unsigned)p.ctas), dim3(W * 32), bytes, s, a, status);
  }
  constexpr int bytes = A8Smem<ROWS, HD, A8_WARPS>::BYTES;
  const auto whole = paged_attn_e4m3_kernel<T, HD, ROWS, false, A8_WARPS>, split = paged_attn_e4m3_kernel<T, HD, ROWS, true, A8_WARPS>;
  const auto kernel = p.split ? split : whole;
  int rc = (int)cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (rc) return rc;
  rc = launch_pdl(kernel, dim3((unsigned)p.ctas), dim3(A8_WARPS * 32), bytes, s, a, status);
  if (rc || !p.split) return rc;
  return launch_join<T, HD, ROWS, 0>(a, p.heads, p.ctas, p.headers, s);
}

static bool refused(const FtkPagedAttnDesc* d) {
  return !d || d->B <= 0 || d->B > (1 << 30) || d->Hkv <= 0 || d->Hq <= 0 || d->Hq % d->Hkv || d->Hq > (1 << 20) || (d->hd != 64 && d->hd != 128) ||
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
  if (p.rows == 8) {
    if (d->hd == 64) return bf ? launch<__nv_bfloat16, 64, 8>(*d, p, scratch, s) : launch<__half, 64, 8>(*d, p, scratch, s);
    return bf ? launch<__nv_bfloat16, 128, 8>(*d, p, scratch, s) : launch<__half, 128, 8>(*d, p, scratch, s);
  }
  if (d->hd == 64) return bf ? launch<__nv_bfloat16, 64, 16>(*d, p, scratch, s) : launch<__half, 64, 16>(*d, p, scratch, s);
  return bf ? launch<__nv_bfloat16, 128, 16>(*d, p, scratch, s) : launch<__half, 128, 16>(*d, p, scratch, s);
}
