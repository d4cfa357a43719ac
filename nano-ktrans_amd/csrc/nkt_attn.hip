// Attention over the paged cache.
#include "nkt_attn_device.h"

namespace nkt {

namespace {

// Positions p0 .. p0 + 63 that a token of the sequence sees, as bits.
template <bool TREE>
__device__ __forceinline__ uint64_t visible(const AttnArgs& a, const Seq& s, int token, int p0) {
  const int inside = s.len - p0;  // > 0
  const uint64_t valid = inside >= 64 ? ~0ull : (1ull << inside) - 1;
  if (!TREE) {
    const int past = s.context + token - p0;
    return past < 0 ? 0 : past >= 63 ? valid : valid & ((2ull << past) - 1);
  }
  const int j0 = p0 - s.context;  // draft index of p0
  if (j0 <= -64) return valid;
  const int64_t* words = a.tree + (int64_t)(s.first + token) * a.words;
  uint64_t bits;
  if (j0 < 0) {
    bits = (1ull << -j0) - 1 | (uint64_t)words[0] << -j0;
  } else {
    const int w = j0 >> 6, sh = j0 & 63;
    bits = w < a.words ? (uint64_t)words[w] >> sh : 0;
    if (sh && w + 1 < a.words) bits |= (uint64_t)words[w + 1] << (64 - sh);
  }
  return bits & valid;
}

// What takes the roundings' common part out of sums of weight x scale: the quotient of
// these before and after.  (Sums that say nothing, of scales that are not finite or of both
// signs, change nothing.)
__device__ __forceinline__ float even_by(float exact, float rounded) {
  const float by = exact / rounded;
  return __builtin_fabsf(by - 1.f) < 0x1p-7f ? by : 1.f;
}

// c + lo(w) + hi(w) of a pair of bf16
__device__ __forceinline__ float add_pair(uint32_t w, float c) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const bf16x2 ones = {(__bf16)1.0f, (__bf16)1.0f};
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w), ones, c, false);
}

__device__ __forceinline__ float max_xor32(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

__device__ __forceinline__ float max_xor16(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

constexpr float kUnseen = -__builtin_huge_valf();  // the running maximum before any score
// Weights may differ by this much (in log2) from what the row's largest score so
// far gives, so that most tiles skip the rescale; neither the fp32 sums nor a bf16
// weight's relative precision notice.  A score that passes the running maximum m
// moves it to `above` over itself, and m moves again once a score passes it by
// kSlack - above.  bf16: above = kSlack, no weight is over 1, and a sum passes
// fp32's range only if the values' own sum may.  int8 rounds weight x scale to bf16,
// where weights of 2^-8 would cost the smallest scales their bits: above = 0
// until the row sees a value's scale past kLargeScale, then as bf16 (2^20 tokens x
// a weight of 2^8 x 127 x kLargeScale are within the range).
constexpr float kSlack = 8.0f;
constexpr float kLargeScale = 0x1p90f;

// 2^(m - top): the factor that brings sums under maximum m to maximum top >= m
// (0 for sums of no score, also where there is no other either).
__device__ __forceinline__ float factor(float m, float top) {
  return __builtin_amdgcn_exp2f(m - fmaxf(top, -__FLT_MAX__));
}

// What a row's weights are told from afterwards: exp2(score - maximum) / sum.
__device__ __forceinline__ void keep_stats(const AttnArgs& a, int token, int head, float m, float l) {
  float* to = a.stats + 2 * ((int64_t)token * a.heads + head);
  to[0] = m;
  to[1] = l;
}

__device__ __forceinline__ bool non_finite_pair(uint32_t w) {
  return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
}

constexpr int kTileRows = 128, kTileKeys = 64;  // of the tile form
constexpr int kPairRows = 64;                   // of the same where a sequence has no more
constexpr int kRowRows = 16;                    // of the row form

// How a launch is cut: items (a tile of rows of one head) x splits (of chunk
// positions each).  Where an item's rows see more than one chunk, each split
// leaves its weighted sum of values (fp32, not divided), running maximum and
// sum in the workspace, and join_kernel adds them in order.
struct Parts {
  int items, splits, chunk;
  int rows;   // of an item
  bool whole;  // an item is a sequence with all its rows
  float* o;   // [items, kv_heads, splits, rows, D]
  float* ml;  // [items, kv_heads, splits, rows, 2]
  __device__ __forceinline__ int64_t row(int item, int h, int kv_heads, int split, int r) const {
    return (((int64_t)item * kv_heads + h) * splits + split) * rows + r;
  }
};

__device__ __forceinline__ int first_row(const AttnArgs& a, int b) { return a.starts ? a.starts[b] : b; }

// The sequence of a tile of kTileRows rows.  Sequence b's tiles start at
// starts[b] G / 128 + b, which ascends and leaves room for its ceil(n G / 128)
// tiles: the last b that starts at or before this tile, found by 64 lanes at a
// time.  block_of_tile: the tile's number in its sequence (which may lie past
// its rows, or before them where starts does not ascend from 0).
__device__ __forceinline__ int sequence_of_tile(const AttnArgs& a, int G, int tile, int lane) {
  int b = 0;
  for (int n = a.seqs; n > 1;) {
    const int step = (n + 63) / 64;
    const int i = b + lane * step;
    const bool before =
        lane * step < n && (int64_t)first_row(a, i < a.seqs ? i : a.seqs - 1) * G / kTileRows + i <= tile;
    const int count = __popcll(__ballot(before));
    const int skip = count > 0 ? (count - 1) * step : 0;
    b += skip;
    n = n - skip < step ? n - skip : step;
  }
  return __builtin_amdgcn_readfirstlane(b);
}
__device__ __forceinline__ int block_of_tile(const AttnArgs& a, int G, int tile, int b, const SeqWords& w) {
  const int first = a.starts ? __builtin_amdgcn_readfirstlane(w.start) : b;
  return tile - ((int)((int64_t)first * G / kTileRows) + b);
}

// One past the last position that some row of rows r0 .. r0 + count - 1 sees.
template <bool TREE>
__device__ __forceinline__ int end_of_rows(const Seq& s, int G, int r0, int count) {
  const int rows = s.n * G;
  const int last = (r0 + count < rows ? r0 + count : rows) - 1;
  const int end = s.context + last / G + 1;
  return TREE || end > s.len ? s.len : end;
}

// ---------------------------------------------------------------------------
// Tile form: one workgroup takes 128 rows (32 per wave) against tiles of 64
// tokens, double-buffered in LDS.
//   S^T = K . Q^T on 32x32x16 matrix instructions: a lane then holds scores of
//   one row (its column) for 32 of the 64 tokens, so the softmax needs one
//   exchange between the wave's halves, and the running rescale of O^T = V^T .
//   P^T (rows = dimensions, column = the lane's row) is one factor per lane.
//   The order of the tokens within a product is free: row r of a key tile
//   holds token r with bits 2 and 3 swapped, which makes the scores that a lane
//   gets the 8 consecutive tokens that it must supply as P^T, and the value
//   layout's 16-byte pieces the V^T operand: nothing moves between lanes.
// Keys lie in LDS as rows of 16-byte chunks, chunk c of row r at c ^ key(r):
// the same chunk of 16 rows lies in 16 places of the 256 bytes that LDS reads
// at a time; values as they come.
// bf16 tiles go straight from global memory into LDS, int8 ones through
// registers (exact bf16 integers; the scales multiply scores and weights).
// A weight is rounded once, to the bf16 operand of the second product: off by
// 2^-8 of itself at most, as the output's own rounding is, and the errors of a
// row's tokens mostly cancel.  Scores, maxima, sums and outputs stay fp32.
//
// The steps of a wave form a pipeline over half tiles u of 32 tokens:
//   S(u + 1) = K(u + 1) Q  beside the exponentials of u,
//   O += V(u) P(u)         beside the maximum of u + 1,
// so that the matrix cores and the vector unit work at the same time; keys run
// one tile ahead of values, and one barrier per tile covers both.
//
// Bound by the two units' shares of a SIMD's time and by power, not by memory.  A
// prompt of 8192 tokens, 32 / 4 heads, D = 128, bf16: 521 us, 1.05 PFLOP/s (a
// library product of 16384^3: 1.36), at a clock that falls to 1.8 of 2.4 GHz (557
// on a card that holds less); matrix cores busy 51 % of it, the vector unit 47 %,
// 5.3 vector instructions per matrix one, waves waiting 20 %, no bank conflict.
// int8, three chunks of up to 1021 tokens on up to 9000, 32 / 8 heads: 405 us and
// 21 of join, 0.70 PFLOP/s; 31 % and 51 %, 10.9 vector instructions: widening the
// codes and the two scales are what it has more.
// ---------------------------------------------------------------------------
template <int D, bool I8>
struct TileLds {
  __align__(16) uint8_t k[2][kTileKeys * D * 2];
  __align__(16) uint8_t v[2][kTileKeys * D * 2];
  __align__(16) float ks[4][I8 ? kTileKeys : 4];  // of tile t at t & 3: read until the end of tile t
  __align__(16) float vs[2][I8 ? kTileKeys : 4];
  int flag;
};

template <int D>
__device__ __forceinline__ int chunk_key(int r) {
  return D == 128 ? r & 15 : r >> 1 & 7;
}

// ROWS = 64 (no sequence has more): one pair of waves takes the rows against the
// first half of every tile's tokens, the other against the second, and their
// results are added at the end: half the products and exponentials that 128
// half-empty rows would cost.  64 drafts of up to 8 tokens on up to 8192, 32 / 4
// heads, int8 117 us, as 128 rows 151; bf16 137 and 153.
//
// STATS: each row's maximum and sum go out as well (keep_stats), the sum of the weights
// before they are rounded to bf16; outputs are divided by that after the rounding, as without
// STATS.  The prompt above, whole calls whose last 64 tokens count: 598 us, with the one sum
// 580 (and outputs off by 0.0021 of their size instead of 0.0019), forward 553.
template <int D, bool I8, bool TREE, int ROWS, bool STATS>
__global__ __launch_bounds__(256, 2) void attn_tile_kernel(CacheView c, AttnArgs a, Parts part) {
  constexpr int kQ = D / 16;       // Q fragments, and key products per half tile
  constexpr int kO = D / 32;       // output tiles
  constexpr int kChunks = D / 8;   // 16-byte chunks of a key row
  constexpr int kLoads = kTileKeys * D * 2 / 4096;  // 16-byte loads per thread, keys or values
  // value fragments read ahead, in 16 tokens (the registers go to int8's staging, to the unrounded sum)
  constexpr int kVAhead = (I8 || (STATS && ROWS == kTileRows)) && D == 128 ? 1 : 2;
  constexpr bool kPairs = ROWS == kPairRows;
  __shared__ TileLds<D, I8> lds;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int half = lane >> 5, col = lane & 31;
  const int HK = c.kv_heads, G = a.heads / HK;
  // heads first: the workgroups of one head run on the same XCDs (workgroup i
  // on XCD i % 8) and find its keys in their L2; late tiles, which see the
  // most, first
  const int h = (int)(blockIdx.x % (unsigned)HK);
  const int rest = (int)(blockIdx.x / (unsigned)HK);
  const int split = rest % part.splits;
  const int tile = part.items - 1 - rest / part.splits;
  const int begin = split * part.chunk;
  const int b = kPairs || part.whole ? tile : sequence_of_tile(a, G, tile, lane);
  const SeqWords words = sequence_words(a, b);
  // 64 entries of the page table from pages_at on
  int pages_at = begin >> c.page_shift;
  int pages = table_entries(a, b, pages_at, lane);
  const int block = kPairs || part.whole ? 0 : block_of_tile(a, G, tile, b, words);
  const Seq s = sequence(c, a, b, words, h == 0 && block == 0 && split == 0 && tid == 0);
  const int rows = s.n * G;
  const int r0 = block * ROWS;
  if (block < 0 || r0 >= rows) return;
  const int mine = kPairs ? __builtin_amdgcn_readfirstlane(wave) >> 1 : 0;  // the wave's half of a tile
  // This lane's row; rows past the end repeat the last one and are not stored.
  // (Worked out again where it is needed, rather than held in registers that
  // the loop has no room for.)
  auto my_row = [&] {
    int lane_col = col;
    __asm__ volatile("" : "+v"(lane_col));
    return r0 + (kPairs ? wave & 1 : wave) * 32 + lane_col;
  };
  auto my_token = [&] {
    const int row = my_row();
    return (row < rows ? row : rows - 1) / G;
  };
  u32x4 qf[kQ];
  {
    const int row = my_row() < rows ? my_row() : rows - 1;
    const int token = row / G;
    const uint16_t* q = a.q + ((int64_t)(s.first + token) * a.heads + h * G + (row - token * G)) * D;
#pragma unroll
    for (int i = 0; i < kQ; ++i) qf[i] = *(const u32x4*)(q + i * 16 + half * 8);
  }

  // the positions that the workgroup takes: its part of those that its rows see
  const int row_end = end_of_rows<TREE>(s, G, r0, ROWS);
  if (split > 0 && begin >= row_end) return;
  const int end = row_end - begin > part.chunk ? begin + part.chunk : row_end;
  // positions below are seen by all rows
  const int all_see = TREE ? s.context : s.context + r0 / G + 1;
  const int open = all_see < s.len ? all_see : s.len;

  f32x16 o[kO];
#pragma unroll
  for (int i = 0; i < kO; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[i][r] = 0.f;
  // Running maximum (log2), sum, and what a score less m must pass for m to move:
  // -infinity until the row has seen a token, then kSlack - above.
  float m = 0.f, l = 0.f, limit = -__builtin_huge_valf();
  // (bf16's 128 rows beside weights have no register for limit: it is 0 once the row has
  // seen a token, and that shows in m, which is never 0 from there on)
  constexpr bool kSeenByM = STATS && !I8 && !kPairs;
  auto row_sees = [&] { return kSeenByM ? !(m == 0.f) : limit >= 0.f; };
  // (as in the row form; bf16: l is the sum of the rounded weights, as without STATS, and
  // exact that before; int8's 128 rows of D = 128 have no registers left for it, and have more
  // rows, so that less of the roundings is common to all)
  constexpr bool kEvens = STATS && (!I8 || D == 64 || kPairs);
  float exact = 0.f, rounded = 0.f;  // (rounded: int8)
  const float scale2 = a.scale * kLog2e;
  const int mask = (1 << c.page_shift) - 1;

  // the first tile at or after p whose page is in the cache (or some p >= end); its (page, head) block
  auto find = [&](int p, int64_t* at) __attribute__((always_inline)) {
    for (; p < end; p += kTileKeys) {
      const int i = p >> c.page_shift;
      if (i - pages_at >= 64) {
        pages_at = i;
        pages = table_entries(a, b, i, lane);
      }
      const int page = __builtin_amdgcn_readlane(pages, i - pages_at);
      if (page >= 0 && page < c.num_pages) {
        *at = (((int64_t)page * HK + h) << c.page_shift) + (p & mask);
        break;
      }
      if (tid == 0) report(c.status, kBadPage);
    }
    return p;
  };
  // Staging.  bf16: straight into LDS.  int8: into registers (load_*), from
  // there converted into LDS (land_*): values in the first half of a tile's
  // step and keys in the second, so that they share the registers.
  struct Raw {
    u32x4 w[I8 ? kLoads / 2 : 1];
    float scale;
  };
  auto load_k = [&](int64_t at, int buf, Raw& raw) __attribute__((always_inline)) {
    if (!I8) {
      const uint8_t* kb = c.k + at * (D * 2);
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const int slot = (wave * kLoads + j) * 64 + lane;
        const int r = slot / kChunks, ch = (slot % kChunks) ^ chunk_key<D>(r);
        const int t = (r & ~12) | (r & 4) << 1 | (r & 8) >> 1;
        load16_to_lds(kb + t * (D * 2) + ch * 16, lds.k[buf] + (wave * kLoads + j) * 1024);
      }
    } else {
      const uint8_t* kb = c.k + at * D;
#pragma unroll
      for (int j = 0; j < kLoads / 2; ++j) raw.w[j] = *(const u32x4*)(kb + (j * 256 + tid) * 16);
      if (tid < kTileKeys) raw.scale = c.k_scales[at + tid];
    }
  };
  auto load_v = [&](int64_t at, int buf, Raw& raw) __attribute__((always_inline)) {
    if (!I8) {
      const uint8_t* vb = c.v + at * (D * 2);
#pragma unroll
      for (int j = 0; j < kLoads; ++j)
        load16_to_lds(vb + ((wave * kLoads + j) * 64 + lane) * 16, lds.v[buf] + (wave * kLoads + j) * 1024);
    } else {
      const uint8_t* vb = c.v + at * D;
#pragma unroll
      for (int j = 0; j < kLoads / 2; ++j) raw.w[j] = *(const u32x4*)(vb + (j * 256 + tid) * 16);
      if (tid < kTileKeys) raw.scale = c.v_scales[at + tid];
    }
  };
  auto widen = [&](u32x4 w, u32x4* x) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t lo, hi;
      bf16_of_codes(w[j], &lo, &hi);
      x[j >> 1][2 * (j & 1)] = lo;
      x[j >> 1][2 * (j & 1) + 1] = hi;
    }
  };
  auto land_k = [&](int buf, int n, Raw& raw) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < kLoads / 2; ++j) {
      const int piece = j * 256 + tid;
      u32x4 x[2];
      __asm__ volatile("" : "+v"(raw.w[j]));  // (widened here, not where it is loaded)
      widen(raw.w[j], x);
      const int t = piece / (D / 16), ch = piece % (D / 16) * 2;
      const int r = (t & ~12) | (t & 4) << 1 | (t & 8) >> 1;
      *(u32x4*)(lds.k[buf] + (r * kChunks + (ch ^ chunk_key<D>(r))) * 16) = x[0];
      *(u32x4*)(lds.k[buf] + (r * kChunks + ((ch + 1) ^ chunk_key<D>(r))) * 16) = x[1];
    }
    if (tid < kTileKeys) lds.ks[n & 3][tid] = raw.scale * scale2;
  };
  auto land_v = [&](int buf, Raw& raw) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < kLoads / 2; ++j) {
      const int piece = j * 256 + tid;
      u32x4 x[2];
      __asm__ volatile("" : "+v"(raw.w[j]));
      widen(raw.w[j], x);
      const int g16 = piece / D, d = piece % D;
      *(u32x4*)(lds.v[buf] + ((2 * g16) * D + d) * 16) = x[0];
      *(u32x4*)(lds.v[buf] + ((2 * g16 + 1) * D + d) * 16) = x[1];
    }
    if (tid < kTileKeys) lds.vs[buf][tid] = raw.scale;
  };

  // Fragments of half tile sub (register r of its scores: token sub 32 + (r >>
  // 3) 16 + half 8 + (r & 7) of the tile).
  u32x4 kf[kQ], vf[2 * kO];
  auto read_k = [&](int buf, int sub) {
    // (key rows of both half tiles have the same chunk keys)
    int at = col * (D * 2) + (half ^ chunk_key<D>(col)) * 16;
    if (I8 && D == 128) __asm__ volatile("" : "+v"(at));  // (no registers to hold every chunk's place)
#pragma unroll
    for (int i = 0; i < kQ; ++i) kf[i] = *(const u32x4*)(lds.k[buf] + sub * 32 * (D * 2) + (at ^ 32 * i));
  };
  auto read_v = [&](int buf, int sub, int from, int to) {
#pragma unroll
    for (int kk = from; kk < to; ++kk)
#pragma unroll
      for (int i = 0; i < kO; ++i)
        vf[kk * kO + i] = *(const u32x4*)(lds.v[buf] + ((sub * 4 + 2 * kk + half) * D + i * 32 + col) * 16);
  };
  f32x16 st;    // scores of the next half tile
  u32x4 pf[2];  // weights of the present one
  auto scores = [&](int from, int to) {
    if (from == 0) {
#pragma unroll
      for (int r = 0; r < 16; ++r) st[r] = 0.f;
    }
#pragma unroll
    for (int i = from; i < to; ++i) st = mfma32_bf16(kf[i], qf[i], st);
  };
  // the scores of half tile sub (int8: of tile n) less the running maximum, in log2
  auto less_maximum = [&](int n, int sub) {
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) {
      f32x4 f = {scale2, scale2, scale2, scale2};
      if (I8) f = *(const f32x4*)(lds.ks[n & 3] + sub * 32 + (q4 >> 1) * 16 + half * 8 + (q4 & 1) * 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) st[q4 * 4 + j] = __builtin_fmaf(st[q4 * 4 + j], f[j], -m);
    }
  };
  // the mask of half tile sub of the tile at p, where it needs one: true if so
  auto mask_scores = [&](int sub, int p) {
    const bool masks = p + sub * 32 + 32 > open || p + sub * 32 + 32 > end;
    if (masks) {
      const uint32_t vis = p < end ? (uint32_t)(visible<TREE>(a, s, my_token(), p) >> (sub * 32 + half * 8)) : 0u;
#pragma unroll
      for (int r = 0; r < 16; ++r)
        st[r] = vis >> ((r >> 3) * 16 + (r & 7)) & 1 ? st[r] : -__builtin_huge_valf();
    }
    return masks;
  };
  auto maximum = [&] {
    float top = fmaxf(fmaxf(st[0], st[1]), st[2]);
#pragma unroll
    for (int r = 3; r < 15; r += 2) top = fmaxf(fmaxf(top, st[r]), st[r + 1]);
    return max_xor32(fmaxf(top, st[15]));
  };
  float top = kUnseen;  // of the next half tile's scores, less m
  // (int8: p is the tile's position, scale the value scale of the lane's token of it)
  auto rescale = [&](int p, float scale) {
    const bool moves = top > (kSeenByM ? row_sees() ? 0.f : -__builtin_huge_valf() : limit);
    if (__any(moves || (I8 && scale > kLargeScale))) {
      const bool seen = row_sees();  // (nothing to rescale before)
      float above = kSeenByM ? kSlack : seen ? kSlack - limit : I8 ? 0.f : kSlack, up = 0.f;
      if (I8) {
        const uint64_t large = __ballot(scale > kLargeScale);
        if (large) {
          const uint64_t vis = p + kTileKeys > open ? visible<TREE>(a, s, my_token(), p) : ~0ull;
          up = above == 0.f && (vis & large) ? kSlack : 0.f;
          above += up;
        }
      }
      const float by = moves ? top + above : seen ? up : 0.f;
      const float fix = seen ? __builtin_amdgcn_exp2f(-by) : 1.f;
      m += by;
      if (kSeenByM)
        m = (moves || seen) && m == 0.f ? 0x1p-100f : m;
      else
        limit = moves || seen ? kSlack - above : limit;
      l *= fix;
      if (kEvens) exact *= fix;
      if (kEvens && I8) rounded *= fix;
#pragma unroll
      for (int r = 0; r < 16; ++r) st[r] -= by;
#pragma unroll
      for (int i = 0; i < kO; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[i][r] *= fix;
    }
  };
  // scores -> pf (buf, sub: the half tile's value scales)
  auto weights = [&](const f32x16& x, int buf, int sub) {
    float sum = 0.f;
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) {
      float w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        w[j] = __builtin_amdgcn_exp2f(x[q4 * 4 + j]);
        if (I8) l += w[j];
      }
      if (I8) {
        const f32x4 f = *(const f32x4*)(lds.vs[buf] + sub * 32 + (q4 >> 1) * 16 + half * 8 + (q4 & 1) * 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] *= f[j];
      }
      pf[q4 >> 1][2 * (q4 & 1)] = pack_pair(w[0], w[1]);
      pf[q4 >> 1][2 * (q4 & 1) + 1] = pack_pair(w[2], w[3]);
      if (kEvens) sum += (w[0] + w[1]) + (w[2] + w[3]);
      if (kEvens && I8)
        rounded = add_pair(pf[q4 >> 1][2 * (q4 & 1)], add_pair(pf[q4 >> 1][2 * (q4 & 1) + 1], rounded));
      if (!I8) l = add_pair(pf[q4 >> 1][2 * (q4 & 1)], add_pair(pf[q4 >> 1][2 * (q4 & 1) + 1], l));
    }
    if (kEvens) exact += sum;
  };
  auto products = [&](int from, int to) {
#pragma unroll
    for (int i = from; i < to; ++i) o[i % kO] = mfma32_bf16(vf[i], pf[i / kO], o[i % kO]);
  };
  // Values that some row must not see (or that lie past the sequence's end)
  // would still meet a weight of zero in the matrix products: 0 x NaN.  In
  // tiles with masked tokens, values past the end become zero, as do those that
  // are not finite, which add_odd adds to the rows that see them (int8:
  // values' scales instead, and such rows are NaN).
  int odd_from = end;  // the first tile with such values
  auto clean = [&](int buf, int p) __attribute__((always_inline)) {
    if (I8) {
      const float f = lds.vs[buf][lane];
      const bool odd = !(__builtin_fabsf(f) < __builtin_huge_valf());
      const uint64_t odds = __ballot(odd);
      if (odds == 0) return;
      if (visible<TREE>(a, s, my_token(), p) & odds) {
        if (!STATS) {
          l = __builtin_nanf("");
        } else {  // (the row's weights are numbers all the same)
#pragma unroll
          for (int i = 0; i < kO; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[i][r] = __builtin_nanf("");
        }
      }
      lds_barrier();  // every wave has read the scales
      if (wave == 0 && odd) lds.vs[buf][lane] = 0.f;
      lds_barrier();
      return;
    }
    if (tid == 0) lds.flag = 0;
    lds_barrier();
    bool odd = false;
    for (int i = tid; i < kTileKeys * kChunks; i += 256) {
      u32x4 w = *(const u32x4*)(lds.v[buf] + i * 16);
      const int inside = s.len - p - i / D * 8;
      if (inside < 8) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          w[j] &= (2 * j < inside ? 0xffffu : 0u) | (2 * j + 1 < inside ? 0xffff0000u : 0u);
        *(u32x4*)(lds.v[buf] + i * 16) = w;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) odd |= non_finite_pair(w[j]);
    }
    if (odd) lds.flag = 1;
    lds_barrier();
    if (!lds.flag) return;
    odd_from = p < odd_from ? p : odd_from;
    for (int i = tid; i < kTileKeys * kChunks; i += 256) {
      u32x4 w = *(const u32x4*)(lds.v[buf] + i * 16);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if ((w[j] & 0x7f80u) == 0x7f80u) w[j] &= 0xffff0000u;
        if ((w[j] & 0x7f800000u) == 0x7f800000u) w[j] &= 0xffffu;
      }
      *(u32x4*)(lds.v[buf] + i * 16) = w;
    }
    lds_barrier();
  };

  // The values that clean took out, from the cache, to the sums of the rows that
  // see them: once nothing rescales these any more (infinity x 0).
  auto add_odd = [&] {
    for (int p = odd_from; p < end; p += kTileKeys) {
      const int64_t page = a.table[(int64_t)b * a.width + (p >> c.page_shift)];
      if (page < 0 || page >= c.num_pages) continue;
      const int64_t at = ((page * HK + h) << c.page_shift) + (p & mask);
      const uint64_t vis = visible<TREE>(a, s, my_token(), p);
      for (int t = 0; t < kTileKeys; ++t) {
        const uint16_t* src = (const uint16_t*)c.v + at * D + (t >> 3) * D * 8 + (t & 7);
        const bool sees = vis >> t & 1;
#pragma unroll
        for (int i = 0; i < kO; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const uint32_t x = src[(i * 32 + (r & 3) + 8 * (r >> 2) + 4 * half) * 8];
            o[i][r] += sees && (x & 0x7f80u) == 0x7f80u ? bf16_bits_to_f32(x) : 0.f;
          }
      }
    }
  };

  // tile t: at position p, in key and value buffer buf; tile t + 1: p1, its
  // keys in the other key buffer by the time of tile t
  int64_t at = 0, at1 = 0, at2 = 0;
  int p = find(begin, &at);
  int p1 = find(p + kTileKeys, &at1);
  int n = 0;  // the tile's number; its buffers are n & 1
  Raw raw = {};
  if (p < end) {
    // the first keys, values and second keys, all asked for at once
    Raw raw_v = {}, raw_k1 = {};
    load_k(at, 0, raw);
    load_v(at, 0, raw_v);
    if (p1 < end) load_k(at1, 1, raw_k1);
    if (I8) {
      land_k(0, 0, raw);
    } else if (p1 < end) {
      wait_vmem_but<2 * kLoads>();
    } else {
      wait_vmem_but<kLoads>();
    }
    lds_barrier();
    read_k(0, mine);
    scores(0, kQ);
    less_maximum(0, mine);
    mask_scores(mine, p);
    top = maximum();
    if (!kPairs) read_k(0, 1);
    if (I8) {
      land_v(0, raw_v);
      land_k(1, 1, raw_k1);
    }
  }
  auto tile_step = [&](auto buffer) __attribute__((always_inline)) {
    constexpr int buf = decltype(buffer)::value;
    wait_vmem();
    lds_barrier();
    const float scale = I8 ? lds.vs[buf][lane] : 0.f;
    __builtin_amdgcn_sched_barrier(0);
    const int p2 = find(p1 + kTileKeys, &at2);
    if (p1 < end) load_v(at1, buf ^ 1, raw);
    if (p + kTileKeys > open) clean(buf, p);
    // Each group of LDS reads is issued behind the first product that waits for
    // the group before it (the wait is for all that are under way), and the
    // scheduler must not move it.
#pragma unroll
    for (int sub = 0; sub < 2; ++sub) {
      rescale(p, scale);
      const f32x16 x = st;
      scores(0, 1);  // of half tile 1 here, or 0 of the next tile
      __builtin_amdgcn_sched_barrier(0);
      read_v(buf, sub, 0, kVAhead);
      __builtin_amdgcn_sched_barrier(0);
      scores(1, kQ);
      weights(x, buf, sub);
      __builtin_amdgcn_sched_barrier(0);
      if (kVAhead == 1) {
        products(0, 1);
        __builtin_amdgcn_sched_barrier(0);
        read_v(buf, sub, 1, 2);
        __builtin_amdgcn_sched_barrier(0);
        products(1, kO);
        __builtin_amdgcn_sched_barrier(0);
      }
      constexpr int kDone = kVAhead == 1 ? kO : 0;
      products(kDone, kDone + 1);
      __builtin_amdgcn_sched_barrier(0);
      read_k(buf ^ 1, sub);
      __builtin_amdgcn_sched_barrier(0);
      products(kDone + 1, 2 * kO);
      less_maximum(n + sub, sub ^ 1);
      top = maximum();
      if (mask_scores(sub ^ 1, sub ? p1 : p)) top = maximum();
      if (sub == 0) {
        if (I8) land_v(buf ^ 1, raw);
        if (p2 < end) load_k(at2, buf, raw);
      }
    }
    if (I8) land_k(buf, n + 2, raw);
    ++n;
    p = p1;
    p1 = p2;
    at1 = at2;
  };
  Raw raw_k = {};
  // The same for a pair: one half tile of each tile, whose keys for the next
  // tile are read at its start.
  auto pair_step = [&](auto buffer) __attribute__((always_inline)) {
    constexpr int buf = decltype(buffer)::value;
    wait_vmem();
    lds_barrier();
    const float scale = I8 ? lds.vs[buf][lane] : 0.f;
    __builtin_amdgcn_sched_barrier(0);
    const int p2 = find(p1 + kTileKeys, &at2);
    if (p1 < end) load_v(at1, buf ^ 1, raw);
    if (p2 < end) load_k(at2, buf, raw_k);
    if (p + kTileKeys > open) clean(buf, p);
    rescale(p, scale);
    const f32x16 x = st;
    __builtin_amdgcn_sched_barrier(0);
    if (!I8) read_k(buf ^ 1, mine);
    weights(x, buf, mine);
    if (I8) read_k(buf ^ 1, mine);
    scores(0, kQ);  // of the next tile
    __builtin_amdgcn_sched_barrier(0);
    read_v(buf, mine, 0, 1);
    products(0, kO);
    __builtin_amdgcn_sched_barrier(0);
    read_v(buf, mine, 1, 2);
    products(kO, 2 * kO);
    less_maximum(n + 1, mine);
    top = maximum();
    if (mask_scores(mine, p1)) top = maximum();
    if (I8) {
      land_v(buf ^ 1, raw);
      land_k(buf, n + 2, raw_k);
    }
    ++n;
    p = p1;
    p1 = p2;
    at1 = at2;
  };
  auto step = [&](auto buffer) __attribute__((always_inline)) {
    if constexpr (kPairs)
      pair_step(buffer);
    else
      tile_step(buffer);
  };
  while (p < end) {
    step(std::integral_constant<int, 0>{});
    if (p >= end) break;
    step(std::integral_constant<int, 1>{});
  }
  l = add_xor32(l);
  if (kEvens) {
    exact = add_xor32(exact);
    const float by = even_by(exact, I8 ? add_xor32(rounded) : l);
    if (!I8) l = exact;
#pragma unroll
    for (int i = 0; i < kO; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[i][r] *= by;
  }
  if (kPairs) {  // the second pair's results, added to the first's (whose keys and values are read)
    float* const s_o = (float*)lds.k + (wave & 1) * (D / 2) * 64 + lane;
    float* const s_ml = (float*)lds.v + (wave & 1) * 128 + lane;
    m = limit >= 0.f ? m : kUnseen;
    lds_barrier();
    if (wave >= 2) {
#pragma unroll
      for (int i = 0; i < kO; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) s_o[(i * 16 + r) * 64] = o[i][r];
      s_ml[0] = m;
      s_ml[64] = l;
    }
    lds_barrier();
    if (wave >= 2) return;
    const float m2 = s_ml[0], both = fmaxf(m, m2);
    const float f = factor(m, both), f2 = factor(m2, both);
    m = both;
    limit = m > kUnseen ? 0.f : limit;
    l = l * f + s_ml[64] * f2;
#pragma unroll
    for (int i = 0; i < kO; ++i) {
#pragma unroll
      for (int r = 0; r < 16; ++r) o[i][r] = o[i][r] * f + s_o[(i * 16 + r) * 64] * f2;
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  if (!I8 && odd_from < end) add_odd();
  const int out_row = my_row();
  if (out_row >= rows) return;
  if (row_end > part.chunk) {  // the join adds the parts
    const int64_t to = part.row(tile, h, HK, split, out_row - r0);
#pragma unroll
    for (int i = 0; i < kO; ++i)
#pragma unroll
      for (int r = 0; r < 16; r += 4)
        *(f32x4*)(part.o + to * D + i * 32 + 8 * (r >> 2) + 4 * half) =
            f32x4{o[i][r], o[i][r + 1], o[i][r + 2], o[i][r + 3]};
    if (half == 0) {
      part.ml[2 * to] = row_sees() ? m : kUnseen;
      part.ml[2 * to + 1] = l;
    }
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  const int out_token = out_row / G;
  if (STATS && half == 0)
    keep_stats(a, s.first + out_token, h * G + out_row - out_token * G, row_sees() ? m : kUnseen, l);
  uint16_t* out = a.out + ((int64_t)(s.first + out_token) * a.heads + h * G + (out_row - out_token * G)) * D;
#pragma unroll
  for (int i = 0; i < kO; ++i)
#pragma unroll
    for (int r = 0; r < 16; r += 4)
      *(u32x2*)(out + i * 32 + 8 * (r >> 2) + 4 * half) =
          u32x2{pack_pair(o[i][r] * inv, o[i][r + 1] * inv), pack_pair(o[i][r + 2] * inv, o[i][r + 3] * inv)};
}

// ---------------------------------------------------------------------------
// Row form: up to 16 rows of a sequence (the G heads of a decode step's token),
// where reading keys and values is all there is.  The workgroup's waves
// take steps of 32 (bf16) or 64 (int8) tokens in turn, 16 KB of D = 128, and
// load them straight into the operands of 16x16x32 matrix instructions, one
// step ahead: no LDS (but for int8's scales, which go through the wave's own)
// and no barrier until the waves' results are added.
//   S^T = K . Q^T, O^T = V^T . P^T as in the tile form: key row r of tile t is
//   token (r / 4) KS / 4 + 4 t + r % 4 of the step, so that a lane's scores are
//   the KS / 4 consecutive tokens that it must supply as P^T and whose values
//   lie in the 16 bytes that it loads.
// Weights are rounded to bf16 once, as in the tile form; kept as a pair of bf16
// (twice the products) they made the batch below 6 % slower for an error of
// 0.0017 instead of 0.0022, of which the output's rounding alone is 0.0017.
//
// Bound by HBM for batches: 16 x 16384 tokens, 32 / 8 heads, bf16 192 us, 5.6
// TB/s; 64 sequences of up to 8192, 32 / 4 heads, int8 75 us, 4.7 TB/s (the
// vector unit busy 28 %, the rest lost to sequences of unequal length).  One
// sequence of 517 tokens takes 9.1 us in four workgroups: 4.7 of launch, first
// loads and the waves' sum, the rest reading at 61 GB/s each (the slope from 517
// to 2000 tokens in one workgroup per key head; int8 46).
// ---------------------------------------------------------------------------
template <int D, bool I8, bool TREE, bool STATS>
__global__ __launch_bounds__(256, 2) void attn_row_kernel(CacheView c, AttnArgs a, Parts part) {
  constexpr int KS = I8 ? 64 : 32;  // tokens per step
  constexpr int NT = KS / 16;       // key tiles per step
  constexpr int KL = I8 ? D / 64 : D / 32;  // 16-byte loads per key row and lane
  constexpr int kO = D / 16;
  constexpr int kNext = 4 * KS;  // from a wave's step to its next
  constexpr int kPad = D + 4;
  __shared__ __align__(16) float s_o[4][kRowRows][kPad];
  __shared__ float s_m[4][kRowRows], s_l[4][kRowRows];
  __shared__ __align__(16) float s_scale[I8 ? 4 : 1][2][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int g = lane >> 4, col = lane & 15;
  const int HK = c.kv_heads, G = a.heads / HK;
  const int h = (int)(blockIdx.x % (unsigned)HK);
  const int rest = (int)(blockIdx.x / (unsigned)HK);
  const int split = rest % part.splits;
  const int b = rest / part.splits;
  const int begin = split * part.chunk;
  // 64 entries of the page table, one per lane: all that a chunk needs (asked
  // for before anything is known of the sequence)
  const int page0 = begin >> c.page_shift;
  const int pages = table_entries(a, b, page0, lane);
  const Seq s = sequence(c, a, b, sequence_words(a, b), h == 0 && split == 0 && tid == 0);
  const int rows = s.n * G;
  if (rows == 0) return;
  const int row_end = end_of_rows<TREE>(s, G, 0, kRowRows);
  if (split > 0 && begin >= row_end) return;
  const int end = row_end - begin > part.chunk ? begin + part.chunk : row_end;
  const int row = col < rows ? col : rows - 1;
  const int token = row / G;
  const uint16_t* q = a.q + ((int64_t)(s.first + token) * a.heads + h * G + (row - token * G)) * D;
  u32x4 qf[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
    qf[i] = *(const u32x4*)(q + (I8 ? (i >> 1) * 64 + g * 16 + (i & 1) * 8 : i * 32 + g * 8));
  const int open = TREE ? s.context : s.context + 1;  // positions below are seen by all rows

  f32x4 o[kO];
#pragma unroll
  for (int i = 0; i < kO; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = kUnseen, l = 0.f, above = I8 ? 0.f : kSlack;
  // Beside the weights of cached tokens: the sum of weights (int8: x scale) before they are
  // rounded to bf16 for the product and after it; the quotient takes what the roundings have in
  // common out of the output.
  constexpr bool kEvens = STATS;
  float exact = 0.f, rounded = 0.f;  // (exact: int8; else that is l)
  const float scale2 = a.scale * kLog2e;
  const int mask = (1 << c.page_shift) - 1;
  const int krow = (col >> 2) * (KS / 4) + (col & 3);

  struct Step {
    u32x4 k[NT * KL], v[kO];
    float ks, vs;  // int8: lane's token
    bool ok;       // the page is in the cache
    int64_t at;    // its first token's place
  };
  // (where there is no such step, every lane asks for the same 16 bytes of the
  // last one: loads behind a branch would make the waits for the step before
  // them wait for these as well)
  auto load = [&](int p, Step& x) {
    const bool real = p < end;
    const int page = __builtin_amdgcn_readlane(pages, ((real ? p : end - 1) >> c.page_shift) - page0);
    x.ok = page >= 0 && page < c.num_pages;
    x.at = (((int64_t)(x.ok ? page : 0) * HK + h) << c.page_shift) + (real ? p & mask : 0);
    const uint8_t* kb = c.k + x.at * (D * (I8 ? 1 : 2)) + (real ? krow * (D * (I8 ? 1 : 2)) + g * 16 : 0);
    const uint8_t* vb = c.v + x.at * (D * (I8 ? 1 : 2)) + (real ? (g * D + col) * 16 : 0);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < KL; ++i) x.k[t * KL + i] = *(const u32x4*)(kb + t * 4 * (D * (I8 ? 1 : 2)) + i * 64);
    if (I8) {
      x.ks = c.k_scales[x.at + lane];
      x.vs = c.v_scales[x.at + lane];
    }
#pragma unroll
    for (int i = 0; i < kO; ++i) x.v[i] = *(const u32x4*)(vb + i * 256);
  };
  auto compute = [&](int p, Step& x) {
    if (I8) {
      // the codes become bf16 here, not where they are loaded (four times the registers)
#pragma unroll
      for (int i = 0; i < NT * KL; ++i) __asm__ volatile("" : "+v"(x.k[i]));
    }
    f32x4 st[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      st[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < KL; ++i) {
        if (!I8) {
          st[t] = mfma_bf16(x.k[t * KL + i], qf[i], st[t]);
        } else {
          u32x4 lo, hi;
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            uint32_t e0, e1;
            bf16_of_codes(x.k[t * KL + i][w], &e0, &e1);
            lo[2 * w] = e0, lo[2 * w + 1] = e1;
            bf16_of_codes(x.k[t * KL + i][w + 2], &e0, &e1);
            hi[2 * w] = e0, hi[2 * w + 1] = e1;
          }
          st[t] = mfma_bf16(lo, qf[2 * i], st[t]);
          st[t] = mfma_bf16(hi, qf[2 * i + 1], st[t]);
        }
      }
      // (one tile's bf16 operands at a time: hoisted together they spill)
      if (I8) __builtin_amdgcn_sched_barrier(0);
    }
    if (I8) {
      // the lane's tokens' scales, by way of the wave's own LDS
      s_scale[wave][0][lane] = x.ks * scale2;
      s_scale[wave][1][lane] = x.vs;
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const f32x4 f = *(const f32x4*)&s_scale[wave][0][g * 16 + t * 4];
#pragma unroll
        for (int r = 0; r < 4; ++r) st[t][r] = rounded_product(st[t][r], f[r]);
      }
    } else {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) st[t][r] = rounded_product(st[t][r], scale2);
    }
    const int valid = x.ok ? s.len - p : 0;  // tokens of the step that exist
    const bool masks = p + KS > open || valid < KS;
    uint32_t vis = ~0u;
    uint64_t bits = 0;
    bool odd = false;
    if (masks) {
      bits = visible<TREE>(a, s, token, p);
      if (valid < KS) bits &= (1ull << valid) - 1;
      vis = (uint32_t)(bits >> (g * (KS / 4)));
      if (!x.ok && lane == 0) report(c.status, kBadPage);
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) st[t][r] = vis >> (t * 4 + r) & 1 ? st[t][r] : -__builtin_huge_valf();
      if (!I8) {
        // values past the end become zero; so do those that are not finite, which
        // some row may not see (0 x NaN): the rows that do get them below
        const int inside = valid - g * 8;
#pragma unroll
        for (int i = 0; i < kO; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t keep = (2 * j < inside ? 0xffffu : 0u) | (2 * j + 1 < inside ? 0xffff0000u : 0u);
            x.v[i][j] &= keep;
            odd |= non_finite_pair(x.v[i][j]);
          }
        odd = __any(odd);
        if (odd) {
#pragma unroll
          for (int i = 0; i < kO; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if ((x.v[i][j] & 0x7f80u) == 0x7f80u) x.v[i][j] &= 0xffff0000u;
              if ((x.v[i][j] & 0x7f800000u) == 0x7f800000u) x.v[i][j] &= 0xffffu;
            }
        }
      }
    }
    if (STATS && a.scores && col < rows) {
      float* to = a.scores + (((int64_t)b * HK + h) * part.rows + col) * a.score_row + p + g * (KS / 4);
#pragma unroll
      for (int t = 0; t < NT; ++t) *(f32x4*)(to + t * 4) = st[t];
    }
    float top = st[0][0];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) top = fmaxf(top, st[t][r]);
    top = max_xor32(max_xor16(top));
    const bool moves = top > m + (kSlack - above);
    if (__any(moves || (I8 && x.vs > kLargeScale))) {
      float up = 0.f;
      if (I8) {
        const uint64_t large = __ballot(x.vs > kLargeScale);
        up = above == 0.f && ((masks ? bits : ~0ull) & large) ? kSlack : 0.f;
        above += up;
      }
      const float to = moves ? top + above : m + up;
      const float fix = to > kUnseen ? __builtin_amdgcn_exp2f(m - to) : 1.f;
      m = to;
      l *= fix;
      if (kEvens && I8) exact *= fix;
      if (kEvens) rounded *= fix;
#pragma unroll
      for (int i = 0; i < kO; ++i) o[i] *= fix;
    }
    if (odd) {  // (past the rescale: infinity x 0)
      for (int t = 0; t < KS && t < valid; ++t) {
        const uint16_t* src = (const uint16_t*)c.v + x.at * D + (t >> 3) * D * 8 + (t & 7);
        const bool sees = bits >> t & 1;
#pragma unroll
        for (int i = 0; i < kO; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const uint32_t e = src[(i * 16 + g * 4 + r) * 8];
            o[i][r] += sees && (e & 0x7f80u) == 0x7f80u ? bf16_bits_to_f32(e) : 0.f;
          }
      }
    }
    const float less = fmaxf(m, -__FLT_MAX__);  // (a number: scores of -infinity have a weight of 0)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        st[t][r] = __builtin_amdgcn_exp2f(st[t][r] - less);
        l += st[t][r];
      }
    if (I8) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const f32x4 f = *(const f32x4*)&s_scale[wave][1][g * 16 + t * 4];
        // (an unseen value's scale may be anything: 0 x NaN)
#pragma unroll
        for (int r = 0; r < 4; ++r) st[t][r] = !masks || (vis >> (t * 4 + r) & 1) ? st[t][r] * f[r] : 0.f;
      }
      __builtin_amdgcn_wave_barrier();
    }
    u32x4 pf[NT / 2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      pf[t >> 1][2 * (t & 1)] = pack_pair(st[t][0], st[t][1]);
      pf[t >> 1][2 * (t & 1) + 1] = pack_pair(st[t][2], st[t][3]);
      if (kEvens && I8) exact += (st[t][0] + st[t][1]) + (st[t][2] + st[t][3]);
      if (kEvens) rounded = add_pair(pf[t >> 1][2 * (t & 1)], add_pair(pf[t >> 1][2 * (t & 1) + 1], rounded));
    }
#pragma unroll
    for (int i = 0; i < kO; ++i) {
      if (!I8) {
        o[i] = mfma_bf16(x.v[i], pf[0], o[i]);
      } else {
        __asm__ volatile("" : "+v"(x.v[i]));
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          u32x4 vf;
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            uint32_t e0, e1;
            bf16_of_codes(x.v[i][2 * j + w], &e0, &e1);
            vf[2 * w] = e0, vf[2 * w + 1] = e1;
          }
          o[i] = mfma_bf16(vf, pf[j], o[i]);
        }
        if (i & 1) __builtin_amdgcn_sched_barrier(0);
      }
    }
  };

  Step x0, x1;
  int p = begin + wave * KS;
  if (p < end) load(p, x0);
  while (p < end) {
    load(p + kNext, x1);
    compute(p, x0);
    p += kNext;
    if (p >= end) break;
    load(p + kNext, x0);
    compute(p, x1);
    p += kNext;
  }

  // the waves' results, added in order
  l = add_xor32(add_xor16(l));
  if (kEvens) {
    const float by = even_by(I8 ? add_xor32(add_xor16(exact)) : l, add_xor32(add_xor16(rounded)));
#pragma unroll
    for (int i = 0; i < kO; ++i) o[i] *= by;
  }
  if (g == 0) {
    s_m[wave][col] = m;
    s_l[wave][col] = l;
  }
#pragma unroll
  for (int i = 0; i < kO; ++i) *(f32x4*)&s_o[wave][col][i * 16 + g * 4] = o[i];
  __syncthreads();
  const int r = tid >> 4, d0 = (tid & 15) * (D / 16);
  if (r >= rows) return;
  float top = s_m[0][r];
#pragma unroll
  for (int w = 1; w < 4; ++w) top = fmaxf(top, s_m[w][r]);
  float sum = 0.f, out[D / 16];
#pragma unroll
  for (int d = 0; d < D / 16; ++d) out[d] = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float f = factor(s_m[w][r], top);
    sum += s_l[w][r] * f;
#pragma unroll
    for (int d = 0; d < D / 16; ++d) out[d] += s_o[w][r][d0 + d] * f;
  }
  if (row_end > part.chunk) {
    const int64_t at = part.row(b, h, HK, split, r);
#pragma unroll
    for (int d = 0; d < D / 16; d += 4)
      *(f32x4*)(part.o + at * D + d0 + d) = f32x4{out[d], out[d + 1], out[d + 2], out[d + 3]};
    if (d0 == 0) {
      part.ml[2 * at] = top;
      part.ml[2 * at + 1] = sum;
    }
    return;
  }
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
  const int tok = r / G;
  if (STATS && d0 == 0) {
    if (a.scores) {
      const int64_t at = part.row(b, h, HK, 0, r);
      part.ml[2 * at] = top;
      part.ml[2 * at + 1] = sum;
    } else {
      keep_stats(a, s.first + tok, h * G + r - tok * G, top, sum);
    }
  }
  uint16_t* dst = a.out + ((int64_t)(s.first + tok) * a.heads + h * G + (r - tok * G)) * D + d0;
#pragma unroll
  for (int d = 0; d < D / 16; d += 4)
    *(u32x2*)(dst + d) = u32x2{pack_pair(out[d] * inv, out[d + 1] * inv), pack_pair(out[d + 2] * inv, out[d + 3] * inv)};
}

// Adds the splits of an item's rows.  A workgroup takes 16 / SP rows at a time,
// each by SP x 16 threads: thread group i the splits i, i + SP, ... in order,
// then the groups in order (the same sums whatever the batch).  A launch of its
// own, so that no counter has to outlive a call: 4 us for few rows (latency), 21
// for the chunks above (2500 tokens x 32 heads in three parts).
template <int D, bool TREE, int ROWS, int SP>
__device__ __forceinline__ void join_rows(const CacheView& c, const AttnArgs& a, const Parts& part, int row_blocks) {
  constexpr int kRows = 16 / SP, kN = D / 16;
  __shared__ float s_m[16], s_l[16];
  __shared__ __align__(16) float s_o[16][SP > 1 ? D : 4];
  const int tid = threadIdx.x, lane = tid & 63;
  const int HK = c.kv_heads, G = a.heads / HK;
  const int h = (int)(blockIdx.x % (unsigned)HK);
  const int rest = (int)(blockIdx.x / (unsigned)HK);
  const int item = rest / row_blocks;
  const int b = part.whole ? item : sequence_of_tile(a, G, item, lane);
  const SeqWords words = sequence_words(a, b);
  const int block = part.whole ? 0 : block_of_tile(a, G, item, b, words);
  const Seq s = sequence(c, a, b, words, false);
  const int rows = s.n * G, r0 = block * ROWS;
  if (block < 0 || r0 >= rows) return;
  const int row_end = end_of_rows<TREE>(s, G, r0, ROWS);
  if (row_end <= part.chunk) return;
  const int splits = (row_end + part.chunk - 1) / part.chunk;
  const int used = rows - r0 < ROWS ? rows - r0 : ROWS;
  const int group = tid >> 4, d0 = (tid & 15) * kN;
  const int sp = group % SP;
  for (int base = rest % row_blocks * kRows; base < used; base += row_blocks * kRows) {
    const int r = base + group / SP;
    float m = kUnseen, l = 0.f, out[kN];
#pragma unroll
    for (int d = 0; d < kN; ++d) out[d] = 0.f;
    for (int i = sp; i < splits && r < used; i += SP) {
      const int64_t at = part.row(item, h, HK, i, r);
      const float mi = part.ml[2 * at], li = part.ml[2 * at + 1];
      const float to = fmaxf(m, mi);
      const float f = factor(m, to), fi = factor(mi, to);
      m = to;
      l = l * f + li * fi;
#pragma unroll
      for (int d = 0; d < kN; d += 4) {
        const f32x4 x = *(const f32x4*)(part.o + at * D + d0 + d);
#pragma unroll
        for (int j = 0; j < 4; ++j) out[d + j] = out[d + j] * f + x[j] * fi;
      }
    }
    if (SP > 1) {
      __syncthreads();  // (of the rows before, the sums are read)
      if ((tid & 15) == 0) {
        s_m[group] = m;
        s_l[group] = l;
      }
#pragma unroll
      for (int d = 0; d < kN; d += 4)
        *(f32x4*)&s_o[group][SP > 1 ? d0 + d : 0] = f32x4{out[d], out[d + 1], out[d + 2], out[d + 3]};
      __syncthreads();
      if (sp == 0) {
#pragma unroll
        for (int i = 1; i < SP; ++i) m = fmaxf(m, s_m[group + i]);
        l = 0.f;
#pragma unroll
        for (int d = 0; d < kN; ++d) out[d] = 0.f;
#pragma unroll
        for (int i = 0; i < SP; ++i) {
          const float f = factor(s_m[group + i], m);
          l += s_l[group + i] * f;
#pragma unroll
          for (int d = 0; d < kN; ++d) out[d] += s_o[group + i][SP > 1 ? d0 + d : 0] * f;
        }
      }
    }
    if (sp == 0 && r < used) {
      const float inv = l == 0.f ? 0.f : 1.0f / l;
      const int tok = (r0 + r) / G;
      if (a.stats && d0 == 0) keep_stats(a, s.first + tok, h * G + r0 + r - tok * G, m, l);
      uint16_t* dst = a.out + ((int64_t)(s.first + tok) * a.heads + h * G + (r0 + r - tok * G)) * D + d0;
#pragma unroll
      for (int d = 0; d < kN; d += 4)
        *(u32x2*)(dst + d) =
            u32x2{pack_pair(out[d] * inv, out[d + 1] * inv), pack_pair(out[d + 2] * inv, out[d + 3] * inv)};
    }
  }
}

template <int D, bool TREE, int ROWS, int SP>
__global__ __launch_bounds__(256) void join_kernel(CacheView c, AttnArgs a, Parts part, int row_blocks) {
  join_rows<D, TREE, ROWS, SP>(c, a, part, row_blocks);
}

// ---------------------------------------------------------------------------
// The weights of cached tokens from the scores that the row form kept, beside the
// join of its parts where there are any: 1024 tokens per workgroup behind the
// join's.  Scores are 4 bytes per row where the keys are 2 D or D: reading them
// back costs a batch less than the keys once more (64 sequences of up to 8192
// tokens, 32 / 4 heads, int8: 93 us of attention that keeps them, 78 without, and 15
// here; the keys once more and the rows' statistics 80).
// ---------------------------------------------------------------------------
constexpr int kWeighTokens = 1024;

template <int D, int SP>
__global__ __launch_bounds__(256) void join_weigh_kernel(CacheView c, WeighArgs w, Parts part, int row_blocks,
                                                         int join_groups) {
  const AttnArgs& a = w.attn;
  if ((int)blockIdx.x < join_groups) {
    join_rows<D, false, kRowRows, SP>(c, a, part, row_blocks);
    return;
  }
  __shared__ float s_m[kRowRows], s_inv[kRowRows];
  const int HK = c.kv_heads, G = a.heads / HK;
  const int tid = threadIdx.x;
  const unsigned index = blockIdx.x - join_groups;
  const int h = (int)(index % (unsigned)HK);
  const int rest = (int)(index / (unsigned)HK);
  const int b = rest / w.blocks;
  const int p = rest % w.blocks * kWeighTokens + tid * 4;
  const Seq s = sequence(c, a, b, sequence_words(a, b), false);
  const int rows = s.n * G;
  if (rows == 0 || rest % w.blocks * kWeighTokens >= s.len) return;
  const int row_end = end_of_rows<false>(s, G, 0, kRowRows);
  const int splits = row_end > part.chunk ? (row_end + part.chunk - 1) / part.chunk : 1;
  const int first = s.n > w.last ? (s.n - w.last) * G : 0;
  // a row's statistics by 16 lanes: lane i the parts i, i + 16, ...
  const int r = tid >> 4, lane = tid & 15;
  float m = kUnseen, l = 0.f;
  for (int i = lane; i < splits && r < rows; i += 16) {
    const int64_t at = part.row(b, h, HK, i, r);
    const float mi = part.ml[2 * at], li = part.ml[2 * at + 1];
    const float to = fmaxf(m, mi);
    l = l * factor(m, to) + li * factor(mi, to);
    m = to;
  }
#pragma unroll
  for (int off = 8; off >= 1; off >>= 1) {
    const float mi = __shfl_xor(m, off), li = __shfl_xor(l, off);
    const float to = fmaxf(m, mi);
    l = l * factor(m, to) + li * factor(mi, to);
    m = to;
  }
  if (lane == 0) {
    s_m[r] = fmaxf(m, -__FLT_MAX__);  // (a number: scores of -infinity have a weight of 0)
    s_inv[r] = l == 0.f ? 0.f : 1.0f / l;
  }
  __syncthreads();
  if (p >= s.len) return;
  const float* scores = a.scores + ((int64_t)b * HK + h) * part.rows * a.score_row + p;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  for (int i = first; i < rows; ++i) {
    const f32x4 x = *(const f32x4*)(scores + (int64_t)i * a.score_row);
    const float less = s_m[i], inv = s_inv[i];
    const int past = s.context + i / G - p;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // (a row of NaN reaches what it sees only)
      const float e = __builtin_amdgcn_exp2f(x[j] - less);
      sum[j] = j <= past ? __builtin_fmaf(e, inv, sum[j]) : sum[j];
    }
  }
  float* to = w.weights + b * w.seq_stride + h * w.head_stride + p;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (p + j < s.len) to[j] += sum[j];
}

// The launch of a forward call: by what the caller knows without asking the
// device (its rows and bounds).
struct Plan {
  bool row_form;
  Parts part;
};

Plan plan_of(const CacheView& c, int heads, int tokens, int seqs, int max_queries, int max_len) {
  Plan p = {};
  const int64_t G = heads / c.kv_heads;
  p.row_form = max_queries * G <= kRowRows;
  const int tile_rows = max_queries * G <= kPairRows ? kPairRows : kTileRows;
  p.part.rows = p.row_form ? (int)(max_queries > 0 ? max_queries * G : G) : tile_rows;
  p.part.whole = p.row_form || max_queries * G <= tile_rows;
  p.part.items = (int)(p.part.whole ? seqs : tokens * G / tile_rows + seqs);
  if (p.part.items < 1) p.part.items = 1;
  const int64_t wgs = (int64_t)p.part.items * c.kv_heads;
  int64_t splits = 1, least = 256, most = (int64_t)1 << 30;
  if (p.row_form) {
    // One workgroup reads about 61 GB/s, 100 of them what HBM gives: fewer
    // share the contexts (one request, bf16, D = 128, in us: 800 tokens 8.5
    // against 10.4, 1000 9.2 against 12.8, 2000 9.5 against 21.6).  Up to 640
    // tokens they do not: both launches take 0.5 less there than the one (517
    // tokens 8.6 against 9.1, 640 8.4 against 9.0; 257 8.3 against 6.9), but the
    // second costs the host 4 in a call outside of a graph (14.8 against 10.7).
    // More only split what would run on after the others: chunks of
    // 2048 against 4096 tokens, 32 x 4000 tokens 52 against 60; over two
    // rounds of workgroups chunks of 4096, the most that a wave holds page
    // numbers for.
    if (wgs < 100 && max_len > 640) splits = (256 + wgs - 1) / wgs;
    most = wgs <= 1024 ? 2048 : 4096;
  } else if (wgs < 512) {
    // About one and a half rounds of workgroups (two run on a CU at a time);
    // in us, for 512, 768 and 1536 of them: 1000 tokens bf16 33, 31, 42; four
    // drafts of 32 on 8000 tokens 41, 39, 52.  One round where the items are
    // counted, not bounded: 32 drafts of 8 on 4000 tokens, 32 / 4 heads, bf16 60
    // for 512, 71 for 768.  Parts of fewer than 256 tokens
    // cost more than they give (512 tokens 20, in parts of 128 24), but for the
    // least launches (a draft of 12 on 500 tokens 13.5, in parts of 128 11.5).
    splits = ((p.part.whole ? 512 : 768) + wgs / 2) / wgs;
    if (wgs <= 64) least = 128;
  } else if (wgs < 1536 && max_len >= 4096) {
    // Up to three rounds of long ones: parts even out the last round (chunks
    // of 1021 on up to 9000 tokens, int8, 648 workgroups: 494 us, in three
    // parts 440); short ones lose by it (8 x 512 tokens 41 us, in two parts 72).
    splits = (1536 + wgs - 1) / wgs;
  }
  int64_t chunk = (max_len + splits - 1) / splits;
  chunk = chunk < most ? chunk : most;
  chunk = (chunk + least - 1) / least * least;
  if (chunk < least) chunk = least;
  p.part.chunk = (int)chunk;
  p.part.splits = max_len > chunk ? (int)((max_len + chunk - 1) / chunk) : 1;
  return p;
}

size_t plan_rows(const CacheView& c, const Plan& p) {
  return p.part.splits > 1 ? (size_t)p.part.items * c.kv_heads * p.part.splits * p.part.rows : 0;
}

// Workgroups per item and head of the join, and its thread groups per row:
// several for a row's splits while workgroups are few; most of many would find
// nothing to do (a workgroup that does costs about 2 us).  Whole calls in us, the
// row form with 4 and 16 groups: 4 splits (1000 tokens) 9.2 and 9.4 (of 16
// sequences of 4000 28.3 and 29.0), 8 (2000) 9.9 and 9.7, 16 (4000) 10.2 and 9.5,
// 32 (8000) 12.0 and 10.2.  The tile form with 4 and 1: 4 items x heads (a draft
// of 12 on 2000) 13.7 and 23.9, 32 (8 of 8 on 4000) 24.6 and 32.4, 96 (24 of 8)
// 43.0 and 43.2, 132 (a prompt of 512) 22.4 and 19.3, 252 (of 1000) 39.8 and 31.9.
struct JoinPlan {
  int groups;
  int64_t row_blocks;
};
JoinPlan join_of(const CacheView& c, const Plan& p) {
  if (p.row_form && p.part.splits <= 8) return {4, (p.part.rows + 3) / 4};
  if (p.row_form) return {16, p.part.rows};
  if ((int64_t)p.part.items * c.kv_heads <= 64) return {4, p.part.rows / 4};
  return {1, 2};
}

}  // namespace

int64_t attn_workgroups(const CacheView& c, int heads, int tokens, int seqs, int max_queries, int max_len) {
  const Plan p = plan_of(c, heads, tokens, seqs, max_queries, max_len);
  const int64_t items = (int64_t)p.part.items * c.kv_heads;
  const int64_t join = p.part.splits > 1 ? join_of(c, p).row_blocks : 0;
  return items * (p.part.splits > join ? p.part.splits : join);
}

size_t attn_workspace_bytes(const CacheView& c, int heads, int tokens, int seqs, int max_queries, int max_len) {
  return plan_rows(c, plan_of(c, heads, tokens, seqs, max_queries, max_len)) * (c.dim + 2) * sizeof(float);
}

namespace {

// Floats of the workspace: the parts' outputs, maxima and sums, then the scores.
struct ScoresPlan {
  size_t o, ml, scores;
  int score_row;
};
ScoresPlan scores_plan(const CacheView& c, const Plan& p, int max_len) {
  ScoresPlan x = {};
  const size_t rows = (size_t)p.part.items * c.kv_heads * p.part.splits * p.part.rows;
  x.o = p.part.splits > 1 ? rows * c.dim : 0;
  x.ml = (rows * 2 + 3) / 4 * 4;
  x.score_row = (max_len + 63) / 64 * 64;
  x.scores = (size_t)p.part.items * c.kv_heads * p.part.rows * x.score_row;
  return x;
}

}  // namespace

size_t attn_scores_workspace_bytes(const CacheView& c, int heads, int tokens, int seqs, int max_queries, int max_len) {
  const Plan p = plan_of(c, heads, tokens, seqs, max_queries, max_len);
  const ScoresPlan x = scores_plan(c, p, max_len);
  const int64_t groups = (int64_t)p.part.items * c.kv_heads *
                         ((max_len + kWeighTokens - 1) / kWeighTokens + (p.part.splits > 1 ? join_of(c, p).row_blocks : 0));
  if (!p.row_form || x.scores * sizeof(float) > ((size_t)1 << 30) || groups >= (int64_t)1 << 24) return 0;
  return (x.o + x.ml + x.scores) * sizeof(float);
}

hipError_t launch_attn_scores(const CacheView& c, WeighArgs w, void* workspace, hipStream_t stream) {
  AttnArgs& a = w.attn;
  Plan p = plan_of(c, a.heads, a.tokens, a.seqs, a.max_queries, a.max_len);
  const ScoresPlan x = scores_plan(c, p, a.max_len);
  p.part.o = (float*)workspace;
  p.part.ml = p.part.o + x.o;
  a.scores = p.part.ml + x.ml;
  a.score_row = x.score_row;
  w.blocks = (a.max_len + kWeighTokens - 1) / kWeighTokens;
  const int64_t items = (int64_t)p.part.items * c.kv_heads;
  const JoinPlan j = join_of(c, p);
  const int join_groups = p.part.splits > 1 ? (int)(items * j.row_blocks) : 0;
  const dim3 grid((unsigned)(items * p.part.splits)), after((unsigned)(join_groups + items * w.blocks));
  by_layout(c, [&](auto dim, auto int8) {
    constexpr int D = decltype(dim)::value;
    constexpr bool I8 = decltype(int8)::value;
    hipLaunchKernelGGL((attn_row_kernel<D, I8, false, true>), grid, dim3(256), 0, stream, c, a, p.part);
    if (after.x == 0) return;
    if (j.groups == 4)
      hipLaunchKernelGGL((join_weigh_kernel<D, 4>), after, dim3(256), 0, stream, c, w, p.part, (int)j.row_blocks,
                         join_groups);
    else
      hipLaunchKernelGGL((join_weigh_kernel<D, 16>), after, dim3(256), 0, stream, c, w, p.part, (int)j.row_blocks,
                         join_groups);
  });
  return hipGetLastError();
}

hipError_t launch_attn(const CacheView& c, const AttnArgs& a, void* workspace, hipStream_t stream) {
  Plan p = plan_of(c, a.heads, a.tokens, a.seqs, a.max_queries, a.max_len);
  p.part.o = (float*)workspace;
  p.part.ml = (float*)workspace + plan_rows(c, p) * c.dim;
  const dim3 grid((unsigned)((int64_t)p.part.items * c.kv_heads * p.part.splits));
  by_layout(c, [&](auto dim, auto int8) {
    constexpr int D = decltype(dim)::value;
    constexpr bool I8 = decltype(int8)::value;
    auto launch = [&](auto tree, auto keeps) {
      constexpr bool TREE = decltype(tree)::value, STATS = decltype(keeps)::value;
      if (p.row_form)
        hipLaunchKernelGGL((attn_row_kernel<D, I8, TREE, STATS>), grid, dim3(256), 0, stream, c, a, p.part);
      else if (p.part.rows == kPairRows)
        hipLaunchKernelGGL((attn_tile_kernel<D, I8, TREE, kPairRows, STATS>), grid, dim3(256), 0, stream, c, a, p.part);
      else
        hipLaunchKernelGGL((attn_tile_kernel<D, I8, TREE, kTileRows, STATS>), grid, dim3(256), 0, stream, c, a, p.part);
      if (p.part.splits == 1) return;
      const JoinPlan j = join_of(c, p);
      const dim3 join_grid((unsigned)(p.part.items * c.kv_heads * j.row_blocks));
      auto join = [&](auto rows, auto groups) {
        constexpr int ROWS = decltype(rows)::value, SP = decltype(groups)::value;
        hipLaunchKernelGGL((join_kernel<D, TREE, ROWS, SP>), join_grid, dim3(256), 0, stream, c, a, p.part,
                           (int)j.row_blocks);
      };
      const std::integral_constant<int, 1> one;
      const std::integral_constant<int, 4> four;
      const std::integral_constant<int, 16> sixteen;
      const std::integral_constant<int, kRowRows> row_form;
      const std::integral_constant<int, kPairRows> narrow;
      const std::integral_constant<int, kTileRows> tile;
      if (p.row_form)
        j.groups == 4 ? join(row_form, four) : join(row_form, sixteen);
      else if (p.part.rows == kPairRows)
        j.groups == 4 ? join(narrow, four) : join(narrow, one);
      else
        j.groups == 4 ? join(tile, four) : join(tile, one);
    };
    if (a.stats)  // (causal calls only)
      launch(std::false_type{}, std::true_type{});
    else if (a.tree)
      launch(std::true_type{}, std::false_type{});
    else
      launch(std::false_type{}, std::false_type{});
  });
  return hipGetLastError();
}

}  // namespace nkt
