// Attention over the paged cache.
#include "nkt_attn_device.h"

namespace nkt {

namespace {

// ---------------------------------------------------------------------------
// A sequence's rows are its n tokens x the G query heads that share a key /
// value head, token by token (row r: token r / G, head r % G), so keys and
// values are read once for all of them.
// ---------------------------------------------------------------------------
struct Seq {
  int first;    // row of q of its first token
  int n;        // tokens of it in this call
  int len;      // positions of it in the cache
  int context;  // position of its first token here (negative: more rows than tokens)
};

__device__ __forceinline__ Seq sequence(const CacheView& c, const AttnArgs& a, int b, bool reports) {
  Seq s;
  s.first = b;
  s.n = 1;
  bool bad = false;
  if (a.starts) {
    const int s0 = a.starts[b], s1 = a.starts[b + 1];
    s.first = s0 < 0 ? 0 : s0 > a.tokens ? a.tokens : s0;
    const int end = s1 > a.tokens ? a.tokens : s1;
    s.n = end > s.first ? end - s.first : 0;
    bad = s.n > a.max_queries;
  }
  const int len = a.lens[b];
  s.context = (len < 0 ? 0 : len) - s.n;
  if (s.n > a.max_queries) s.n = a.max_queries;
  const int64_t table = (int64_t)a.width << c.page_shift;
  const int most = table < a.max_len ? (int)table : a.max_len;
  s.len = len < 0 ? 0 : len > most ? most : len;
  if (reports && (bad || len < 0 || len > most)) report(c.status, kBadLength);
  return s;
}

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

__device__ __forceinline__ uint32_t pack_p(float lo, float hi) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, bf16x2));
}

typedef float f32x16 __attribute__((ext_vector_type(16)));

// 32x32x16 bf16: lane l supplies A[l%32][8*(l/32) .. +7] and B[8*(l/32) ..
// +7][l%32]; D[(v&3) + 8*(v>>2) + 4*(l/32)][l%32] lands in register v.
__device__ __forceinline__ f32x16 mfma32_bf16(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                 0);
}

__device__ __forceinline__ float max_xor32(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

__device__ __forceinline__ float max_xor16(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -1.0e38f;  // the running maximum before any score
// The running maximum moves only when a score passes it by this much (in
// log2): weights then reach 2^8 at most, which neither the fp32 sums nor a
// bf16 weight's relative precision notice, and most tiles skip the rescale.
constexpr float kSlack = 8.0f;

__device__ __forceinline__ bool non_finite_pair(uint32_t w) {
  return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
}

// int8 codes of one 32-bit word -> two words of bf16 (exact)
__device__ __forceinline__ void bf16_of_codes(uint32_t w, uint32_t* lo, uint32_t* hi) {
  const float f0 = (float)(int8_t)w, f1 = (float)(int8_t)(w >> 8), f2 = (float)(int8_t)(w >> 16),
              f3 = (float)(int8_t)(w >> 24);
  *lo = __builtin_amdgcn_perm(__float_as_uint(f1), __float_as_uint(f0), 0x07060302u);
  *hi = __builtin_amdgcn_perm(__float_as_uint(f3), __float_as_uint(f2), 0x07060302u);
}

constexpr int kTileRows = 128, kTileKeys = 64;  // of the tile form
constexpr int kRowRows = 16;                    // of the row form

// How a launch is cut: items (a tile of rows of one head) x splits (of chunk
// positions each).  Where an item's rows see more than one chunk, each split
// leaves its weighted sum of values (fp32, not divided), running maximum and
// sum in the workspace, and join_kernel adds them in order.
struct Parts {
  int items, splits, chunk;
  float* o;   // [items, kv_heads, splits, rows, D]
  float* ml;  // [items, kv_heads, splits, rows, 2]
  __device__ __forceinline__ int64_t row(int item, int h, int kv_heads, int split, int rows, int r) const {
    return (((int64_t)item * kv_heads + h) * splits + split) * rows + r;
  }
};

__device__ __forceinline__ int first_row(const AttnArgs& a, int b) { return a.starts ? a.starts[b] : b; }

// The sequence of a tile of kTileRows rows, and the tile's number in it (which
// may lie past its rows).  Sequence b's tiles start at starts[b] G / 128 + b,
// which ascends and leaves room for its ceil(n G / 128) tiles: the last b that
// starts at or before this tile, found by 64 lanes at a time.
__device__ __forceinline__ bool sequence_of_tile(const AttnArgs& a, int G, int tile, int lane, int* seq, int* block) {
  int b = 0;
  for (int n = a.seqs; n > 1;) {
    const int step = (n + 63) / 64;
    const int i = b + lane * step;
    const bool before =
        lane * step < n && (int64_t)first_row(a, i < a.seqs ? i : a.seqs - 1) * G / kTileRows + i <= tile;
    const int count = __popcll(__ballot(before));
    if (count == 0) return false;
    const int skip = (count - 1) * step;
    b += skip;
    n = n - skip < step ? n - skip : step;
  }
  *seq = __builtin_amdgcn_readfirstlane(b);
  *block = tile - ((int)((int64_t)first_row(a, *seq) * G / kTileRows) + *seq);
  return *block >= 0;
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
// Keys lie in LDS as rows of 16-byte chunks, chunk c of row r at c ^ (r & 7)
// (consecutive rows' same chunk in different banks); values as they come.
// bf16 tiles go straight from global memory into LDS, int8 ones through
// registers (exact bf16 integers; the scales multiply scores and weights).
// ---------------------------------------------------------------------------

template <int D, bool I8>
struct TileLds {
  __align__(16) uint8_t k[2][kTileKeys * D * 2];
  __align__(16) uint8_t v[2][kTileKeys * D * 2];
  __align__(16) float ks[2][I8 ? kTileKeys : 4];
  __align__(16) float vs[2][I8 ? kTileKeys : 4];
  int flag;
};

template <int D, bool I8, bool TREE>
__global__ __launch_bounds__(256, 2) void attn_tile_kernel(CacheView c, AttnArgs a, Parts part) {
  constexpr int kQ = D / 16;       // Q fragments, and key products per subtile
  constexpr int kO = D / 32;       // output tiles
  constexpr int kChunks = D / 8;   // 16-byte chunks of a key row
  constexpr int kLoads = kTileKeys * D * 2 / 4096;  // 16-byte loads per thread, keys or values
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
  int b, block;
  if (!sequence_of_tile(a, G, tile, lane, &b, &block)) return;
  const Seq s = sequence(c, a, b, h == 0 && block == 0 && split == 0 && tid == 0);
  const int rows = s.n * G;
  const int r0 = block * kTileRows;
  if (block < 0 || r0 >= rows) return;
  // this lane's row (rows past the end repeat the last one and are not stored)
  const int my_row = r0 + wave * 32 + col;
  const int row = my_row < rows ? my_row : rows - 1;
  const int token = row / G;
  const int64_t qo = ((int64_t)(s.first + token) * a.heads + h * G + (row - token * G)) * D;
  u32x4 qf[kQ];
#pragma unroll
  for (int i = 0; i < kQ; ++i) qf[i] = *(const u32x4*)(a.q + qo + i * 16 + half * 8);

  // the positions that the workgroup takes: its part of those that its rows see
  const int row_end = end_of_rows<TREE>(s, G, r0, kTileRows);
  const int begin = split * part.chunk;
  if (split > 0 && begin >= row_end) return;
  const int end = row_end - begin > part.chunk ? begin + part.chunk : row_end;
  const int open = TREE ? s.context : s.context + r0 / G + 1;  // positions below are seen by all
  const int wave_first = (r0 + wave * 32 < rows ? r0 + wave * 32 : rows - 1) / G;
  const int wave_open = TREE ? s.context : s.context + wave_first + 1;
  const int wave_last = (r0 + wave * 32 + 31 < rows ? r0 + wave * 32 + 31 : rows - 1) / G;
  const int wave_end = TREE ? s.len : s.context + wave_last + 1;

  f32x16 o[kO];
#pragma unroll
  for (int i = 0; i < kO; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[i][r] = 0.f;
  float m = kLowest, l = 0.f;
  const float scale2 = a.scale * kLog2e;
  const int mask = (1 << c.page_shift) - 1;

  // the first tile at or after p whose page is in the cache; its (page, head) block
  int64_t block_at = 0;
  auto find = [&](int p) {
    for (; p < end; p += kTileKeys) {
      const int page = a.table[(int64_t)b * a.width + (p >> c.page_shift)];
      if (page >= 0 && page < c.num_pages) {
        block_at = (((int64_t)page * HK + h) << c.page_shift) + (p & mask);
        break;
      }
      if (tid == 0) report(c.status, kBadPage);
    }
    return p;
  };
  // LDS row of a key tile that this thread's j-th 16 bytes belong to, and the token there
  u32x4 kreg[I8 ? kLoads / 2 : 1], vreg[I8 ? kLoads / 2 : 1];
  float sreg = 0.f;
  auto stage = [&](int buf) {  // the tile of block_at
    if (!I8) {
      const uint8_t* kb = c.k + block_at * (D * 2);
      const uint8_t* vb = c.v + block_at * (D * 2);
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const int slot = (wave * kLoads + j) * 64 + lane;
        const int r = slot / kChunks, ch = (slot % kChunks) ^ (r & 7);
        const int t = (r & ~12) | (r & 4) << 1 | (r & 8) >> 1;
        load16_to_lds(kb + t * (D * 2) + ch * 16, lds.k[buf] + (wave * kLoads + j) * 1024);
        load16_to_lds(vb + slot * 16, lds.v[buf] + (wave * kLoads + j) * 1024);
      }
    } else {
      const uint8_t* kb = c.k + block_at * D;
      const uint8_t* vb = c.v + block_at * D;
#pragma unroll
      for (int j = 0; j < kLoads / 2; ++j) {
        kreg[j] = *(const u32x4*)(kb + (j * 256 + tid) * 16);
        vreg[j] = *(const u32x4*)(vb + (j * 256 + tid) * 16);
      }
      if (tid < 2 * kTileKeys) sreg = (tid < kTileKeys ? c.k_scales : c.v_scales)[block_at + (tid & (kTileKeys - 1))];
    }
  };
  auto land = [&](int buf) {  // int8: the staged registers into LDS
    if (!I8) return;
#pragma unroll
    for (int j = 0; j < kLoads / 2; ++j) {
      const int piece = j * 256 + tid;
      u32x4 x[2];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint32_t lo, hi;
        bf16_of_codes(kreg[j][w], &lo, &hi);
        x[w >> 1][2 * (w & 1)] = lo;
        x[w >> 1][2 * (w & 1) + 1] = hi;
      }
      const int t = piece / (D / 16), ch = piece % (D / 16) * 2;
      const int r = (t & ~12) | (t & 4) << 1 | (t & 8) >> 1;
      *(u32x4*)(lds.k[buf] + (r * kChunks + (ch ^ (r & 7))) * 16) = x[0];
      *(u32x4*)(lds.k[buf] + (r * kChunks + ((ch + 1) ^ (r & 7))) * 16) = x[1];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint32_t lo, hi;
        bf16_of_codes(vreg[j][w], &lo, &hi);
        x[w >> 1][2 * (w & 1)] = lo;
        x[w >> 1][2 * (w & 1) + 1] = hi;
      }
      const int g16 = piece / D, d = piece % D;
      *(u32x4*)(lds.v[buf] + ((2 * g16) * D + d) * 16) = x[0];
      *(u32x4*)(lds.v[buf] + ((2 * g16 + 1) * D + d) * 16) = x[1];
    }
    if (tid < kTileKeys)
      lds.ks[buf][tid] = sreg * scale2;
    else if (tid < 2 * kTileKeys)
      lds.vs[buf][tid - kTileKeys] = sreg;
  };

  int buf = 0;
  int p = find(begin);
  if (p < end) {
    stage(0);
    land(0);
  }
  while (p < end) {
    wait_vmem();
    lds_barrier();
    const int next = find(p + kTileKeys);
    if (next < end) stage(buf ^ 1);
    // Values that some row must not see (or that lie past the sequence's end)
    // would still meet a weight of zero in the matrix products: 0 x NaN.  In
    // tiles with masked tokens, values past the end become zero, and if a
    // value is not finite, it is added by hand to the rows that see it.
    uint64_t vis = ~0ull;
    if (!I8 && p + kTileKeys > open) {
      if (tid == 0) lds.flag = 0;
      lds_barrier();
      bool odd = false;
      for (int i = tid; i < kTileKeys * kChunks; i += 256) {
        const int t = i / D * 8;
        u32x4 w = *(const u32x4*)(lds.v[buf] + i * 16);
        const int inside = s.len - p - t;
        if (inside < 8) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t keep = (2 * j < inside ? 0xffffu : 0u) | (2 * j + 1 < inside ? 0xffff0000u : 0u);
            w[j] &= keep;
          }
          *(u32x4*)(lds.v[buf] + i * 16) = w;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) odd |= non_finite_pair(w[j]);
      }
      if (odd) lds.flag = 1;
      lds_barrier();
      if (lds.flag) {
        vis = visible<TREE>(a, s, token, p);
        for (int t = 0; t < kTileKeys; ++t) {
          const uint16_t* src = (const uint16_t*)lds.v[buf] + (t >> 3) * D * 8 + (t & 7);
          const bool sees = vis >> t & 1;
#pragma unroll
          for (int i = 0; i < kO; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const uint32_t x = src[(i * 32 + (r & 3) + 8 * (r >> 2) + 4 * half) * 8];
              o[i][r] += sees && (x & 0x7f80u) == 0x7f80u ? bf16_bits_to_f32(x) : 0.f;
            }
        }
        lds_barrier();
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
      }
    }
    if (p < wave_end) {
      f32x16 st[2];
#pragma unroll
      for (int sub = 0; sub < 2; ++sub) {
#pragma unroll
        for (int r = 0; r < 16; ++r) st[sub][r] = 0.f;
        const int kr = sub * 32 + col;
        const uint8_t* krow = lds.k[buf] + kr * (D * 2);
#pragma unroll
        for (int i = 0; i < kQ; ++i) {
          const u32x4 kf = *(const u32x4*)(krow + ((2 * i + half) ^ (kr & 7)) * 16);
          st[sub] = mfma32_bf16(kf, qf[i], st[sub]);
        }
      }
      // register r of subtile sub: token sub 32 + (r >> 3) 16 + half 8 + (r & 7)
      if (I8) {
#pragma unroll
        for (int q4 = 0; q4 < 8; ++q4) {
          const f32x4 f = *(const f32x4*)(lds.ks[buf] + (q4 >> 1) * 16 + half * 8 + (q4 & 1) * 4);
#pragma unroll
          for (int j = 0; j < 4; ++j) st[q4 >> 2][(q4 & 3) * 4 + j] *= f[j];
        }
      }
      const bool masks = p + kTileKeys > wave_open || p + kTileKeys > s.len;
      if (masks) {
        vis = visible<TREE>(a, s, token, p) >> (8 * half);
#pragma unroll
        for (int sub = 0; sub < 2; ++sub)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            st[sub][r] = vis >> (sub * 32 + (r >> 3) * 16 + (r & 7)) & 1 ? st[sub][r] : -__builtin_huge_valf();
      }
      float top = st[0][0];
#pragma unroll
      for (int r = 1; r < 32; ++r) top = fmaxf(top, st[r >> 4][r & 15]);
      top = max_xor32(top);
      if (!I8) top *= scale2;
      const bool moves = top > m + kSlack;
      if (__any(moves)) {
        const float to = moves ? top : m;
        const float fix = __builtin_amdgcn_exp2f(m - to);
        m = to;
        l *= fix;
#pragma unroll
        for (int i = 0; i < kO; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[i][r] *= fix;
      }
      u32x4 pf[4];
#pragma unroll
      for (int r = 0; r < 32; r += 2) {
        const float s0 = st[r >> 4][r & 15], s1 = st[r >> 4][(r & 15) + 1];
        const float p0 = __builtin_amdgcn_exp2f(I8 ? s0 - m : s0 * scale2 - m);
        const float p1 = __builtin_amdgcn_exp2f(I8 ? s1 - m : s1 * scale2 - m);
        l += p0 + p1;
        st[r >> 4][r & 15] = p0;
        st[r >> 4][(r & 15) + 1] = p1;
      }
      if (I8) {
#pragma unroll
        for (int q4 = 0; q4 < 8; ++q4) {
          const f32x4 f = *(const f32x4*)(lds.vs[buf] + (q4 >> 1) * 16 + half * 8 + (q4 & 1) * 4);
#pragma unroll
          for (int j = 0; j < 4; ++j) st[q4 >> 2][(q4 & 3) * 4 + j] *= f[j];
        }
        if (masks) {  // an unseen value's scale may be anything: 0 x NaN
#pragma unroll
          for (int r = 0; r < 32; ++r)
            st[r >> 4][r & 15] = vis >> ((r >> 3) * 16 + (r & 7)) & 1 ? st[r >> 4][r & 15] : 0.f;
        }
      }
#pragma unroll
      for (int r = 0; r < 32; r += 2) pf[r >> 3][(r & 7) >> 1] = pack_p(st[r >> 4][r & 15], st[r >> 4][(r & 15) + 1]);
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
#pragma unroll
        for (int i = 0; i < kO; ++i) {
          const u32x4 vf = *(const u32x4*)(lds.v[buf] + ((2 * kk + half) * D + i * 32 + col) * 16);
          o[i] = mfma32_bf16(vf, pf[kk], o[i]);
        }
    }
    if (next < end) land(buf ^ 1);
    buf ^= 1;
    p = next;
  }
  l = add_xor32(l);
  if (my_row >= rows) return;
  if (row_end > part.chunk) {  // the join adds the parts
    const int64_t at = part.row(tile, h, HK, split, kTileRows, wave * 32 + col);
#pragma unroll
    for (int i = 0; i < kO; ++i)
#pragma unroll
      for (int r = 0; r < 16; r += 4)
        *(f32x4*)(part.o + at * D + i * 32 + 8 * (r >> 2) + 4 * half) =
            f32x4{o[i][r], o[i][r + 1], o[i][r + 2], o[i][r + 3]};
    if (half == 0) {
      part.ml[2 * at] = m;
      part.ml[2 * at + 1] = l;
    }
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
  for (int i = 0; i < kO; ++i)
#pragma unroll
    for (int r = 0; r < 16; r += 4)
      *(u32x2*)(a.out + qo + i * 32 + 8 * (r >> 2) + 4 * half) =
          u32x2{pack_p(o[i][r] * inv, o[i][r + 1] * inv), pack_p(o[i][r + 2] * inv, o[i][r + 3] * inv)};
}

// ---------------------------------------------------------------------------
// Row form: up to 16 rows of a sequence (the G heads of a decode step's token),
// where reading keys and values is all there is.  The workgroup's four waves
// take steps of 32 (bf16) or 64 (int8) tokens in turn, 16 KB of D = 128, and
// load them straight into the operands of 16x16x32 matrix instructions, one
// step ahead: no LDS and no barrier until the waves' results are added.
//   S^T = K . Q^T, O^T = V^T . P^T as in the tile form: key row r of tile t is
//   token (r / 4) KS / 4 + 4 t + r % 4 of the step, so that a lane's scores are
//   the KS / 4 consecutive tokens that it must supply as P^T and whose values
//   lie in the 16 bytes that it loads.
// ---------------------------------------------------------------------------
template <int D, bool I8, bool TREE>
__global__ __launch_bounds__(256, 2) void attn_row_kernel(CacheView c, AttnArgs a, Parts part, int blocks) {
  constexpr int KS = I8 ? 64 : 32;  // tokens per step
  constexpr int NT = KS / 16;       // key tiles per step
  constexpr int KL = I8 ? D / 64 : D / 32;  // 16-byte loads per key row and lane
  constexpr int kO = D / 16;
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
  const int item = rest / part.splits;
  const int b = item / blocks, block = item - b * blocks;
  const Seq s = sequence(c, a, b, h == 0 && block == 0 && split == 0 && tid == 0);
  const int rows = s.n * G, r0 = block * kRowRows;
  if (r0 >= rows) return;
  const int row_end = end_of_rows<TREE>(s, G, r0, kRowRows);
  const int begin = split * part.chunk;
  if (split > 0 && begin >= row_end) return;
  const int end = row_end - begin > part.chunk ? begin + part.chunk : row_end;
  const int row = r0 + col < rows ? r0 + col : rows - 1;
  const int token = row / G;
  const uint16_t* q = a.q + ((int64_t)(s.first + token) * a.heads + h * G + (row - token * G)) * D;
  u32x4 qf[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
    qf[i] = *(const u32x4*)(q + (I8 ? (i >> 1) * 64 + g * 16 + (i & 1) * 8 : i * 32 + g * 8));
  const int open = TREE ? s.context : s.context + r0 / G + 1;  // positions below are seen by all rows

  f32x4 o[kO];
#pragma unroll
  for (int i = 0; i < kO; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = kLowest, l = 0.f;
  const float scale2 = a.scale * kLog2e;
  const int mask = (1 << c.page_shift) - 1;
  const int krow = (col >> 2) * (KS / 4) + (col & 3);

  struct Step {
    u32x4 k[NT * KL], v[kO];
    float ks, vs;  // int8: lane's token
    bool ok;       // the page is in the cache
    int64_t at;    // its first token's place
  };
  auto load = [&](int p, Step& x) {
    const int page = a.table[(int64_t)b * a.width + (p >> c.page_shift)];
    x.ok = page >= 0 && page < c.num_pages;
    x.at = (((int64_t)(x.ok ? page : 0) * HK + h) << c.page_shift) + (p & mask);
    const uint8_t* kb = c.k + x.at * (D * (I8 ? 1 : 2)) + krow * (D * (I8 ? 1 : 2)) + g * 16;
    const uint8_t* vb = c.v + x.at * (D * (I8 ? 1 : 2)) + (g * D + col) * 16;
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
        for (int r = 0; r < 4; ++r) st[t][r] *= f[r];
      }
    }
    const int valid = x.ok ? s.len - p : 0;  // tokens of the step that exist
    const bool masks = p + KS > open || valid < KS;
    uint32_t vis = ~0u;
    if (masks) {
      uint64_t bits = visible<TREE>(a, s, token, p);
      if (valid < KS) bits &= (1ull << valid) - 1;
      vis = (uint32_t)(bits >> (g * (KS / 4)));
      if (!x.ok && lane == 0) report(c.status, kBadPage);
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) st[t][r] = vis >> (t * 4 + r) & 1 ? st[t][r] : -__builtin_huge_valf();
      if (!I8) {
        // values past the end become zero; one that is not finite, which some
        // row may not see, is added by hand to the rows that do (0 x NaN)
        const int inside = valid - g * 8;
        bool odd = false;
#pragma unroll
        for (int i = 0; i < kO; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t keep = (2 * j < inside ? 0xffffu : 0u) | (2 * j + 1 < inside ? 0xffff0000u : 0u);
            x.v[i][j] &= keep;
            odd |= non_finite_pair(x.v[i][j]);
          }
        if (__any(odd)) {
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
    float top = st[0][0];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) top = fmaxf(top, st[t][r]);
    top = max_xor32(max_xor16(top));
    if (!I8) top *= scale2;
    const bool moves = top > m + kSlack;
    if (__any(moves)) {
      const float to = moves ? top : m;
      const float fix = __builtin_amdgcn_exp2f(m - to);
      m = to;
      l *= fix;
#pragma unroll
      for (int i = 0; i < kO; ++i) o[i] *= fix;
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        st[t][r] = __builtin_amdgcn_exp2f(I8 ? st[t][r] - m : st[t][r] * scale2 - m);
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
      pf[t >> 1][2 * (t & 1)] = pack_p(st[t][0], st[t][1]);
      pf[t >> 1][2 * (t & 1) + 1] = pack_p(st[t][2], st[t][3]);
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
    if (p + 4 * KS < end) load(p + 4 * KS, x1);
    compute(p, x0);
    p += 4 * KS;
    if (p >= end) break;
    if (p + 4 * KS < end) load(p + 4 * KS, x0);
    compute(p, x1);
    p += 4 * KS;
  }

  // the four waves' results, added in order
  l = add_xor32(add_xor16(l));
  if (g == 0) {
    s_m[wave][col] = m;
    s_l[wave][col] = l;
  }
#pragma unroll
  for (int i = 0; i < kO; ++i) *(f32x4*)&s_o[wave][col][i * 16 + g * 4] = o[i];
  __syncthreads();
  const int r = tid >> 4, d0 = (tid & 15) * (D / 16);
  if (r0 + r >= rows) return;
  float top = s_m[0][r];
#pragma unroll
  for (int w = 1; w < 4; ++w) top = fmaxf(top, s_m[w][r]);
  float sum = 0.f, out[D / 16];
#pragma unroll
  for (int d = 0; d < D / 16; ++d) out[d] = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float f = __builtin_amdgcn_exp2f(s_m[w][r] - top);
    sum += s_l[w][r] * f;
#pragma unroll
    for (int d = 0; d < D / 16; ++d) out[d] += s_o[w][r][d0 + d] * f;
  }
  if (row_end > part.chunk) {
    const int64_t at = part.row(item, h, HK, split, kRowRows, r);
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
  const int tok = (r0 + r) / G;
  uint16_t* dst = a.out + ((int64_t)(s.first + tok) * a.heads + h * G + (r0 + r - tok * G)) * D + d0;
#pragma unroll
  for (int d = 0; d < D / 16; d += 4)
    *(u32x2*)(dst + d) = u32x2{pack_p(out[d] * inv, out[d + 1] * inv), pack_p(out[d + 2] * inv, out[d + 3] * inv)};
}

// Adds the splits of one item's rows, in order: 16 rows per workgroup.
template <int D, bool TREE, int ROWS>
__global__ __launch_bounds__(256) void join_kernel(CacheView c, AttnArgs a, Parts part, int blocks) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int HK = c.kv_heads, G = a.heads / HK;
  constexpr int kBlocks = ROWS / 16;
  const int h = (int)(blockIdx.x % (unsigned)HK);
  const int rest = (int)(blockIdx.x / (unsigned)HK);
  const int item = rest / kBlocks;
  int b, block;
  if (ROWS == kRowRows) {
    b = item / blocks;
    block = item - b * blocks;
  } else if (!sequence_of_tile(a, G, item, lane, &b, &block)) {
    return;
  }
  const Seq s = sequence(c, a, b, false);
  const int rows = s.n * G, r0 = block * ROWS;
  const int r = rest % kBlocks * 16 + (tid >> 4), d0 = (tid & 15) * (D / 16);
  if (r0 >= rows) return;
  const int row_end = end_of_rows<TREE>(s, G, r0, ROWS);
  if (row_end <= part.chunk || r0 + r >= rows) return;
  const int splits = (row_end + part.chunk - 1) / part.chunk;
  float top = kLowest;
  for (int i = 0; i < splits; ++i) top = fmaxf(top, part.ml[2 * part.row(item, h, HK, i, ROWS, r)]);
  float sum = 0.f, out[D / 16];
#pragma unroll
  for (int d = 0; d < D / 16; ++d) out[d] = 0.f;
#pragma unroll 4
  for (int i = 0; i < splits; ++i) {
    const int64_t at = part.row(item, h, HK, i, ROWS, r);
    const float f = __builtin_amdgcn_exp2f(part.ml[2 * at] - top);
    sum += part.ml[2 * at + 1] * f;
#pragma unroll
    for (int d = 0; d < D / 16; d += 4) {
      const f32x4 x = *(const f32x4*)(part.o + at * D + d0 + d);
#pragma unroll
      for (int j = 0; j < 4; ++j) out[d + j] += x[j] * f;
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
  const int tok = (r0 + r) / G;
  uint16_t* dst = a.out + ((int64_t)(s.first + tok) * a.heads + h * G + (r0 + r - tok * G)) * D + d0;
#pragma unroll
  for (int d = 0; d < D / 16; d += 4)
    *(u32x2*)(dst + d) = u32x2{pack_p(out[d] * inv, out[d + 1] * inv), pack_p(out[d + 2] * inv, out[d + 3] * inv)};
}

// The launch of a forward call: by what the caller knows without asking the
// device (its rows and bounds).
struct Plan {
  bool row_form;
  int blocks;  // row form: row blocks of a sequence
  int rows;    // of an item
  Parts part;
};

Plan plan_of(const CacheView& c, int heads, int tokens, int seqs, int max_queries, int max_len) {
  Plan p = {};
  const int64_t G = heads / c.kv_heads;
  p.row_form = max_queries * G <= kRowRows;
  p.rows = p.row_form ? kRowRows : kTileRows;
  p.blocks = 1;
  p.part.items = (int)(p.row_form ? seqs : tokens * G / kTileRows + seqs);
  const int64_t wgs = (int64_t)p.part.items * c.kv_heads;
  // enough workgroups for the chip
  const int64_t want = p.row_form ? 2048 : 512;
  const int least = 256, most = p.row_form ? 1024 : 1 << 30;
  int64_t chunk = max_len;
  if (wgs < want) {
    const int64_t splits = (want + wgs - 1) / wgs;
    chunk = (max_len + splits - 1) / splits;
  }
  chunk = chunk < most ? chunk : most;
  chunk = (chunk + least - 1) / least * least;
  if (chunk < least) chunk = least;
  p.part.chunk = (int)chunk;
  p.part.splits = (int)((max_len + chunk - 1) / chunk);
  if (p.part.splits < 1) p.part.splits = 1;
  return p;
}

size_t plan_rows(const CacheView& c, const Plan& p) {
  return p.part.splits > 1 ? (size_t)p.part.items * c.kv_heads * p.part.splits * p.rows : 0;
}

}  // namespace

size_t attn_workspace_bytes(const CacheView& c, int heads, int tokens, int seqs, int max_queries, int max_len) {
  return plan_rows(c, plan_of(c, heads, tokens, seqs, max_queries, max_len)) * (c.dim + 2) * sizeof(float);
}

hipError_t launch_attn(const CacheView& c, const AttnArgs& a, void* workspace, hipStream_t stream) {
  Plan p = plan_of(c, a.heads, a.tokens, a.seqs, a.max_queries, a.max_len);
  p.part.o = (float*)workspace;
  p.part.ml = (float*)workspace + plan_rows(c, p) * c.dim;
  const dim3 grid((unsigned)((int64_t)p.part.items * c.kv_heads * p.part.splits));
  const dim3 join_grid((unsigned)((int64_t)p.part.items * c.kv_heads * (p.rows / 16)));
  by_layout(c, [&](auto dim, auto int8) {
    constexpr int D = decltype(dim)::value;
    constexpr bool I8 = decltype(int8)::value;
    auto launch = [&](auto tree) {
      constexpr bool TREE = decltype(tree)::value;
      if (p.row_form)
        hipLaunchKernelGGL((attn_row_kernel<D, I8, TREE>), grid, dim3(256), 0, stream, c, a, p.part, p.blocks);
      else
        hipLaunchKernelGGL((attn_tile_kernel<D, I8, TREE>), grid, dim3(256), 0, stream, c, a, p.part);
      if (p.part.splits > 1) {
        if (p.row_form)
          hipLaunchKernelGGL((join_kernel<D, TREE, kRowRows>), join_grid, dim3(256), 0, stream, c, a, p.part, p.blocks);
        else
          hipLaunchKernelGGL((join_kernel<D, TREE, kTileRows>), join_grid, dim3(256), 0, stream, c, a, p.part, p.blocks);
      }
    };
    a.tree ? launch(std::true_type{}) : launch(std::false_type{});
  });
  return hipGetLastError();
}

}  // namespace nkt
