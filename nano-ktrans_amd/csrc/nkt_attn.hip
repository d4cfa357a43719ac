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
constexpr int kTileRows = 128, kTileKeys = 64;

template <int D, bool I8>
struct TileLds {
  __align__(16) uint8_t k[2][kTileKeys * D * 2];
  __align__(16) uint8_t v[2][kTileKeys * D * 2];
  __align__(16) float ks[2][I8 ? kTileKeys : 4];
  __align__(16) float vs[2][I8 ? kTileKeys : 4];
  int flag;
};

template <int D, bool I8, bool TREE>
__global__ __launch_bounds__(256, 2) void attn_tile_kernel(CacheView c, AttnArgs a, int tiles) {
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
  const int tile = tiles - 1 - (int)(blockIdx.x / (unsigned)HK);
  // sequence b's tiles start at starts[b] G / 128 + b, ascending and with room
  // for its ceil(n G / 128): the last b that starts at or before this tile
  int b = 0, block;
  if (a.starts) {
    for (int n = a.seqs; n > 1;) {
      const int step = (n + 63) / 64;
      const int i = b + lane * step;
      const bool before =
          lane * step < n && (int64_t)a.starts[i < a.seqs ? i : a.seqs] * G / kTileRows + i <= tile;
      const int count = __popcll(__ballot(before));
      if (count == 0) return;
      const int skip = (count - 1) * step;
      b += skip;
      n = n - skip < step ? n - skip : step;
    }
    b = __builtin_amdgcn_readfirstlane(b);
    block = tile - ((int)((int64_t)a.starts[b] * G / kTileRows) + b);
  } else {
    const int per = (G + kTileRows - 1) / kTileRows;
    b = tile / per;
    block = tile - b * per;
  }
  const Seq s = sequence(c, a, b, h == 0 && block == 0 && tid == 0);
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

  // the tokens that the workgroup's rows see, and what no row has to mask
  const int first_token = r0 / G;
  const int last_row = r0 + kTileRows < rows ? r0 + kTileRows - 1 : rows - 1;
  const int last_token = last_row / G;
  int end = s.len;
  if (!TREE && s.context + last_token + 1 < end) end = s.context + last_token + 1;
  const int open = TREE ? s.context : s.context + first_token + 1;  // positions below are seen by all
  const int wave_first = (r0 + wave * 32 < rows ? r0 + wave * 32 : rows - 1) / G;
  const int wave_open = TREE ? s.context : s.context + wave_first + 1;
  const int wave_last = (r0 + wave * 32 + 31 < rows ? r0 + wave * 32 + 31 : rows - 1) / G;
  const int wave_end = TREE ? end : s.context + wave_last + 1;

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
  int p = find(0);
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
  const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
  for (int i = 0; i < kO; ++i)
#pragma unroll
    for (int r = 0; r < 16; r += 4)
      *(u32x2*)(a.out + qo + i * 32 + 8 * (r >> 2) + 4 * half) =
          u32x2{pack_p(o[i][r] * inv, o[i][r + 1] * inv), pack_p(o[i][r + 2] * inv, o[i][r + 3] * inv)};
}

// One wave per (row, query head): tiles of 64 tokens, one per lane for the
// scores (running maximum and sum in fp32), one dimension per lane for P . V.
template <int D, bool I8, bool TREE>
__global__ __launch_bounds__(64) void attn_row_kernel(CacheView c, AttnArgs a) {
  constexpr int U = I8 ? 16 : 8;
  const int lane = threadIdx.x;
  const int row = (int)(blockIdx.x / (unsigned)a.heads), qh = (int)(blockIdx.x % (unsigned)a.heads);
  const int h = qh / (a.heads / c.kv_heads);
  __shared__ float s_q[D];
  __shared__ float s_p[64];
  // the row's sequence
  int b = row, first = row, n = 1;
  if (a.starts) {
    b = -1;
    for (int i0 = 0; i0 < a.seqs; i0 += 64) {
      const int i = i0 + lane;
      const bool mine = i < a.seqs && a.starts[i] <= row && row < a.starts[i + 1];
      const uint64_t m = __ballot(mine);
      if (m) b = i0 + __builtin_ctzll(m);
    }
    if (b < 0) return;
    first = a.starts[b];
    n = a.starts[b + 1] - first;
    if (row - first >= a.max_queries) {
      if (lane == 0) report(c.status, kBadLength);
      return;
    }
  }
  int64_t most = (int64_t)a.width << c.page_shift;
  most = most < a.max_len ? most : a.max_len;
  int len = a.lens[b];
  if (len < 0 || len > most) {
    if (lane == 0) report(c.status, kBadLength);
    len = len < 0 ? 0 : (int)most;
  }
  const int context = a.lens[b] < 0 ? 0 - n : a.lens[b] - n;
  const int last = TREE ? len - 1 : context + row - first;  // last position that may be seen
  const int64_t qo = ((int64_t)row * a.heads + qh) * D;
  for (int d = lane; d < D; d += 64) s_q[d] = bf16_bits_to_f32(a.q[qo + d]) * a.scale;
  __syncthreads();
  float m = -__builtin_huge_valf(), l = 0.f;
  float acc[D / 64];
#pragma unroll
  for (int j = 0; j < D / 64; ++j) acc[j] = 0.f;
  const int mask = (1 << c.page_shift) - 1;
  for (int p0 = 0; p0 <= last && p0 < len; p0 += 64) {
    const int64_t page = a.table[(int64_t)b * a.width + (p0 >> c.page_shift)];
    if (page < 0 || page >= c.num_pages) {
      if (lane == 0) report(c.status, kBadPage);
      continue;
    }
    const int64_t blk = block_of(c, page, h);
    const int off = p0 & mask;
    const int pos = p0 + lane;
    bool sees = pos <= last && pos < len;
    if (TREE && sees && pos >= context) {
      const int j = pos - context;
      sees = j / 64 < a.words && ((a.tree[(int64_t)row * a.words + j / 64] >> (j & 63)) & 1);
    }
    float s = 0.f, vs = 1.f;
    for (int d = 0; d < D; ++d)
      s += s_q[d] * (I8 ? (float)(int8_t)c.k[blk + (off + lane) * D + d]
                        : bf16_bits_to_f32(((const uint16_t*)c.k)[blk + (off + lane) * D + d]));
    if (I8) {
      const int64_t sa = ((page * c.kv_heads + h) << c.page_shift) + off + lane;
      s *= c.k_scales[sa];
      vs = c.v_scales[sa];
    }
    s = sees ? s : -__builtin_huge_valf();
    const float top = fmaxf(m, wave_max(s));
    const float use = top == -__builtin_huge_valf() ? 0.f : top;
    const float p = sees ? __expf(s - use) : 0.f;
    const float fix = __expf(m - use);
    l = l * fix + wave_sum_butterfly(p);
    m = top;
    s_p[lane] = sees ? p * vs : 0.f;
    const uint64_t seen = __ballot(sees);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < D / 64; ++j) {
      const int d = lane + 64 * j;
      float o = acc[j] * fix;
      for (int t = 0; t < 64; ++t) {
        if (!(seen >> t & 1)) continue;
        const int64_t at = blk + ((off + t) & ~(U - 1)) * D + d * U + ((off + t) & (U - 1));
        o += s_p[t] * (I8 ? (float)(int8_t)c.v[at] : bf16_bits_to_f32(((const uint16_t*)c.v)[at]));
      }
      acc[j] = o;
    }
    __syncthreads();
  }
#pragma unroll
  for (int j = 0; j < D / 64; ++j)
    a.out[qo + lane + 64 * j] = (uint16_t)f32_to_bf16_bits(l > 0.f || l != l ? acc[j] / l : 0.f);
}

}  // namespace

size_t attn_workspace_bytes(const CacheView& c, int heads, int tokens, int seqs, int max_queries, int max_len) {
  return 0;
}

hipError_t launch_attn(const CacheView& c, const AttnArgs& a, void* workspace, hipStream_t stream) {
  by_layout(c, [&](auto dim, auto int8) {
    constexpr int D = decltype(dim)::value;
    constexpr bool I8 = decltype(int8)::value;
    const int G = a.heads / c.kv_heads;
    if (a.max_queries * (int64_t)G > 16) {
      const int64_t tiles = a.starts ? (int64_t)a.tokens * G / kTileRows + a.seqs
                                     : (int64_t)a.seqs * ((G + kTileRows - 1) / kTileRows);
      const dim3 tile_grid((unsigned)(tiles * c.kv_heads));
      if (a.tree)
        hipLaunchKernelGGL((attn_tile_kernel<D, I8, true>), tile_grid, dim3(256), 0, stream, c, a, (int)tiles);
      else
        hipLaunchKernelGGL((attn_tile_kernel<D, I8, false>), tile_grid, dim3(256), 0, stream, c, a, (int)tiles);
      return;
    }
    const dim3 grid((unsigned)a.tokens * a.heads);
    if (a.tree)
      hipLaunchKernelGGL((attn_row_kernel<D, I8, true>), grid, dim3(64), 0, stream, c, a);
    else
      hipLaunchKernelGGL((attn_row_kernel<D, I8, false>), grid, dim3(64), 0, stream, c, a);
  });
  return hipGetLastError();
}

}  // namespace nkt
