// Low-rank adapters of many requests beside a shared projection.
#include <type_traits>

#include "nkt_common.h"
#include "nkt_lora_internal.h"

namespace nkt {

namespace {

constexpr int kTile = 32;  // tokens of a workgroup: one side of a 32x32x16 product

typedef float f32x16 __attribute__((ext_vector_type(16)));

// 32x32x16 bf16: lane l supplies A[l%32][8*(l/32) .. +7] and B[8*(l/32) ..
// +7][l%32]; D[(v&3) + 8*(v>>2) + 4*(l/32)][l%32] lands in register v.
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                 0);
}
__device__ __forceinline__ f32x16 zeros() {
  f32x16 x;
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = 0.f;
  return x;
}

// Two floats -> packed bf16 pair (lo = first), round to nearest even.
__device__ __forceinline__ uint32_t pair_of(float lo, float hi) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, bf16x2));
}

constexpr int kMaxAdapters = 4096;  // (whose counts lie in LDS)
constexpr int kNone = -1, kPast = -2;

// The adapter of the tile's token in this lane (lanes l and l + 32 have the same
// one): kNone without one, kPast behind the last token.
__device__ __forceinline__ int adapter_of(const LoraView& v, const LoraArgs& a, int tile, int col, bool reports) {
  const int t = tile * kTile + col;
  if (t >= a.tokens) return kPast;
  const int64_t i = a.index[t];
  if (i >= v.adapters) {
    if (reports) __hip_atomic_fetch_or(v.status, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return kNone;
  }
  return i < 0 ? kNone : (int)i;
}

// The slot-th distinct adapter of the tile (kNone counts where `none` does), kPast: there are fewer.
__device__ __forceinline__ int distinct(int mine, int slot, bool none) {
  uint64_t todo = __ballot(none ? mine != kPast : mine >= 0);
  int found = kPast;
  for (int i = 0; i <= slot; ++i) {
    if (todo == 0) return kPast;
    found = __builtin_amdgcn_readlane(mine, __builtin_ctzll(todo));
    todo &= ~__ballot(mine == found);
  }
  return found;
}

// The tile of workgroup x of a launch: runs of tiles, which mostly share an adapter,
// on one XCD (workgroup i runs on XCD i % 8) and so on one copy of it in its L2.
__device__ __forceinline__ int tile_of(int x, int tiles) {
  const int run = (tiles + 7) / 8;
  return tiles < 64 ? x : x % 8 * run + x / 8;
}
// (workgroups so that every tile has one; those past the last tile end at once)
int tile_groups(int tiles) { return tiles < 64 ? tiles : (tiles + 7) / 8 * 8; }

// ---------------------------------------------------------------------------
// Tokens by adapter, in tiles of 32 that each have one adapter (kNone: without one,
// where these have to be copied; kPast: no tile), for more tokens than one launch
// takes.  By one workgroup: the counts stay in LDS, and 8418 tokens take 9 us (1000 about
// 5, mostly the launch).  Which place of its adapter's tiles a token gets depends on
// the order in which waves arrive; what is computed for it does not depend on its
// place.
// ---------------------------------------------------------------------------
constexpr int kGroupThreads = 1024;

__global__ __launch_bounds__(kGroupThreads) void group_kernel(LoraView v, LoraArgs a, int tiles, bool copies) {
  __shared__ int s_count[kMaxAdapters + 1], s_place[kMaxAdapters + 1], s_sums[kGroupThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = v.adapters + 1;  // (the last: without an adapter)
  for (int i = tid; i < n; i += kGroupThreads) s_count[i] = 0;
  __syncthreads();
  // (of kEach tokens at once: one at a time their latency is all there is)
  constexpr int kEach = 8;
  // A token's group, told from its index once and kept where low comes to lie: told again it
  // could be another one, if the index changes meanwhile, and places would stay unwritten.
  int32_t* const groups = (int32_t*)a.low;
  // (of a wave's tokens, those of the first one's adapter in one addition)
  auto count = [&](int group, int* to) __attribute__((always_inline)) {
    const int lead = __builtin_amdgcn_readfirstlane(group);
    const uint64_t sames = __ballot(group == lead);
    int at = 0;
    if (lead != kPast) {
      if (lane == 0) at = atomicAdd(&to[lead], __popcll(sames));
      at = __builtin_amdgcn_readfirstlane(at) + __popcll(sames & ((1ull << lane) - 1));
    }
    if (group != lead && group != kPast) at = atomicAdd(&to[group], 1);
    return at;
  };
  for (int t = tid; t - lane < a.tokens; t += kEach * kGroupThreads) {
    int64_t index[kEach];
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int from = t + j * kGroupThreads;
      index[j] = a.index[from < a.tokens ? from : a.tokens - 1];
    }
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int at = t + j * kGroupThreads;
      if (at - lane >= a.tokens) break;
      const int64_t i = index[j];
      const int group = at >= a.tokens ? kPast : i < 0 || i >= v.adapters ? v.adapters : (int)i;
      if (group != kPast) {
        if (i >= v.adapters) __hip_atomic_fetch_or(v.status, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        groups[at] = group;
      }
      count(group, s_count);
    }
  }
  __syncthreads();
  // first tiles, by a scan over the groups: thread t has groups t each ... on
  const int each = (n + kGroupThreads - 1) / kGroupThreads;
  auto tiles_of = [&](int group) { return group == v.adapters && !copies ? 0 : (s_count[group] + kTile - 1) / kTile; };
  int sum = 0;
  for (int i = tid * each; i < (tid + 1) * each && i < n; ++i) sum += tiles_of(i);
  const int upto = wave_inclusive_scan(sum);
  if (lane == 63) s_sums[wave] = upto;
  __syncthreads();
  int first = upto - sum, total = 0;
#pragma unroll
  for (int i = 0; i < kGroupThreads / 64; ++i) {
    first += i < wave ? s_sums[i] : 0;
    total += s_sums[i];
  }
  for (int i = tid * each; i < (tid + 1) * each && i < n; ++i) {
    s_place[i] = first * kTile;
    first += tiles_of(i);
  }
  __syncthreads();
  // a group's tiles by its wave: which adapter, and no token behind its last one
  for (int i = wave; i < n; i += kGroupThreads / 64) {
    const int from = s_place[i] / kTile, number = tiles_of(i);
    for (int t = lane; t < number; t += 64) a.tile_adapter[from + t] = i == v.adapters ? kNone : i;
    const int last = (number - 1) * kTile + lane;
    if (number > 0 && lane < kTile && s_count[i] <= last) a.order[from * kTile + last] = -1;
  }
  for (int t = total + tid; t < tiles; t += kGroupThreads) a.tile_adapter[t] = kPast;
  __syncthreads();
  for (int t = tid; t - lane < a.tokens; t += kEach * kGroupThreads) {
    int group[kEach];
#pragma unroll
    for (int j = 0; j < kEach; ++j) {  // (the thread's own)
      const int at = t + j * kGroupThreads;
      group[j] = at < a.tokens ? groups[at] : kPast;
    }
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int at = t + j * kGroupThreads;
      if (at - lane >= a.tokens) break;
      const int place = count(group[j], s_place);
      if (group[j] != kPast && (group[j] < v.adapters || copies)) a.order[place] = at;
    }
  }
}

// low, as the operands of the second product: two bf16 values whose sum is a rank's
// fp32 value to 2^-16 of it (its upper 16 bits, and the rest rounded).  The second is
// zero only where the value is (an infinity's is one too), so that an infinity of B
// stays one.  Per tile, part, 16 ranks and which of the two: 64 lanes x 8 ranks.
__device__ __forceinline__ uint16_t* low_at(const LoraView& v, const LoraArgs& a, int tile, int part, int s, int which) {
  return a.low + ((((int64_t)tile * v.parts + part) * (v.rank / 16) + s) * 2 + which) * 512;
}

// A part's rank of an adapter, within what its matrices hold (the caller's buffer may say anything).
__device__ __forceinline__ int rank_of(const LoraView& v, int adapter, int part) {
  const int rank = v.ranks[adapter * v.parts + part];
  return rank < 0 ? 0 : rank < v.rank ? rank : v.rank;
}
// The adapter's ranks, one per part and lane.
__device__ __forceinline__ int lane_ranks(const LoraView& v, int adapter, int lane) {
  return lane < v.parts ? rank_of(v, adapter, lane) : 0;
}

// A wave's share of 32 tokens of x times MB blocks of A: groups of 64 features kw, kw +
// KWAVES, ...  Both operands come straight from memory, RING groups ahead: A lies as its
// operand; x as rows of 128 bytes (a lane of its own row would cost the memory pipeline
// a turn per lane: 64 for 1 KB instead of 16), turned in 4 KB of LDS of the wave's own.
// xs: the lane's pieces of x, of row 8 i + lane / 8, chunk lane % 8 of a group's 8.
template <int MB, int KWAVES, int RING>
__device__ __forceinline__ void times_a(const uint16_t* const (&xs)[4], const uint16_t* const (&w)[MB], int groups,
                                        int kw, int lane, uint8_t* turn, f32x16 (&acc)[MB]) {
  const int half = lane >> 5, col = lane & 31;
  const int turns = kw < groups ? (groups - 1 - kw) / KWAVES + 1 : 0;
#pragma unroll
  for (int m = 0; m < MB; ++m) acc[m] = zeros();
  u32x4 xr[RING][4], af[RING][MB][4];
  // (behind the last group: the last one again, rather than a branch that would make
  // the waits for one group wait for those behind it as well)
  auto load = [&](int n, int at) __attribute__((always_inline)) {
    const int k = n * KWAVES + kw < groups ? n * KWAVES + kw : groups - 1;
#pragma unroll
    for (int i = 0; i < 4; ++i) xr[at][i] = *(const u32x4*)(xs[i] + k * 64);
#pragma unroll
    for (int m = 0; m < MB; ++m)
#pragma unroll
      for (int j = 0; j < 4; ++j) af[at][m][j] = *(const u32x4*)(w[m] + (k * 4 + j) * 512);
    __builtin_amdgcn_sched_barrier(0);  // (in this order, so that a group's wait is for it alone)
  };
#pragma unroll
  for (int n = 0; n < RING; ++n) load(n, n);
  for (int n0 = 0; n0 < turns; n0 += RING) {
#pragma unroll
    for (int n = 0; n < RING; ++n) {
      if (n0 + n >= turns) break;
      // chunk c of row r lies at c ^ r % 8
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = i * 8 + (lane >> 3);
        *(u32x4*)(turn + (r * 8 + ((lane & 7) ^ (r & 7))) * 16) = xr[n][i];
      }
      __builtin_amdgcn_wave_barrier();
      u32x4 xf[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) xf[j] = *(const u32x4*)(turn + (col * 8 + ((half * 4 + j) ^ (col & 7))) * 16);
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int m = 0; m < MB; ++m)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[m] = mfma32(af[n][m][j], xf[j], acc[m]);
      __builtin_amdgcn_sched_barrier(0);
      load(n0 + n + RING, n);
    }
  }
}

// Eight ranks of a token, first .. first + 7 of a part, from the waves' sums of a block of
// 32 rows (row 8 run + i: register 4 run + i % 4 of half i / 4): scaled, and split.
template <int KWAVES>
__device__ __forceinline__ void split_ranks(const float* sums, int run, int token, int first, int rank, float scale,
                                            u32x4* h, u32x4* r) {
  uint32_t high[8];
  float rest[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float sum = 0.f;
#pragma unroll
    for (int u = 0; u < KWAVES; ++u) sum += sums[(u * 64 + (i >> 2) * 32 + token) * 17 + run * 4 + (i & 3)];
    // (a rank that the adapter does not have is zero whatever x holds)
    const float y = first + i < rank ? sum * scale : 0.f;
    const uint32_t bits = __float_as_uint(y);
    high[i] = y != y ? 0x7fc00000u : bits & 0xffff0000u;
    // (0 times an infinity is NaN: in the place of no rest 2^-32 of y, which its fp32 sums lose)
    rest[i] = y - __uint_as_float(high[i]);
    rest[i] = rest[i] == 0.f || (bits & 0x7f800000u) == 0x7f800000u ? y * 0x1p-32f : rest[i];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    (*h)[i] = high[2 * i] >> 16 | high[2 * i + 1];
    (*r)[i] = pair_of(rest[2 * i], rest[2 * i + 1]);
  }
}

// ---------------------------------------------------------------------------
// low = scale x A^T: one workgroup per tile of 32 tokens and MB blocks of 32 rows of
// A, of those that hold a rank of the tile's adapter.  KWAVES waves share the input's
// features and add up in LDS in order.  Measured on 8192 tokens of 4096 features, 3
// parts of rank 64: 48 us, 0.53 PFLOP/s; bound by what the two sets of blocks read of x
// and A through the L2.
// ---------------------------------------------------------------------------
template <int MB, int KWAVES>
__global__ __launch_bounds__(KWAVES * 64) void shrink_kernel(LoraView v, LoraArgs a, int tiles) {
  // (the waves' turning places, then their sums: 64 lanes x 16, padded to 17)
  __shared__ __align__(16) uint8_t s_lds[KWAVES * 64 * 17 * 4];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int tile = tile_of((int)blockIdx.x, tiles);
  if (tile >= tiles) return;
  const uint16_t* xs[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = a.order[tile * kTile + i * 8 + (lane >> 3)];
    xs[i] = a.x + (t < 0 || t >= a.tokens ? 0 : t) * a.x_stride + (lane & 7) * 8;  // (past the tiles: anything)
  }
  const int adapter = __builtin_amdgcn_readfirstlane(a.tile_adapter[tile]);
  if (adapter < 0) return;
  // the blocks that hold a rank of the adapter, as bits (lane m looks at block m: its
  // rows are one part's, or 16 of two)
  const int ranks = lane_ranks(v, adapter, lane);
  const int part_at = lane * 32 / v.rank;
  const int rank_at = __shfl(ranks, part_at & 63), rank_behind = __shfl(ranks, (part_at + 1) & 63);
  uint32_t used = (uint32_t)__ballot(lane < v.row_blocks && (lane * 32 - part_at * v.rank < rank_at ||
                                                            (v.rank == 16 && rank_behind > 0)));
  for (int i = (int)blockIdx.y * MB; i > 0 && used; --i) used &= used - 1;
  if (used == 0) return;
  const int count = __popc(used);
  int blocks[MB];  // (behind the last one: the last one again, for nothing)
  const uint16_t* w[MB];
#pragma unroll
  for (int m = 0; m < MB; ++m) {
    blocks[m] = __builtin_ctz(used);
    if (used & (used - 1)) used &= used - 1;
    w[m] = v.a + ((int64_t)adapter * v.row_blocks + blocks[m]) * ((int64_t)v.in * 32) + lane * 8;
  }
  f32x16 acc[MB];
  times_a<MB, KWAVES, 2>(xs, w, v.in / 64, wave, lane, s_lds + wave * 4096, acc);
  float* const sums = (float*)s_lds;
#pragma unroll
  for (int m = 0; m < MB; ++m) {
    if (m >= count) break;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 16; ++i) sums[tid * 17 + i] = acc[m][i];
    __syncthreads();
    // a thread takes 8 rows of a token
    const int token = tid & 31, run = tid >> 5;
    const int row = blocks[m] * 32 + run * 8;
    const int part = row / v.rank, first = row - part * v.rank;
    const int rank = __shfl(ranks, part & 63);
    if (run >= 4 || part >= v.parts) continue;
    if (first >= (rank + 15) / 16 * 16) continue;  // (not read)
    u32x4 h, r;
    split_ranks<KWAVES>(sums, run, token, first, rank, v.scales[adapter * v.parts + part], &h, &r);
    const int lane_of = (first >> 3 & 1) * 32 + token;
    *(u32x4*)(low_at(v, a, tile, part, first >> 4, 0) + lane_of * 8) = h;
    *(u32x4*)(low_at(v, a, tile, part, first >> 4, 1) + lane_of * 8) = r;
  }
}

// ---------------------------------------------------------------------------
// out = base + low B^T: one workgroup per tile of 32 tokens and 4 x per_wave x 64
// columns.  A wave computes 32 tokens x 64 columns at a time: tokens in registers, a
// pair of neighbouring columns in a lane, so that 32 lanes read and write 128 bytes of
// a token's row.  The base of all its turns is asked for at once.  KS = R / 16.
// Bound by the base and the output: 8418 tokens of 6144 columns, ranks 64 and 32, take 57
// us, 3.6 TB/s; B, read anew by every tile of 32 tokens, is about 150 MB through the L2
// beside them.
//
// Ranks that fill KS or half of it have copies of their own, whose loads are all asked for
// at once.  Whole calls of 8192 tokens on 4096 -> 6144 columns, in us: R = 64, rank 64 103
// (by the loop over ranks 113), 32 93 (94), by the loop 48 110 and 16 92 (105 and 90 in a
// kernel that has nothing but the loop); R = 128, rank 128 151 (163), 64 112 (114), 96 160
// (138), 32 107 (96); R = 32 on 2048 -> 5120, rank 32 58 (60), 24 58 (60).  300 tokens
// differ by 1.5 at most.
// ---------------------------------------------------------------------------
constexpr int kTurns = 2;  // of a wave, at most

template <int KS>
__global__ __launch_bounds__(256, 2) void expand_kernel(LoraView v, LoraArgs a, int tiles, int per_wave) {
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = lane >> 5, col = lane & 31;
  const int tile = tile_of((int)blockIdx.x, tiles);
  if (tile >= tiles) return;
  const int pairs = v.columns / 64;
  const int c0 = ((int)blockIdx.y * 4 + wave) * per_wave;  // the wave's first 64 columns
  if (c0 >= pairs) return;
  const int turns = pairs - c0 < per_wave ? pairs - c0 : per_wave;
  const int adapter = __builtin_amdgcn_readfirstlane(a.tile_adapter[tile]);
  // register r is token (r & 3) + 8 (r >> 2) + 4 half of the tile
  int tokens[16];
#pragma unroll
  for (int r = 0; r < 16; r += 4) {
    const u32x4 x = *(const u32x4*)(a.order + tile * kTile + 8 * (r >> 2) + 4 * half);
#pragma unroll
    for (int i = 0; i < 4; ++i) tokens[r + i] = (int)x[i];
  }
  if (adapter == kPast) return;
  uint32_t y[kTurns][16];
#pragma unroll
  for (int i = 0; i < kTurns; ++i) {
    const uint16_t* src = a.base + (c0 + (i < turns ? i : turns - 1)) * 64 + 2 * col;
#pragma unroll
    for (int r = 0; r < 16; ++r) y[i][r] = *(const uint32_t*)(src + (tokens[r] < 0 ? 0 : tokens[r]) * a.base_stride);
  }
  auto store = [&](int i) __attribute__((always_inline)) {
    uint16_t* dst = a.out + (c0 + i) * 64 + 2 * col;
#pragma unroll
    for (int r = 0; r < 16; ++r)
      if (tokens[r] >= 0) *(uint32_t*)(dst + tokens[r] * a.out_stride) = y[i][r];
  };
  if (adapter < 0) {
#pragma unroll
    for (int i = 0; i < kTurns; ++i)
      if (i < turns) store(i);
    return;
  }
  const uint16_t* b = v.b + ((int64_t)adapter * pairs + c0) * (KS * 1024) + lane * 8;
  const int ranks = lane_ranks(v, adapter, lane);
  // the parts all have NS steps of 16 ranks, or any number (NS = 0)
  auto run = [&](auto ns) __attribute__((always_inline)) {
    constexpr int NS = decltype(ns)::value;
    int loaded = -1;
    u32x4 high[NS > 0 ? NS : 1], rest[NS > 0 ? NS : 1];
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
      if (i >= turns) break;
      const int part = (c0 + i >= v.part_end[0]) + (c0 + i >= v.part_end[1]) + (c0 + i >= v.part_end[2]);
      f32x16 acc[2] = {zeros(), zeros()};
      if constexpr (NS > 0) {
        u32x4 w[NS][2];
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
          for (int e = 0; e < 2; ++e) w[s][e] = *(const u32x4*)(b + (i * KS + s) * 1024 + e * 512);
        if (part != loaded) {
#pragma unroll
          for (int s = 0; s < NS; ++s) {
            high[s] = *(const u32x4*)(low_at(v, a, tile, part, s, 0) + lane * 8);
            rest[s] = *(const u32x4*)(low_at(v, a, tile, part, s, 1) + lane * 8);
          }
          loaded = part;
        }
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            acc[e] = mfma32(rest[s], w[s][e], acc[e]);
            acc[e] = mfma32(high[s], w[s][e], acc[e]);
          }
      } else {
        const int steps = (__builtin_amdgcn_readlane(ranks, part) + 15) / 16;
        for (int s = 0; s < steps; ++s) {
          const u32x4 h = *(const u32x4*)(low_at(v, a, tile, part, s, 0) + lane * 8);
          const u32x4 r = *(const u32x4*)(low_at(v, a, tile, part, s, 1) + lane * 8);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const u32x4 w = *(const u32x4*)(b + (i * KS + s) * 1024 + e * 512);
            acc[e] = mfma32(r, w, acc[e]);
            acc[e] = mfma32(h, w, acc[e]);
          }
        }
      }
#pragma unroll
      for (int r = 0; r < 16; ++r)
        y[i][r] = pair_of(__uint_as_float(y[i][r] << 16) + acc[0][r],
                          __uint_as_float(y[i][r] & 0xffff0000u) + acc[1][r]);
      store(i);
    }
  };
  const int steps = (ranks + 15) / 16;
  if (__ballot(lane < v.parts && steps != KS) == 0)
    run(std::integral_constant<int, KS>{});
  else if (KS > 1 && __ballot(lane < v.parts && steps != KS / 2) == 0)
    run(std::integral_constant<int, (KS + 1) / 2>{});
  else
    run(std::integral_constant<int, 0>{});
}

// ---------------------------------------------------------------------------
// Both products in one launch, for few tokens: one workgroup per tile, slot (the
// slot-th distinct adapter of the tile) and 512 x per_wave columns of a part.  Each
// computes the part's low for itself (R x in_features values of A from the L2, which
// cost less than a second launch) and leaves it in LDS; its waves' base and B are on
// their way meanwhile.  Bound by latency: a launch, x and A, B.  One token of 2048
// features to 5120 columns, rank 16: 8.9 us; 64 tokens of 24 adapters of rank 32, 4096
// features and columns: 15.5 us, of which x is a part: all 32 rows of the tile, also those
// of other adapters.
// ---------------------------------------------------------------------------
template <int KS>
__global__ __launch_bounds__(512) void both_kernel(LoraView v, LoraArgs a, int slots, int per_wave) {
  constexpr int kWaves = 8, RB = KS > 2 ? KS / 2 : 1;  // blocks of 32 rows of a part
  __shared__ __align__(16) uint8_t s_lds[kWaves * 64 * 17 * 4];
  __shared__ __align__(16) uint16_t s_low[KS][2][512];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = lane >> 5, col = lane & 31;
  const int slot = (int)(blockIdx.x % (unsigned)slots), tile = (int)(blockIdx.x / (unsigned)slots);
  const int mine = adapter_of(v, a, tile, col, tid < 32 && slot == 0 && blockIdx.y == 0);
  // the part and its columns that blockIdx.y counts to
  const int width = kWaves * per_wave;
  int part = 0, begin = 0, chunk = (int)blockIdx.y;
  while (chunk >= (v.part_end[part] - begin + width - 1) / width) {
    chunk -= (v.part_end[part] - begin + width - 1) / width;
    begin = v.part_end[part++];
  }
  const int end = v.part_end[part], c0 = begin + chunk * width + wave;  // the wave's 64 columns: c0, c0 + 8, ...
  const int adapter = distinct(mine, slot, a.base != a.out);
  if (adapter == kPast) return;
  const uint32_t seen = (uint32_t)__ballot(mine == adapter) >> (4 * half);
  // register r is token (r & 3) + 8 (r >> 2) + 4 half of the tile, the lane columns 2 col, 2 col + 1
  const uint16_t* const base = a.base + (int64_t)tile * kTile * a.base_stride;
  uint16_t* const out = a.out + (int64_t)tile * kTile * a.out_stride;
  const int base_lane = half * 4 * (int)a.base_stride + 2 * col, out_lane = half * 4 * (int)a.out_stride + 2 * col;
  uint32_t y[16];
  auto load = [&](int c) __attribute__((always_inline)) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int row = (r & 3) + 8 * (r >> 2);
      y[r] = 0;
      if (c < end && (seen >> row & 1)) y[r] = *(const uint32_t*)(base + c * 64 + row * a.base_stride + base_lane);
    }
  };
  auto store = [&](int c) __attribute__((always_inline)) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int row = (r & 3) + 8 * (r >> 2);
      if (c < end && (seen >> row & 1)) *(uint32_t*)(out + c * 64 + row * a.out_stride + out_lane) = y[r];
    }
  };
  load(c0);
  if (adapter < 0) {
    store(c0);
    for (int i = 1; i < per_wave; ++i) {
      load(c0 + i * kWaves);
      store(c0 + i * kWaves);
    }
    return;
  }
  const int rank = rank_of(v, adapter, part);
  const float scale = v.scales[adapter * v.parts + part];
  const uint16_t* b = v.b + (int64_t)adapter * (v.columns / 64) * (KS * 1024) + lane * 8;
  constexpr int kAhead = KS < 2 ? KS : 2;  // steps of B asked for before low
  u32x4 w[kAhead][2];
  auto load_b = [&](int c) __attribute__((always_inline)) {
#pragma unroll
    for (int s = 0; s < kAhead; ++s)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        w[s][e] = *(const u32x4*)(b + ((int64_t)(c < end ? c : begin) * KS + s) * 1024 + e * 512);
  };
  load_b(c0);
  const uint16_t* xs[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = tile * kTile + i * 8 + (lane >> 3);
    xs[i] = a.x + (t < a.tokens ? t : a.tokens - 1) * a.x_stride + (lane & 7) * 8;
  }
  const int block0 = part * v.rank / 32, skip = part * v.rank % 32;  // (16 ranks: half a block)
  float* const sums = (float*)s_lds;
  // (rank 128: two blocks at a time)
  constexpr int MB = RB < 2 ? RB : 2;
#pragma unroll
  for (int m0 = 0; m0 < RB; m0 += MB) {
    const uint16_t* wa[MB];
#pragma unroll
    for (int m = 0; m < MB; ++m)
      wa[m] = v.a + ((int64_t)adapter * v.row_blocks + block0 + m0 + m) * ((int64_t)v.in * 32) + lane * 8;
    f32x16 acc[MB];
    __syncthreads();  // (of the blocks before, the sums are read)
    times_a<MB, kWaves, MB == 1 ? 4 : 2>(xs, wa, v.in / 64, wave, lane, s_lds + wave * 4096, acc);
#pragma unroll
    for (int m = 0; m < MB; ++m) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 16; ++i) sums[tid * 17 + i] = acc[m][i];
      __syncthreads();
      const int token = tid & 31, run = tid >> 5;
      const int first = (m0 + m) * 32 + run * 8 - skip;
      if (run >= 4 || first < 0 || first >= KS * 16) continue;
      u32x4 h, r;
      split_ranks<kWaves>(sums, run, token, first, rank, scale, &h, &r);
      const int lane_of = (first >> 3 & 1) * 32 + token;
      *(u32x4*)(&s_low[first >> 4][0][lane_of * 8]) = h;
      *(u32x4*)(&s_low[first >> 4][1][lane_of * 8]) = r;
    }
  }
  __syncthreads();
  const int steps = __builtin_amdgcn_readfirstlane((rank + 15) / 16);
  for (int i = 0; i < per_wave; ++i) {
    const int c = c0 + i * kWaves;
    f32x16 acc[2] = {zeros(), zeros()};
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      if (s >= steps) break;
      const u32x4 high = *(const u32x4*)(&s_low[s][0][lane * 8]), rest = *(const u32x4*)(&s_low[s][1][lane * 8]);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const u32x4 wb = s < kAhead ? w[s < kAhead ? s : 0][e]
                                    : *(const u32x4*)(b + ((int64_t)(c < end ? c : begin) * KS + s) * 1024 + e * 512);
        acc[e] = mfma32(rest, wb, acc[e]);
        acc[e] = mfma32(high, wb, acc[e]);
      }
    }
#pragma unroll
    for (int r = 0; r < 16; ++r)
      y[r] = pair_of(__uint_as_float(y[r] << 16) + acc[0][r], __uint_as_float(y[r] & 0xffff0000u) + acc[1][r]);
    store(c);
    if (i + 1 < per_wave) {
      load(c + kWaves);
      load_b(c + kWaves);
    }
  }
}

// One launch for up to 64 tokens: three launches cost the host about 8 us more in a call
// outside of a graph, which then takes 19 to 20 at least.  One launch against grouped tokens,
// us on the GPU, and of whole calls in brackets where the GPU is not all of them; adapters
// dealt out in turn (of one adapter):
//                                        1 token       8 tokens      32 tokens     64 tokens
//   8 of rank 16, 2048 -> 5120            8.5 / 12.3    9.2 / 12.7    9.4 / 12.7    9.7 / 12.7  (9.3 / 13.1)
//        whole calls                       12 / 20       12 / 20       12 / 20       12 / 19
//   24 of rank 32, 4096 -> 4096          10.3 / 14.2   11.0 / 14.7   15.5 / 15.2   17.0 / 15.2  (12.4 / 15.2)
//        whole calls                       12 / 20       12 / 20       15 / 19       17 / 20
//   64 of rank 32, 4096 -> 4096          10.3 / 15.0   11.0 / 15.4   15.9 / 16.4   18.4 / 19.6  (15.5 / 16.4)
//   8 of rank 64, 4096 -> 6144           13.9 / 14.6   16.8 / 15.7   17.8 / 15.7   19.4 / 16.0  (14.9 / 15.9)
//        whole calls                       14 / 20       16 / 19       17 / 19       19 / 19
//   8 of rank 128, 4096 -> 6144          23.8 / 15.5   28.4 / 18.4   30.6 / 18.5   33.6 / 19.2  (24.7 / 16.4)
//   64 of rank 128, 4096 -> 4096         23.6 / 15.7   27.5 / 16.6   36.6 / 23.3   44.3 / 39.8  (32.5 / 18.9)
//   8 of rank 16, 4096 -> 28672          10.5 / 13.8   12.6 / 15.6   14.0 / 15.9   17.3 / 16.2  (15.2 / 15.5)
//   64 of rank 16, 4096 -> 28672         10.5 / 14.6   12.5 / 16.4   30.8 / 25.6   46.5 / 30.7  (47.1 / 22.8)
// So the number of tokens alone chooses right up to rank 64 and a few thousand columns;
// ranks over 64, and wide outputs beside many adapters (whose workgroups are given more
// columns by the adapters that there could be), lose by it.
constexpr int kBothTokens = 64;

// Tiles of grouped tokens: each group may leave one tile open.
int grouped_tiles(const LoraView& v, int tokens) {
  const int groups = v.adapters + 1 < tokens ? v.adapters + 1 : tokens;
  return (tokens + kTile - 1) / kTile + groups;
}
size_t low_bytes(const LoraView& v, int tiles) { return (size_t)tiles * v.parts * (v.rank / 16) * 2048; }

}  // namespace

size_t lora_workspace_bytes(const LoraView& v, int tokens) {
  if (tokens <= kBothTokens) return 0;
  const int tiles = grouped_tiles(v, tokens);
  return low_bytes(v, tiles) + (size_t)tiles * (kTile + 1) * sizeof(int32_t);
}

hipError_t launch_lora(const LoraView& v, LoraArgs a, void* workspace, hipStream_t stream) {
  const std::integral_constant<int, 1> c1;
  const std::integral_constant<int, 2> c2;
  const std::integral_constant<int, 3> c3;
  const std::integral_constant<int, 4> c4;
  const std::integral_constant<int, 8> c8;
  auto by_rank = [&](auto fn) {
    if (v.rank == 16)
      fn(c1);
    else if (v.rank == 32)
      fn(c2);
    else if (v.rank == 64)
      fn(c4);
    else
      fn(c8);
  };
  const bool copies = a.base != a.out;
  if (a.tokens <= kBothTokens) {
    const int tiles = (a.tokens + kTile - 1) / kTile;
    const int most = v.adapters < kTile ? v.adapters : kTile;
    const int slots = (a.tokens < most ? a.tokens : most) + (copies ? 1 : 0);
    // more columns per workgroup once these are more than run at a time, had the tile all
    // adapters that it could have (64 tokens of 24 adapters, 4096 columns: 16.8 us, with 512
    // columns each 27.2)
    int chunks = 0, per_wave = 1;
    for (;; per_wave *= 2) {
      chunks = 0;
      for (int p = 0, begin = 0; p < v.parts; begin = v.part_end[p++])
        chunks += (v.part_end[p] - begin + 8 * per_wave - 1) / (8 * per_wave);
      if (tiles * slots * chunks <= 256 || chunks == v.parts) break;
    }
    by_rank([&](auto ks) {
      hipLaunchKernelGGL((both_kernel<decltype(ks)::value>), dim3(tiles * slots, chunks), dim3(512), 0, stream, v, a,
                         slots, per_wave);
    });
    return hipGetLastError();
  }
  const int tiles = grouped_tiles(v, a.tokens);
  a.low = (uint16_t*)workspace;
  a.order = (int32_t*)((uint8_t*)workspace + low_bytes(v, tiles));
  a.tile_adapter = a.order + (size_t)tiles * kTile;
  hipLaunchKernelGGL(group_kernel, dim3(1), dim3(kGroupThreads), 0, stream, v, a, tiles, copies);
  const unsigned groups = (unsigned)tile_groups(tiles);
  auto shrink = [&](auto mb, auto kwaves) {
    constexpr int MB = decltype(mb)::value, KW = decltype(kwaves)::value;
    hipLaunchKernelGGL((shrink_kernel<MB, KW>), dim3(groups, (v.row_blocks + MB - 1) / MB), dim3(KW * 64), 0, stream, v,
                       a, tiles);
  };
  // (fewer blocks at a time read x more often, but fill the card: 256 tokens, 3 parts of
  // rank 64, 20.4 us by one block and 24.9 by three; 2048 tokens, 3 parts of rank 16,
  // 25.2 and 27.6; 4096 tokens of rank 64 63.7 and 60.8)
  if (tiles <= 128 || v.row_blocks == 1)
    shrink(c1, c8);
  else if (v.row_blocks == 2)
    shrink(c2, c8);
  else
    shrink(c3, c4);
  // (256 tokens: 19.4 us with one turn, 19.9 with two; 8192 tokens 63 and 56 us of
  // this launch)
  const int per_wave = tiles <= 64 ? 1 : kTurns;
  const dim3 grid(groups, (v.columns / 64 + 4 * per_wave - 1) / (4 * per_wave));
  by_rank([&](auto ks) {
    hipLaunchKernelGGL((expand_kernel<decltype(ks)::value>), grid, dim3(256), 0, stream, v, a, tiles, per_wave);
  });
  return hipGetLastError();
}

}  // namespace nkt
