// Eviction from the paged cache by weight: which tokens of a sequence stay, per
// key / value head, and moving them into the places of those that do not.
#include "nkt_attn_device.h"

namespace nkt {

namespace {

constexpr int kSelectThreads = 1024;
constexpr int kWaves = kSelectThreads / 64;
constexpr int kBins = 4096;  // of the first 12 bits of a key; then 1024 and 1024
constexpr int kMoveThreads = 256;
constexpr int kRowLanes = 16;  // lanes per moved token

// Per (sequence, head) in the workspace: the head (Moves), then the moves' sources
// and destinations.
constexpr int kHead = 4;
__host__ __device__ __forceinline__ int64_t most_moves(int max_len) { return max_len / 2 + 1; }
__host__ __device__ __forceinline__ int64_t moves_row(int max_len) { return kHead + 2 * most_moves(max_len); }

// A weight as bits in its order: larger weights are larger numbers, the zeros are
// one number, a NaN is below all.
__device__ __forceinline__ uint32_t key_of(float w) {
  const uint32_t u = __float_as_uint(w + 0.0f);
  return w != w ? 0u : u >> 31 ? ~u : u | 0x80000000u;
}

// What the waves before this one counted (v: this wave's, the same in all lanes), and all.
// s_sums is free at the call before last.
__device__ __forceinline__ int waves_before(int v, int* s_sums, int* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (lane == 0) s_sums[wave] = v;
  lds_barrier();
  const int upto = wave_inclusive_scan(lane < kWaves ? s_sums[lane] : 0);
  *total = __builtin_amdgcn_readlane(upto, kWaves - 1);
  return wave == 0 ? 0 : __builtin_amdgcn_readlane(upto, __builtin_amdgcn_readfirstlane(wave) - 1);
}

// ---------------------------------------------------------------------------
// The selection of one (sequence, head), by a workgroup: the `front` largest of its C
// candidates by a radix selection on the keys (three histograms of 12, 10 and 10
// bits), the moves in order of position, and the weights of what stays.  A wave holds
// a run of the positions, N keys per lane (N = 0: read again for each pass).
// Bound by latency: barriers, LDS additions and scans of one workgroup.  30011 tokens
// with N = 32 35 us, read again 41; 8190 tokens with N = 8 16.6 us, with N = 32 22,
// read again 19.6.
// ---------------------------------------------------------------------------
struct Moves {
  int count;   // of tokens into the places of evicted ones
  int C, front, keep;  // tokens C .. go to front .. keep - 1 (C = front: none)
  int32_t* from;
  int32_t* to;
};

struct SelectLds {
  int bins[kBins];
  int sums[6][kWaves];
  int found[3];
};

template <int N>
__device__ __forceinline__ Moves select_tokens(const CacheView& c, const EvictArgs& e, int b, int h, SelectLds& lds) {
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const float* w = e.weights + b * e.seq_stride + h * e.head_stride;
  float* out = e.out + b * e.out_seq_stride + h * e.out_head_stride;
  int32_t* head = e.moves + ((int64_t)b * c.kv_heads + h) * moves_row(e.max_len);
  int32_t* from = head + kHead;
  int32_t* to = from + most_moves(e.max_len);
  const int len = e.lens[b], budget = e.budgets[b];
  const int64_t table = (int64_t)e.width << c.page_shift;
  int most = table < e.max_len ? (int)table : e.max_len;
  most = most < e.weights_width ? most : e.weights_width;
  const bool fits = len >= 0 && len <= most && budget >= 0;
  if (!fits && h == 0 && tid == 0) report(c.status, budget < 0 ? kBadKept : kBadLength);
  const int keep = !fits || budget > len ? len : budget;
  if (h == 0 && tid == 0) e.lens_out[b] = keep;
  const int window = keep < e.recent ? keep : e.recent;
  const int C = len - window, front = keep - window;
  if (!fits || keep == len) {
    const int stays = fits ? len : e.weights_width;
    for (int i = tid; i < e.weights_width; i += kSelectThreads) out[i] = i < stays ? w[i] : 0.f;
    return {0, 0, 0, 0, from, to};
  }

  // (front < C) the wave's positions
  const int run = (C + kSelectThreads - 1) / kSelectThreads * 64;
  const int p0 = wave * run, p1 = p0 + run < C ? p0 + run : C;
  uint32_t keys[N > 0 ? N : 1];
  if (N > 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int p = p0 + i * 64 + lane;
      keys[i] = p < p1 ? __float_as_uint(w[p]) : 0u;
    }
  }
  for (int i = tid; i < kBins; i += kSelectThreads) lds.bins[i] = 0;
  if (N > 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) keys[i] = key_of(__uint_as_float(keys[i]));
  }
  lds_barrier();
  // fn(position, key, the lane has one) over the wave's positions, 64 at a time
  auto each = [&](auto fn) __attribute__((always_inline)) {
    if constexpr (N > 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (p0 + i * 64 < p1) fn(p0 + i * 64 + lane, keys[i], p0 + i * 64 + lane < p1);
      }
    } else {
      for (int p = p0; p < p1; p += 8 * 64) {
        float x[8];  // (asked for together)
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = p + i * 64 + lane < p1 ? w[p + i * 64 + lane] : 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (p + i * 64 < p1) fn(p + i * 64 + lane, key_of(x[i]), p + i * 64 + lane < p1);
      }
    }
  };

  // The threshold: keys above it stay, and `ties` of those that are equal.
  uint32_t threshold = 0xffffffffu;
  int ties = 0, equals = 0;
  int total;
  if (front > 0) {
    uint32_t prefix = 0;
    int want = front;  // of the keys that share the prefix
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 20 : pass == 1 ? 10 : 0;
      const int bins = pass == 0 ? kBins : 1024;
      each([&](int, uint32_t key, bool real) __attribute__((always_inline)) {
        const bool counts = real && (pass == 0 || (key >> (pass == 1 ? 20 : 10)) == prefix);
        const int digit = (int)(key >> shift) & (bins - 1);
        // (many weights of one number, as zeros are: one addition for all of them)
        const uint64_t all = __ballot(counts);
        if (all == 0) return;
        const int lead = __builtin_ctzll(all);
        const bool same = counts && digit == __builtin_amdgcn_readlane(digit, lead);
        const int sames = __popcll(__ballot(same));
        if (sames >= 8) {
          if (lane == lead) atomicAdd(&lds.bins[digit], sames);
          if (counts && !same) atomicAdd(&lds.bins[digit], 1);
        } else if (counts) {
          atomicAdd(&lds.bins[digit], 1);
        }
      });
      lds_barrier();
      // thread t looks at bins from the top, 4 or 1 of them
      const int mine = bins / kSelectThreads;
      const int top = bins - 1 - tid * mine;
      int sum = 0;
      for (int i = 0; i < mine; ++i) sum += lds.bins[top - i];
      const int upto = wave_inclusive_scan(sum);
      int above = waves_before(__builtin_amdgcn_readlane(upto, 63), lds.sums[pass], &total) + upto - sum;
      if (above < want && above + sum >= want) {
        int i = 0;
        while (above + lds.bins[top - i] < want) above += lds.bins[top - i++];
        lds.found[0] = top - i;
        lds.found[1] = above;
        lds.found[2] = lds.bins[top - i];
      }
      lds_barrier();
      prefix = prefix << (pass == 0 ? 12 : 10) | (uint32_t)lds.found[0];
      want -= lds.found[1];
      equals = lds.found[2];
      if (pass < 2) {
        lds.bins[tid] = 0;
        lds_barrier();
      }
    }
    threshold = prefix;
    ties = want;
  }
  // Ranks in order of position: of equal keys where not all of them stay, then of holes
  // and of what fills them.
  const uint64_t below = (1ull << lane) - 1;
  int tie = 0;
  if (ties < equals) {
    int equal = 0;
    each([&](int, uint32_t key, bool real) __attribute__((always_inline)) {
      equal += __popcll(__ballot(real && key == threshold));
    });
    tie = waves_before(equal, lds.sums[3], &total);
  }
  auto stays = [&](uint32_t key, bool real, int& rank) __attribute__((always_inline)) {
    if (ties == equals) return real && front > 0 && key >= threshold;
    const bool is_tie = real && front > 0 && key == threshold;
    const uint64_t all = __ballot(is_tie);
    const bool yes = real && front > 0 && (key > threshold || (is_tie && rank + __popcll(all & below) < ties));
    rank += __popcll(all);
    return yes;
  };
  int holes = 0, fills = 0, rank = tie;
  each([&](int p, uint32_t key, bool real) __attribute__((always_inline)) {
    const bool yes = stays(key, real, rank);
    holes += __popcll(__ballot(real && !yes && p < front));
    fills += __popcll(__ballot(yes && p >= front));
  });
  int hole = waves_before(holes, lds.sums[4], &total);
  int fill = waves_before(fills, lds.sums[5], &total);
  rank = tie;
  each([&](int p, uint32_t key, bool real) __attribute__((always_inline)) {
    const bool yes = stays(key, real, rank);
    const bool is_hole = real && !yes && p < front, is_fill = yes && p >= front;
    const uint64_t hs = __ballot(is_hole), fs = __ballot(is_fill);
    if (is_hole) to[hole + __popcll(hs & below)] = p;
    if (is_fill) from[fill + __popcll(fs & below)] = p;
    hole += __popcll(hs);
    fill += __popcll(fs);
  });
  // The weights: what stays where it is, what moves, the window, zeros.  (out may
  // be w: nothing is written before all that lies there has been read.)
  if (out != w)
    for (int i = tid; i < front; i += kSelectThreads) out[i] = w[i];
  __syncthreads();
  for (int i = tid; i < total; i += kSelectThreads) out[to[i]] = w[from[i]];
  // (the window's first tokens: read beside those)
  float x = tid < window ? w[C + tid] : 0.f;
  __syncthreads();
  for (int i0 = 0; i0 < window; i0 += kSelectThreads) {
    if (i0 > 0) {
      x = i0 + tid < window ? w[C + i0 + tid] : 0.f;
      __syncthreads();
    }
    if (i0 + tid < window) out[front + i0 + tid] = x;
  }
  // (what is behind the kept ones was read before the last barrier)
  for (int i = keep + tid; i < e.weights_width; i += kSelectThreads) out[i] = 0.f;
  return {total, C, front, keep, from, to};
}

__device__ __forceinline__ int64_t slot_at(const CacheView& c, const EvictArgs& e, int b, int p) {
  const int64_t page = e.table[(int64_t)b * e.width + (p >> c.page_shift)];
  if (page < 0 || page >= c.num_pages) {
    report(c.status, kBadPage);
    return -1;
  }
  return (page << c.page_shift) | (p & ((1 << c.page_shift) - 1));
}

__device__ __forceinline__ int64_t lane_value(int64_t v, int lane) {
  return ((int64_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32) |
         (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}

// ---------------------------------------------------------------------------
// Values move by units of U tokens, the 16-byte pieces of the value layout: a wave
// holds one dimension's piece of the unit in each lane (two of D = 128), puts the
// moved tokens' values into it and writes it back whole.
// ---------------------------------------------------------------------------
template <int D, bool I8>
struct Unit {
  static constexpr int U = I8 ? 16 : 8;
  static constexpr int kPieces = D / 64;
  u32x4 w[kPieces];

  // where a token's unit begins, in bytes of the values
  static __device__ __forceinline__ int64_t base(const CacheView& c, int64_t slot, int h) {
    const int off = (int)slot & ((1 << c.page_shift) - 1) & ~(U - 1);
    return (block_of(c, slot >> c.page_shift, h) + off * D) * (I8 ? 1 : 2);
  }
  // The unit at `to`, whose first place is `begin`, and into it the tokens of the lanes
  // whose place lies in it: lane's token is number `at` of the unit at `from`.
  __device__ __forceinline__ void read(const CacheView& c, int64_t to, int lane, int begin, int place, int64_t from,
                                       int at) {
    constexpr int kBytes = I8 ? 1 : 2;
#pragma unroll
    for (int j = 0; j < kPieces; ++j) w[j] = *((const u32x4*)(c.v + to) + lane + 64 * j);
    const int64_t word = from + (at * kBytes & ~3);  // the word that holds it, of dimension 0
    const uint32_t byte = at * kBytes & 3;
    // all that moves here is asked for before any of it is put in place
    uint32_t x[U][kPieces], select[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const uint64_t who = __ballot(place == begin + i);
      select[i] = 0x07060504u;  // (the word as it is)
#pragma unroll
      for (int j = 0; j < kPieces; ++j) x[i][j] = 0;
      if (who) {
        const int l = __builtin_ctzll(who);
        const uint8_t* src = c.v + lane_value(word, l);
#pragma unroll
        for (int j = 0; j < kPieces; ++j) x[i][j] = *(const uint32_t*)(src + (lane + 64 * j) * 16);
        const uint32_t b = __builtin_amdgcn_readlane(byte, l);
        const int sh = i * kBytes % 4 * 8;
        select[i] = I8 ? (select[i] & ~(0xffu << sh)) | b << sh : (select[i] & ~(0xffffu << sh)) | (b | (b + 1) << 8) << sh;
      }
    }
#pragma unroll
    for (int i = 0; i < U; ++i)
#pragma unroll
      for (int j = 0; j < kPieces; ++j)
        w[j][i * kBytes / 4] = __builtin_amdgcn_perm(w[j][i * kBytes / 4], x[i][j], select[i]);
  }
  __device__ __forceinline__ void write(const CacheView& c, int64_t to, int lane) const {
#pragma unroll
    for (int j = 0; j < kPieces; ++j) *((u32x4*)c.v + lane + to / 16 + 64 * j) = w[j];
  }
};

// 1 / 16 of a key's bytes.
template <int D, bool I8>
struct KeyPart {
  static constexpr int kWords = D * (I8 ? 1 : 2) / (4 * kRowLanes);
  typedef uint32_t Words __attribute__((ext_vector_type(kWords)));
  static __device__ __forceinline__ Words* at(const CacheView& c, int64_t slot, int h, int l) {
    const int off = (int)slot & ((1 << c.page_shift) - 1);
    return (Words*)(c.k + (block_of(c, slot >> c.page_shift, h) + off * D) * (I8 ? 1 : 2)) + l;
  }
};

// The moves into evicted places, by a workgroup of WAVES waves: moves first, first +
// step ... on, kGroup at a time.  Destinations lie before `front`, sources at or past
// it, so groups are independent of each other; the moves into one unit are one wave's,
// that of the group which the first of them lies in.  A token's value lies in D pieces
// 16 bytes apart, of which a unit's other tokens have the rest: units are read and written
// whole.  64 sequences of up to 8190 tokens to 2500, 4 heads, int8: 101 us, 217 MB of
// HBM and about 0.9 GB through the L2, bound by the latency of its short reads; more
// waves per SIMD (fewer registers) took 126 us, two units at a time 104.
constexpr int kGroup = 48;  // (and up to 16 more that belong to the last one's unit)

template <int D, bool I8, int WAVES>
__device__ __forceinline__ void move_tokens(const CacheView& c, const EvictArgs& e, int b, int h, const Moves& m,
                                            int first, int step) {
  constexpr int U = Unit<D, I8>::U;
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  for (int g = first; g < m.count; g += step) {
    const int i = g + lane;
    const bool real = i < m.count;
    const int place = m.to[real ? i : m.count - 1], source = m.from[real ? i : m.count - 1];
    const int before = i > 0 && real ? m.to[i - 1] : -U;
    int64_t src = slot_at(c, e, b, source);
    const int64_t dst = slot_at(c, e, b, place);
    if (dst < 0) src = -1;
    const int64_t unit_to = Unit<D, I8>::base(c, dst < 0 ? 0 : dst, h);
    const int64_t unit_from = Unit<D, I8>::base(c, src < 0 ? 0 : src, h);
    const int moves_to = real && src >= 0 ? place : -1;
    // keys and scales
    constexpr int kRows = WAVES * 4, kTurns = (kGroup + kRows - 1) / kRows;
    const int l = lane % kRowLanes;
    typename KeyPart<D, I8>::Words k[kTurns];
    int64_t row_src[kTurns], row_dst[kTurns];
#pragma unroll
    for (int j = 0; j < kTurns; ++j) {
      const int row = j * kRows + wave * 4 + lane / kRowLanes;
      const int r = row < 64 ? row : 63;
      row_src[j] = ((int64_t)__shfl((int)(src >> 32), r) << 32) | (uint32_t)__shfl((int)src, r);
      row_dst[j] = ((int64_t)__shfl((int)(dst >> 32), r) << 32) | (uint32_t)__shfl((int)dst, r);
      if (row >= kGroup || g + row >= m.count) row_src[j] = -1;
      if (row_src[j] >= 0) k[j] = *KeyPart<D, I8>::at(c, row_src[j], h, l);
    }
    const bool scales = I8 && wave == 0 && lane < kGroup && real && src >= 0;
    float ks = 0.f, vs = 0.f;
    if (scales) {
      ks = c.k_scales[scale_of(c, src, h)];
      vs = c.v_scales[scale_of(c, src, h)];
    }
    // values: the wave's units
    uint64_t firsts = __ballot(real && lane < kGroup && place / U != before / U);
    for (int n = 0; firsts; ++n) {
      const int at = __builtin_ctzll(firsts);
      firsts &= firsts - 1;
      if (n % WAVES != wave) continue;
      const int unit = __builtin_amdgcn_readlane(place, at) / U;
      if (lane_value(dst, at) < 0) continue;
      const int64_t to = lane_value(unit_to, at);
      Unit<D, I8> t;
      t.read(c, to, lane, unit * U, moves_to, unit_from, (int)src & (U - 1));
      t.write(c, to, lane);
    }
#pragma unroll
    for (int j = 0; j < kTurns; ++j)
      if (row_src[j] >= 0) *KeyPart<D, I8>::at(c, row_dst[j], h, l) = k[j];
    if (scales) {
      c.k_scales[scale_of(c, dst, h)] = ks;
      c.v_scales[scale_of(c, dst, h)] = vs;
    }
  }
}

// The window, behind the rest: it only moves towards the front, so a token still to
// be read lies past every one written before it.  A unit per wave at a time, each
// read whole (by all waves) before any of it is written.  256 tokens, bf16: 13 us, a
// launch and a chain of two turns.
template <int D, bool I8, int WAVES>
__device__ __forceinline__ void move_window(const CacheView& c, const EvictArgs& e, int b, int h, const Moves& m) {
  constexpr int U = Unit<D, I8>::U;
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int l = lane % kRowLanes;
  for (int p0 = m.front / U * U; p0 < m.keep; p0 += WAVES * U) {
    // lane i < U: place p + i of the wave's unit
    const int p = p0 + wave * U;
    const int begin = p < m.front ? m.front - p : 0;
    const int count = (m.keep - p < U ? m.keep - p : U) - begin;  // tokens of the window from place `begin` on
    const bool real = lane >= begin && lane < begin + count;
    int64_t src = -1;
    const int64_t dst = count > 0 ? slot_at(c, e, b, p) : -1;
    if (real && dst >= 0) src = slot_at(c, e, b, m.C + p + lane - m.front);
    const int64_t to = Unit<D, I8>::base(c, dst < 0 ? 0 : dst, h);
    const int64_t from = Unit<D, I8>::base(c, src < 0 ? 0 : src, h);
    Unit<D, I8> t;
    typename KeyPart<D, I8>::Words k[U / 4];
    int64_t row_src[U / 4];
    float ks = 0.f, vs = 0.f;
    if (dst >= 0) {
      t.read(c, to, lane, 0, src < 0 ? -1 : lane, from, (int)src & (U - 1));
#pragma unroll
      for (int j = 0; j < U / 4; ++j) {
        const int r = j * 4 + lane / kRowLanes;
        row_src[j] = ((int64_t)__shfl((int)(src >> 32), r) << 32) | (uint32_t)__shfl((int)src, r);
        if (row_src[j] >= 0) k[j] = *KeyPart<D, I8>::at(c, row_src[j], h, l);
      }
      if (I8 && src >= 0) {
        ks = c.k_scales[scale_of(c, src, h)];
        vs = c.v_scales[scale_of(c, src, h)];
      }
    }
    __syncthreads();
    if (dst >= 0) {
      t.write(c, to, lane);
#pragma unroll
      for (int j = 0; j < U / 4; ++j)
        if (row_src[j] >= 0) *KeyPart<D, I8>::at(c, dst + j * 4 + lane / kRowLanes, h, l) = k[j];
      if (I8 && src >= 0) {
        c.k_scales[scale_of(c, dst + lane, h)] = ks;
        c.v_scales[scale_of(c, dst + lane, h)] = vs;
      }
    }
  }
}

__device__ __forceinline__ Moves moves_of(const CacheView& c, const EvictArgs& e, int pair) {
  int32_t* head = e.moves + pair * moves_row(e.max_len);
  Moves m;
  m.count = head[0];
  m.C = head[1];
  m.front = head[2];
  m.keep = head[3];
  m.from = head + kHead;
  m.to = m.from + most_moves(e.max_len);
  return m;
}

// The whole of it by one workgroup per (sequence, head), for sequences of up to 4096 tokens.
// Calls in us, in one launch and in three, 4 heads: one sequence of 2112 tokens to 2048 20
// and 25, of 4096 to 4032 21 and 26, 64 of them (bf16) 27 and 78; but one of 1024 to 512 23
// and 18, of 4096 to 1024 49 and 22, 16 of these 55 and 38, 64 of these 91 and 94 (int8 61
// and 58), of 1024 to 512 31 and 37.  A program that evicts as it goes moves few tokens at a
// time; where a whole prompt is cut at once, sixteen waves per head do what the three launches
// give to the whole card, and lose until there are sequences enough.
template <int D, bool I8, int N>
__global__ __launch_bounds__(kSelectThreads) void evict_kernel(CacheView c, EvictArgs e) {
  __shared__ SelectLds lds;
  const int b = (int)(blockIdx.x / (unsigned)c.kv_heads), h = (int)(blockIdx.x % (unsigned)c.kv_heads);
  const Moves m = select_tokens<N>(c, e, b, h, lds);
  if (m.C == m.front) return;
  move_tokens<D, I8, kWaves>(c, e, b, h, m, 0, kGroup);
  __syncthreads();
  move_window<D, I8, kWaves>(c, e, b, h, m);
}

template <int N>
__global__ __launch_bounds__(kSelectThreads) void select_kernel(CacheView c, EvictArgs e) {
  __shared__ SelectLds lds;
  const int b = (int)(blockIdx.x / (unsigned)c.kv_heads), h = (int)(blockIdx.x % (unsigned)c.kv_heads);
  const Moves m = select_tokens<N>(c, e, b, h, lds);
  if (threadIdx.x == 0) {
    int32_t* head = e.moves + (int64_t)blockIdx.x * moves_row(e.max_len);
    head[0] = m.count;
    head[1] = m.C;
    head[2] = m.front;
    head[3] = m.keep;
  }
}

template <int D, bool I8>
__global__ __launch_bounds__(kMoveThreads) void fill_kernel(CacheView c, EvictArgs e, int groups) {
  const int pair = (int)(blockIdx.x / (unsigned)groups), group = (int)(blockIdx.x % (unsigned)groups);
  const int b = (int)((unsigned)pair / (unsigned)c.kv_heads), h = (int)((unsigned)pair % (unsigned)c.kv_heads);
  const Moves m = moves_of(c, e, pair);
  move_tokens<D, I8, kMoveThreads / 64>(c, e, b, h, m, group * kGroup, groups * kGroup);
}

template <int D, bool I8>
__global__ __launch_bounds__(1024) void window_kernel(CacheView c, EvictArgs e) {
  const int b = (int)(blockIdx.x / (unsigned)c.kv_heads), h = (int)(blockIdx.x % (unsigned)c.kv_heads);
  const Moves m = moves_of(c, e, (int)blockIdx.x);
  if (m.C == m.front) return;
  move_window<D, I8, 1024 / 64>(c, e, b, h, m);
}

}  // namespace

size_t evict_workspace_bytes(const CacheView& c, int seqs, int max_len) {
  return (size_t)seqs * c.kv_heads * moves_row(max_len) * sizeof(int32_t);
}

hipError_t launch_evict(const CacheView& c, const EvictArgs& e, hipStream_t stream) {
  const unsigned pairs = (unsigned)e.seqs * c.kv_heads;
  const dim3 grid(pairs), threads(kSelectThreads);
  const std::integral_constant<int, 4> four;
  if (e.max_len <= decltype(four)::value * kSelectThreads) {
    by_layout(c, [&](auto dim, auto int8) {
      hipLaunchKernelGGL((evict_kernel<decltype(dim)::value, decltype(int8)::value, decltype(four)::value>), grid,
                         threads, 0, stream, c, e);
    });
    return hipGetLastError();
  }
  if (e.max_len <= 8 * kSelectThreads)
    hipLaunchKernelGGL(select_kernel<8>, grid, threads, 0, stream, c, e);
  else if (e.max_len <= 32 * kSelectThreads)
    hipLaunchKernelGGL(select_kernel<32>, grid, threads, 0, stream, c, e);
  else
    hipLaunchKernelGGL(select_kernel<0>, grid, threads, 0, stream, c, e);
  // about 4096 workgroups (of one sequence of 30011 tokens, 8 heads, the fill takes
  // 16 us; with 2048 workgroups 20)
  int64_t groups = (most_moves(e.max_len) + kGroup - 1) / kGroup;
  const int64_t share = (4096 + pairs - 1) / pairs;
  if (groups > share) groups = share;
  by_layout(c, [&](auto dim, auto int8) {
    constexpr int D = decltype(dim)::value;
    constexpr bool I8 = decltype(int8)::value;
    hipLaunchKernelGGL((fill_kernel<D, I8>), dim3(pairs * (unsigned)groups), dim3(kMoveThreads), 0, stream, c, e,
                       (int)groups);
    hipLaunchKernelGGL((window_kernel<D, I8>), dim3(pairs), dim3(1024), 0, stream, c, e);
  });
  return hipGetLastError();
}

}  // namespace nkt
