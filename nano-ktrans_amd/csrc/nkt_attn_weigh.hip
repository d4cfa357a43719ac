// What each cached token got of the attention's weights: the second pass over
// the keys behind a forward call that kept its rows' maxima and sums.
#include "nkt_attn_device.h"

namespace nkt {

namespace {

constexpr int kThreads = 256;
constexpr int kWaveTokens = 64;
constexpr int kBlockTokens = 4 * kWaveTokens;
constexpr int kStepRows = 32;

// Past this a row's maximum (log2) is told again (recount_kernel).  The attention
// kernels move their running maximum by rounded steps, each off by 2^-24 of it at
// most: up to 512 that is 2^-15, a factor of 2^-15 on the row's weights, which a
// score of that size has from its own fp32 sum as well.  From 2^24 on it would be
// whole powers of two.
constexpr float kRecountFrom = 512.0f;

__device__ __forceinline__ bool recounts(float m, float l) {
  return !(__builtin_fabsf(m) < kRecountFrom) && !(l == 0.f);  // (NaN, infinity: told again, with the same end)
}

// A wave's operands.  The order of the dimensions within a product is free, so a
// lane's fragments are the 16-byte pieces that it loads: bf16 fragment i holds
// dimensions 16 i + 8 half on, int8 fragments 2 j and 2 j + 1 the piece at
// 32 j + 16 half.
template <int D, bool I8>
__device__ __forceinline__ void load_query(const uint16_t* q, int half, u32x4* f) {
#pragma unroll
  for (int i = 0; i < D / 16; ++i)
    f[i] = *(const u32x4*)(q + (I8 ? (i >> 1) * 32 + half * 16 + (i & 1) * 8 : i * 16 + half * 8));
}
// keys of 32 tokens, the lane's one `col`; at: place of the first one in the cache
template <int D, bool I8>
__device__ __forceinline__ void load_keys(const CacheView& c, int64_t at, int col, int half, u32x4* f) {
  if (!I8) {
    const uint16_t* src = (const uint16_t*)c.k + (at + col) * D + half * 8;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) f[i] = *(const u32x4*)(src + i * 16);
  } else {
    const uint8_t* src = c.k + (at + col) * D + half * 16;
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
      const u32x4 w = *(const u32x4*)(src + j * 32);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        uint32_t lo, hi;
        bf16_of_codes(w[x], &lo, &hi);
        f[2 * j + (x >> 1)][2 * (x & 1)] = lo;
        f[2 * j + (x >> 1)][2 * (x & 1) + 1] = hi;
      }
    }
  }
}
// of token (v & 3) + 8 (v >> 2) + 4 half in register v: what its product is
// multiplied by to give a score in log2
template <bool I8>
__device__ __forceinline__ f32x16 score_factors(const CacheView& c, int64_t at, int half, float scale2) {
  f32x16 f;
#pragma unroll
  for (int v = 0; v < 16; v += 4) {
    f32x4 x = {scale2, scale2, scale2, scale2};
    if (I8) x = *(const f32x4*)(c.k_scales + at + 8 * (v >> 2) + 4 * half) * scale2;
#pragma unroll
    for (int j = 0; j < 4; ++j) f[v + j] = x[j];
  }
  return f;
}
template <int D>
__device__ __forceinline__ f32x16 products(const u32x4* k, const u32x4* q) {
  f32x16 st;
#pragma unroll
  for (int v = 0; v < 16; ++v) st[v] = 0.f;
#pragma unroll
  for (int i = 0; i < D / 16; ++i) st = mfma32_bf16(k[i], q[i], st);
  return st;
}

// The page of position p as a place in the cache (tokens of all heads' blocks), -1: none.
__device__ __forceinline__ int64_t place_of(const CacheView& c, const AttnArgs& a, int b, int h, int p) {
  const int entry = p >> c.page_shift;
  const int page = entry < a.width ? __builtin_amdgcn_readfirstlane(a.table[(int64_t)b * a.width + entry]) : -1;
  if (page < 0 || page >= c.num_pages) return -1;
  return (((int64_t)page * c.kv_heads + h) << c.page_shift) + (p & ((1 << c.page_shift) - 1));
}

// Where a row of a head lies among rows of q (token after token, all heads), and its
// head of the group, moved 32 rows at a time without a division.
struct Row {
  int place, g;
  __device__ __forceinline__ Row() {}
  __device__ __forceinline__ Row(int row, int G, int heads) : place(row / G * heads + row % G), g(row % G) {}
  // EVEN: G divides 32, the head stays
  template <bool EVEN>
  __device__ __forceinline__ void next(int places, int heads_on, int G, int wrap) {
    place += places;
    if (EVEN) return;
    g += heads_on;
    const bool over = g >= G;
    g -= over ? G : 0;
    place += over ? wrap : 0;
  }
};

// ---------------------------------------------------------------------------
// The rows' statistics as weigh_kernel takes them: maximum and 1 / sum, (0, 0) for a
// row that saw nothing.  One workgroup per 256 rows of a head.  Rows whose maximum is
// past kRecountFrom (broken or extreme inputs) get both from rounded scores again,
// 32 rows at a time: the waves take 32 tokens in turn.  5 us, a launch's latency, where
// there is none of them.
// ---------------------------------------------------------------------------
constexpr int kStatRows = 256;

template <int D, bool I8>
__global__ __launch_bounds__(kThreads) void recount_kernel(CacheView c, WeighArgs w, int row_blocks) {
  const AttnArgs& a = w.attn;
  __shared__ float s_m[4][2][32], s_l[4][2][32];
  __shared__ int s_again[kStatRows / kStepRows];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int half = lane >> 5, col = lane & 31;
  const int HK = c.kv_heads, G = a.heads / HK;
  const int h = (int)(blockIdx.x % (unsigned)HK);
  const int rest = (int)(blockIdx.x / (unsigned)HK);
  const int b = rest / row_blocks;
  const Seq s = sequence(c, a, b, sequence_words(a, b), false);
  const int first = s.n > w.last ? s.n - w.last : 0;
  const int rows = (s.n - first) * G;
  const int r0 = rest % row_blocks * kStatRows;
  if (r0 >= rows) return;
  auto at_row = [&](int row) {
    return (int64_t)(s.first + first + row / G) * a.heads + h * G + row % G;
  };
  auto keep = [&](float* to, float m, float l) {
    to[0] = l == 0.f ? 0.f : m;
    to[1] = l == 0.f ? 0.f : 1.0f / l;
  };
  {
    const int row = r0 + tid;
    bool again = false;
    if (row < rows) {
      float* stats = a.stats + 2 * at_row(row);
      const float m = stats[0], l = stats[1];
      again = recounts(m, l);
      if (!again) keep(stats, m, l);
    }
    const uint64_t any = __ballot(again);
    if (lane == 0) {
      s_again[2 * wave] = (uint32_t)any != 0;
      s_again[2 * wave + 1] = (uint32_t)(any >> 32) != 0;
    }
  }
  __syncthreads();
  if (tid == 0) {
    int any = 0;
#pragma unroll
    for (int i = 0; i < kStatRows / kStepRows; ++i) any |= s_again[i];
    w.extreme[((int64_t)b * HK + h) * row_blocks + rest % row_blocks] = any;
  }
  const float scale2 = a.scale * kLog2e;
  for (int block = 0; block < kStatRows / kStepRows; ++block) {
    if (!s_again[block]) continue;
    const int rb = r0 + block * kStepRows;
    const int row = rb + col < rows ? rb + col : rows - 1;
    float* stats = a.stats + 2 * at_row(row);
    u32x4 q[D / 16];
    load_query<D, I8>(a.q + at_row(row) * D, half, q);
    const int past = s.context + first + row / G;  // the last position that the row sees
    const int last_row = rb + kStepRows - 1 < rows ? rb + kStepRows - 1 : rows - 1;
    const int row_end = s.context + first + last_row / G + 1;
    const int end = row_end < s.len ? row_end : s.len;
    float m = -__builtin_huge_valf(), l = 0.f;
    for (int p = wave * 32; p < end; p += 128) {
      const int64_t at = place_of(c, a, b, h, p);
      if (at < 0) continue;
      u32x4 k[D / 16];
      load_keys<D, I8>(c, at, col, half, k);
      const f32x16 f = score_factors<I8>(c, at, half, scale2);
      f32x16 st = products<D>(k, q);
      float top = m;
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        const int pos = p + (v & 3) + 8 * (v >> 2) + 4 * half;
        st[v] = pos <= past && pos < s.len ? rounded_product(st[v], f[v]) : -__builtin_huge_valf();
        top = fmaxf(top, st[v]);
      }
      const float less = fmaxf(top, -__FLT_MAX__);
      l *= __builtin_amdgcn_exp2f(m - less);
#pragma unroll
      for (int v = 0; v < 16; ++v) l += __builtin_amdgcn_exp2f(st[v] - less);
      m = top;
    }
    __syncthreads();  // (of the rows before, the sums are read)
    s_m[wave][half][col] = m;
    s_l[wave][half][col] = l;
    __syncthreads();
    // (the other rows of the 32 have theirs already, changed: told again as well, they
    // are those of rounded scores too)
    if (tid < 32 && rb + col < rows) {
      m = s_m[0][0][col];
#pragma unroll
      for (int i = 1; i < 8; ++i) m = fmaxf(m, s_m[i >> 1][i & 1][col]);
      l = 0.f;
      const float less = fmaxf(m, -__FLT_MAX__);
#pragma unroll
      for (int i = 0; i < 8; ++i) l += s_l[i >> 1][i & 1][col] * __builtin_amdgcn_exp2f(s_m[i >> 1][i & 1][col] - less);
      keep(stats, m, l);
    }
  }
}

// ---------------------------------------------------------------------------
// Weights of 64 tokens per wave, 256 per workgroup, summed over a part of the
// rows that see them.  S = K . Q^T on 32x32x16 matrix instructions with the keys
// held in registers: a lane's column is a row and its registers are tokens, so
// that the sum over rows stays in the lane until the end, and the row's maximum
// and sum are one value per lane.  The waves share the rows: 32 at a time go
// straight into LDS, three steps ahead (one where rows may not see all tokens; chunk
// c of row r at c ^ key(r), so that the rows' same chunk lies in 16 places of the 256
// bytes that LDS reads at a time).
//
// Bound by the matrix cores and an exponential per score beside them: a prompt of
// 8192 tokens that all count, 32 / 4 heads, D = 128, bf16: 352 us, 0.78 PFLOP/s of the
// repeated product alone (kept scores would be 4.3 GB each way); three chunks of up to
// 1021 tokens on up to 9000, 32 / 8 heads, int8, of which the last 64 tokens count:
// 31 us.
// ---------------------------------------------------------------------------
template <int OFF, int CTRL>
__device__ __forceinline__ void exchange(float* x, int col) {
  const bool high = col & OFF;
#pragma unroll
  for (int v = 0; v < OFF; ++v) {
    float low_one = x[v], high_one = x[v + OFF];
    __asm__ volatile("" : "+v"(low_one), "+v"(high_one));  // (else the selection becomes one of an index)
    const float keep = high ? high_one : low_one, give = high ? low_one : high_one;
    x[v] = keep + __uint_as_float(dpp_u32<CTRL>(__float_as_uint(give)));
  }
}

template <int D>
__device__ __forceinline__ int query_key(int r) {
  return D == 128 ? r & 15 : r >> 1 & 7;
}

template <int D, bool I8, bool EVEN>
__global__ __launch_bounds__(kThreads, 2) void weigh_kernel(CacheView c, WeighArgs w) {
  constexpr int kChunks = D / 8;                      // 16-byte chunks of a row
  constexpr int kLoads = kStepRows * kChunks / 256;   // of a step, per thread
  // (arrays of their own: the compiler has a read from LDS wait for every load that may
  // go into the same one)
  constexpr int kBytes = kStepRows * D * 2;
  __shared__ __align__(1024) uint8_t s_q0[kBytes], s_q1[kBytes], s_q2[kBytes], s_q3[kBytes];
  __shared__ __align__(1024) float s_stats0[8 * kStepRows], s_stats1[8 * kStepRows], s_stats2[8 * kStepRows],
      s_stats3[8 * kStepRows];
  __shared__ __align__(16) float s_factor[I8 ? kBlockTokens : 4];  // of the tokens
  const AttnArgs& a = w.attn;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = lane >> 5, col = lane & 31;
  const int HK = c.kv_heads, G = a.heads / HK;
  const int h = (int)(blockIdx.x % (unsigned)HK);
  int rest = (int)(blockIdx.x / (unsigned)HK);
  const int block = rest % w.blocks;
  rest /= w.blocks;
  const int chunk = rest % w.chunks;
  const int b = rest / w.chunks;
  const int p = block * kBlockTokens + wave * kWaveTokens;
  const SeqWords words = sequence_words(a, b);
  const int64_t found = place_of(c, a, b, h, p);  // (asked for with the sequence's words)
  const Seq s = sequence(c, a, b, words, false);
  if (block * kBlockTokens >= s.len) return;
  const int64_t at = p < s.len ? found : -1;
  // rows: the last tokens' ones, from the first that sees the block's first position
  const int first = s.n > w.last ? s.n - w.last : 0;
  const int rows = (s.n - first) * G;
  const int end = rows < (chunk + 1) * w.chunk_rows ? rows : (chunk + 1) * w.chunk_rows;
  const int sees = block * kBlockTokens - s.context - first;  // the first token (of those counted) that does
  int r = chunk * w.chunk_rows;
  if (sees > 0 && (int64_t)sees * G > r) r = (int64_t)sees * G < end ? sees * G : end;

  f32x16 acc[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int v = 0; v < 16; ++v) acc[i][v] = 0.f;
  // (parts of the rows before, which see nothing of the block, are not added either)
  if (w.chunks > 1 && r >= end) return;
  bool extreme = false;
  for (int i = r / kStatRows; i * kStatRows < end; ++i)
    extreme |= w.extreme[((int64_t)b * HK + h) * w.row_blocks + i] != 0;
  if (r < end) {
    const float scale2 = a.scale * kLog2e;
    // (a wave without tokens reads some others')
    u32x4 k[2][D / 16];
    const int64_t keys_at = at >= 0 ? at : 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) load_keys<D, I8>(c, keys_at + 32 * i, col, half, k[i]);
    if (I8) s_factor[wave * kWaveTokens + lane] = c.k_scales[keys_at + lane] * scale2;  // (only this wave's)
    // rows of q and statistics from the sequence's first on; what lies past the rows
    // repeats the last one and is masked
    const uint16_t* const q0 = a.q + ((int64_t)(s.first + first) * a.heads + h * G) * D;
    const float* const stats0 = a.stats + 2 * ((int64_t)(s.first + first) * a.heads + h * G);
    const int last_place = (end - 1) / G * a.heads + (end - 1) % G;
    const int dt = kStepRows / G, dg = kStepRows % G;
    const int places = dt * a.heads + dg, wrap = a.heads - G;
    Row load_rows[kLoads], stat_row;
    auto start = [&] {  // the next load is of rows r on
#pragma unroll
      for (int j = 0; j < kLoads; ++j) load_rows[j] = Row(r + ((wave * kLoads + j) * 64 + lane) / kChunks, G, a.heads);
      stat_row = Row(r + (lane >> 1), G, a.heads);
    };
    auto load = [&](uint8_t* to_q, float* to_stats) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const int slot = (wave * kLoads + j) * 64 + lane;
        const int64_t x = load_rows[j].place < last_place ? load_rows[j].place : last_place;
        load16_to_lds(q0 + x * D + ((slot % kChunks) ^ query_key<D>(slot / kChunks)) * 8,
                      to_q + (wave * kLoads + j) * 1024);
        load_rows[j].template next<EVEN>(places, dg, G, wrap);
      }
      const int64_t x = stat_row.place < last_place ? stat_row.place : last_place;
      load4_to_lds(stats0 + 2 * x + (lane & 1), (uint8_t*)(to_stats + wave * 2 * kStepRows));
      stat_row.template next<EVEN>(places, dg, G, wrap);
    };
    u32x4 q[D / 16];
    // (the chunk that load_query takes, 2 i + half or 4 (i / 2) + 2 half + i % 2, at its
    // place in the row: worked out each time, there are no registers to hold them all)
    int q_at = (col * kChunks + ((I8 ? 2 * half : half) ^ query_key<D>(col))) * 16;
    auto read = [&](const uint8_t* from_q, int i) __attribute__((always_inline)) {
      if (D == 128) __asm__ volatile("" : "+v"(q_at));
      q[i] = *(const u32x4*)(from_q + (q_at ^ (I8 ? (i >> 1) * 4 + (i & 1) : 2 * i) * 16));
    };
    // what registers 4 v .. 4 v + 3 of half i's products are multiplied by (read where
    // it is needed: there are no registers to hold it)
    auto factor = [&](int i, int v) __attribute__((always_inline)) {
      if (!I8) return f32x4{scale2, scale2, scale2, scale2};
      int at4 = wave * kWaveTokens + 4 * half;
      __asm__ volatile("" : "+v"(at4));
      return *(const f32x4*)&s_factor[at4 + 32 * i + 8 * v];
    };
    f32x16 st[2];
    auto product = [&](int t, int i) __attribute__((always_inline)) {
      if (i == 0) {
#pragma unroll
        for (int v = 0; v < 16; ++v) st[t][v] = 0.f;
      }
      st[t] = mfma32_bf16(k[t][i], q[i], st[t]);
    };
    float m, inv;
    auto read_stats = [&](const float* stats) __attribute__((always_inline)) {
      m = stats[wave * 2 * kStepRows + 2 * col];
      inv = stats[wave * 2 * kStepRows + 2 * col + 1];
    };
    const int seen_from = p - s.context - first;  // the first token (of those counted) that sees the wave's first one

    // Steps whose rows may not see all tokens, whose maxima may be extreme, or that the
    // rows end in: one step's rows on the way into LDS at a time.
    auto any_steps = [&](int to) __attribute__((always_inline)) {
      auto any_step = [&](const uint8_t* now_q, const float* now_stats, uint8_t* next_q,
                          float* next_stats) __attribute__((always_inline)) {
        wait_vmem();
        lds_barrier();
        if (r + kStepRows < to) load(next_q, next_stats);
        const int left = end - r < kStepRows ? end - r : kStepRows;
        if (at >= 0 && (r + left - 1) / G >= seen_from) {  // (else none of these rows sees the wave's tokens)
#pragma unroll
          for (int i = 0; i < D / 16; ++i) read(now_q, i);
          read_stats(now_stats);
          // tokens of the lane's that its row sees: as many from 4 half on (eight apart in fours)
          int sees = col < left ? (r + col) / G - seen_from + 1 - 4 * half : -64;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int i = 0; i < D / 16; ++i) product(t, i);
#pragma unroll
            for (int v = 0; v < 16; v += 4) {
              const f32x4 f = factor(t, v >> 2);
              __asm__ volatile("" : "+v"(sees));  // (all comparisons at once would not fit the scalar registers)
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const float e = __builtin_amdgcn_exp2f(rounded_product(st[t][v + j], f[j]) - m);
                acc[t][v + j] = 32 * t + 2 * v + j < sees ? __builtin_fmaf(e, inv, acc[t][v + j]) : acc[t][v + j];
              }
            }
          }
        }
        r += kStepRows;
      };
      if (r >= to) return;
      start();
      lds_barrier();  // (of the steps before, all is read)
      load(s_q0, s_stats0);
      while (true) {
        any_step(s_q0, s_stats0, s_q1, s_stats1);
        if (r >= to) break;
        any_step(s_q1, s_stats1, s_q0, s_stats0);
        if (r >= to) break;
      }
    };

    // Steps whose rows all see all of the workgroup's tokens.  Rows go into LDS three
    // steps ahead and from there into registers one step ahead; the weights of one half
    // of the tokens are worked out beside the products of the other: half 1 with this
    // step's rows (the next one's follow into their registers), then half 0 with those.
    // (Behind the last step: the last row again, for products that nothing takes.)
    auto all_steps = [&](int to) __attribute__((always_inline)) {
      auto add = [&](auto half_of, const uint8_t* next_q) __attribute__((always_inline)) {
        constexpr int t = decltype(half_of)::value;
        constexpr int kEach = 16 / (D / 16);  // values beside a product
        f32x4 f;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          product(1 - t, i);
          if (t == 0) read(next_q, i);
#pragma unroll
          for (int v = i * kEach; v < (i + 1) * kEach; ++v) {
            if ((v & 3) == 0) f = factor(t, v >> 2);
            acc[t][v] = __builtin_fmaf(__builtin_amdgcn_exp2f(__builtin_fmaf(st[t][v], f[v & 3], -m)), inv, acc[t][v]);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      };
      auto all_step = [&](const float* stats, const uint8_t* next_q, uint8_t* free_q,
                          float* free_stats) __attribute__((always_inline)) {
        wait_vmem_but<kLoads + 1>();
        lds_barrier();
        load(free_q, free_stats);
        read_stats(stats);
        add(std::integral_constant<int, 0>{}, next_q);
        add(std::integral_constant<int, 1>{}, next_q);
        r += kStepRows;
      };
      if (r >= to) return;
      start();
      lds_barrier();  // (of the steps before, all is read)
      load(s_q0, s_stats0);
      load(s_q1, s_stats1);
      load(s_q2, s_stats2);
      wait_vmem_but<2 * (kLoads + 1)>();
      lds_barrier();
#pragma unroll
      for (int i = 0; i < D / 16; ++i) read(s_q0, i);
#pragma unroll
      for (int i = 0; i < D / 16; ++i) product(0, i);
      while (true) {
        all_step(s_stats0, s_q1, s_q3, s_stats3);
        if (r >= to) break;
        all_step(s_stats1, s_q2, s_q0, s_stats0);
        if (r >= to) break;
        all_step(s_stats2, s_q3, s_q1, s_stats1);
        if (r >= to) break;
        all_step(s_stats3, s_q0, s_q2, s_stats2);
        if (r >= to) break;
      }
      wait_vmem();  // (loads into LDS end before it is used again)
    };
    // whole steps from the first row that sees the workgroup's last token on
    int plain_from = end;
    if (!extreme) {
      const int token = sees + kBlockTokens - 1;
      const int64_t row = token > 0 ? (int64_t)token * G : 0;
      if (row < end) plain_from = row > r ? r + ((int)row - r + kStepRows - 1) / kStepRows * kStepRows : r;
    }
    if (plain_from > end - kStepRows) plain_from = end;
    any_steps(plain_from);
    if (plain_from < end) {
      all_steps(r + (end - r) / kStepRows * kStepRows);
      any_steps(end);
    }
  }
  // the sum over the 32 columns, with register `col` of the 32 left in lane col: lanes
  // that differ in a bit of it exchange the half of the registers that they do not keep
  float x[32];
#pragma unroll
  for (int v = 0; v < 16; ++v) {
    const auto t = __builtin_amdgcn_permlane16_swap(__float_as_uint(acc[0][v]), __float_as_uint(acc[1][v]), false, false);
    x[v] = __uint_as_float(t[0]) + __uint_as_float(t[1]);
  }
  exchange<8, 0x128>(x, col);  // lane ^ 8
  exchange<4, 0x141>(x, col);  // lane ^ 7
  exchange<2, 0x4e>(x, col);   // lane ^ 2
  exchange<1, 0xb1>(x, col);   // lane ^ 1
  const int pos = p + (col >> 4) * 32 + (col & 3) + 8 * ((col & 15) >> 2) + 4 * half;
  if (pos >= s.len) return;
  if (w.chunks > 1) {
    w.parts[(((int64_t)chunk * a.seqs + b) * HK + h) * ((int64_t)w.blocks * kBlockTokens) + pos] = at >= 0 ? x[0] : 0.f;
  } else if (at >= 0) {
    w.weights[b * w.seq_stride + h * w.head_stride + pos] += x[0];
  }
}

// Adds the parts of the rows to the weights, in order.  8192 tokens x 4 heads, up to 32
// parts: 10 us, most of it the chain of reads.
__global__ __launch_bounds__(kThreads) void weigh_join_kernel(CacheView c, WeighArgs w) {
  const AttnArgs& a = w.attn;
  const int HK = c.kv_heads;
  const int h = (int)(blockIdx.x % (unsigned)HK);
  const int rest = (int)(blockIdx.x / (unsigned)HK);
  const int b = rest / w.blocks;
  const int pos = rest % w.blocks * kBlockTokens + (int)threadIdx.x;
  const Seq s = sequence(c, a, b, sequence_words(a, b), false);
  if (pos >= s.len) return;
  const int64_t row = (int64_t)w.blocks * kBlockTokens;
  // the chunks with rows that see the token's block
  const int G = a.heads / HK, first = s.n > w.last ? s.n - w.last : 0;
  const int rows = (s.n - first) * G, sees = rest % w.blocks * kBlockTokens - s.context - first;
  const int64_t from = sees > 0 ? (int64_t)sees * G : 0;
  float sum = 0.f;
  for (int i = from < rows ? (int)from / w.chunk_rows : w.chunks; i < w.chunks && i * w.chunk_rows < rows; ++i)
    sum += w.parts[(((int64_t)i * a.seqs + b) * HK + h) * row + pos];
  w.weights[b * w.seq_stride + h * w.head_stride + pos] += sum;
}

struct WeighPlan {
  int blocks, chunks, chunk_rows, row_blocks;
};

WeighPlan weigh_plan(const CacheView& c, int heads, int seqs, int max_queries, int max_len, int last) {
  WeighPlan p = {};
  const int64_t rows = (int64_t)(last < max_queries ? last : max_queries) * (heads / c.kv_heads);
  p.blocks = (max_len + kBlockTokens - 1) / kBlockTokens;
  p.row_blocks = (int)((rows + kStatRows - 1) / kStatRows);
  const int64_t wgs = (int64_t)seqs * c.kv_heads * p.blocks;
  // Parts of the rows until there are about 8192 workgroups, of at least 2048 rows each
  // (8192 tokens, 32 / 4 heads, with the join, in us: 366; 2048 workgroups 390, parts of
  // 512 rows 390, whole rows 1093: the first tokens are seen by all rows).
  int64_t chunks = wgs > 0 ? (8192 + wgs - 1) / wgs : 1;
  const int64_t most = (rows + 2047) / 2048;
  if (chunks > most) chunks = most;
  if (chunks < 1) chunks = 1;
  const int64_t chunk_rows = ((rows + chunks - 1) / chunks + kStepRows - 1) / kStepRows * kStepRows;
  p.chunk_rows = (int)(chunk_rows > 0 ? chunk_rows : kStepRows);
  p.chunks = rows > 0 ? (int)((rows + p.chunk_rows - 1) / p.chunk_rows) : 1;
  return p;
}

// floats of the workspace behind the statistics: the flags, then the parts
size_t flags_of(const CacheView& c, const WeighPlan& p, int seqs) { return (size_t)seqs * c.kv_heads * p.row_blocks; }
size_t parts_of(const CacheView& c, const WeighPlan& p, int seqs) {
  return p.chunks > 1 ? (size_t)p.chunks * seqs * c.kv_heads * p.blocks * kBlockTokens : 0;
}

}  // namespace

int64_t weigh_workgroups(const CacheView& c, int heads, int seqs, int max_queries, int max_len, int last) {
  const WeighPlan p = weigh_plan(c, heads, seqs, max_queries, max_len, last);
  const int64_t weigh = (int64_t)p.blocks * p.chunks;
  return (int64_t)seqs * c.kv_heads * (weigh > p.row_blocks ? weigh : p.row_blocks);
}

size_t weigh_workspace_floats(const CacheView& c, int heads, int tokens, int seqs, int max_queries, int max_len,
                              int last) {
  const WeighPlan p = weigh_plan(c, heads, seqs, max_queries, max_len, last);
  return (size_t)tokens * heads * 2 + flags_of(c, p, seqs) + parts_of(c, p, seqs);
}

hipError_t launch_weigh(const CacheView& c, WeighArgs w, float* workspace, hipStream_t stream) {
  const AttnArgs& a = w.attn;
  const WeighPlan p = weigh_plan(c, a.heads, a.seqs, a.max_queries, a.max_len, w.last);
  if (p.blocks == 0 || p.row_blocks == 0) return hipSuccess;
  w.blocks = p.blocks;
  w.chunks = p.chunks;
  w.chunk_rows = p.chunk_rows;
  w.row_blocks = p.row_blocks;
  w.extreme = (int32_t*)(workspace + (size_t)a.tokens * a.heads * 2);
  w.parts = workspace + (size_t)a.tokens * a.heads * 2 + flags_of(c, p, a.seqs);
  const unsigned pairs = (unsigned)a.seqs * c.kv_heads;
  by_layout(c, [&](auto dim, auto int8) {
    constexpr int D = decltype(dim)::value;
    constexpr bool I8 = decltype(int8)::value;
    hipLaunchKernelGGL((recount_kernel<D, I8>), dim3(pairs * p.row_blocks), dim3(kThreads), 0, stream, c, w,
                       p.row_blocks);
    const dim3 grid(pairs * p.blocks * p.chunks);
    // (a lane's head then stays over the steps: 356 us instead of 368 for the prompt above)
    if (kStepRows % (a.heads / c.kv_heads) == 0)
      hipLaunchKernelGGL((weigh_kernel<D, I8, true>), grid, dim3(kThreads), 0, stream, c, w);
    else
      hipLaunchKernelGGL((weigh_kernel<D, I8, false>), grid, dim3(kThreads), 0, stream, c, w);
  });
  if (p.chunks > 1) hipLaunchKernelGGL(weigh_join_kernel, dim3(pairs * p.blocks), dim3(kThreads), 0, stream, c, w);
  return hipGetLastError();
}

}  // namespace nkt
