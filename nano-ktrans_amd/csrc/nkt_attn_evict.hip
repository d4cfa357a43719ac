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

// Per (sequence, head) in the workspace: the number of moves, the first position
// of the window and where it goes, then the moves' sources and destinations.
constexpr int kHead = 4;
__host__ __device__ __forceinline__ int64_t most_moves(int max_len) { return max_len / 2 + 1; }
__host__ __device__ __forceinline__ int64_t moves_row(int max_len) { return kHead + 2 * most_moves(max_len); }

// A weight as bits in its order: larger weights are larger numbers, the zeros are
// one number, a NaN is below all.
__device__ __forceinline__ uint32_t key_of(float w) {
  const uint32_t u = __float_as_uint(w + 0.0f);
  return w != w ? 0u : u >> 31 ? ~u : u | 0x80000000u;
}

// Exclusive prefix sum over the workgroup's threads; *total: of all.
__device__ __forceinline__ int block_scan(int v, int* s_sums, int* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int upto = wave_inclusive_scan(v);
  __syncthreads();  // (what was read of s_sums before)
  if (lane == 63) s_sums[wave] = upto;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    const int x = s_sums[i];
    before += i < wave ? x : 0;
    all += x;
  }
  *total = all;
  return before + upto - v;
}

// ---------------------------------------------------------------------------
// One workgroup per (sequence, head): the `front` largest of its C candidates by
// a radix selection on the keys (three histograms of 12, 10 and 10 bits), the
// moves in order of position, and the weights of what stays.  A wave holds a run of
// the positions, N keys per lane (N = 0: read again for each pass).
// ---------------------------------------------------------------------------
template <int N>
__global__ __launch_bounds__(kSelectThreads) void select_kernel(CacheView c, EvictArgs e) {
  __shared__ int s_bins[kBins];
  __shared__ int s_sums[kWaves];
  __shared__ int s_found[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int b = (int)(blockIdx.x / (unsigned)c.kv_heads), h = (int)(blockIdx.x % (unsigned)c.kv_heads);
  const float* w = e.weights + b * e.seq_stride + h * e.head_stride;
  float* out = e.out + b * e.out_seq_stride + h * e.out_head_stride;
  int32_t* head = e.moves + (int64_t)blockIdx.x * moves_row(e.max_len);
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
    if (tid == 0) head[0] = head[1] = head[2] = 0;
    const int stays = fits ? len : e.weights_width;
    for (int i = tid; i < e.weights_width; i += kSelectThreads) out[i] = i < stays ? w[i] : 0.f;
    return;
  }

  // (front < C) the wave's positions
  const int run = (C + kSelectThreads - 1) / kSelectThreads * 64;
  const int p0 = wave * run, p1 = p0 + run < C ? p0 + run : C;
  uint32_t keys[N > 0 ? N : 1];
  if (N > 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int p = p0 + i * 64 + lane;
      keys[i] = p < p1 ? key_of(w[p]) : 0u;
    }
  }
  // fn(position, key, the lane has one) over the wave's positions, 64 at a time
  auto each = [&](auto fn) __attribute__((always_inline)) {
    if constexpr (N > 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (p0 + i * 64 < p1) fn(p0 + i * 64 + lane, keys[i], p0 + i * 64 + lane < p1);
      }
    } else {
      for (int p = p0 + lane; p - lane < p1; p += 64) fn(p, p < p1 ? key_of(w[p]) : 0u, p < p1);
    }
  };

  // The threshold: keys above it stay, and `ties` of those that are equal.
  uint32_t threshold = 0xffffffffu;
  int ties = 0;
  if (front > 0) {
    uint32_t prefix = 0;
    int want = front;  // of the keys that share the prefix
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 20 : pass == 1 ? 10 : 0;
      const int bins = pass == 0 ? kBins : 1024;
      for (int i = tid; i < bins; i += kSelectThreads) s_bins[i] = 0;
      __syncthreads();
      each([&](int, uint32_t key, bool real) {
        const bool counts = real && (pass == 0 || (key >> (pass == 1 ? 20 : 10)) == prefix);
        const int digit = (int)(key >> shift) & (bins - 1);
        // (many weights of one number, as zeros are: one addition for all of them)
        const uint64_t all = __ballot(counts);
        if (all == 0) return;
        const int lead = __builtin_ctzll(all);
        const bool same = counts && digit == __builtin_amdgcn_readlane(digit, lead);
        const int sames = __popcll(__ballot(same));
        if (sames >= 8) {
          if (lane == lead) atomicAdd(&s_bins[digit], sames);
          if (counts && !same) atomicAdd(&s_bins[digit], 1);
        } else if (counts) {
          atomicAdd(&s_bins[digit], 1);
        }
      });
      __syncthreads();
      // thread t looks at bins from the top, 4 or 1 of them
      const int mine = bins / kSelectThreads;
      const int top = bins - 1 - tid * mine;
      int sum = 0;
      for (int i = 0; i < mine; ++i) sum += s_bins[top - i];
      int total;
      int above = block_scan(sum, s_sums, &total);
      if (above < want && above + sum >= want) {
        int i = 0;
        while (above + s_bins[top - i] < want) above += s_bins[top - i++];
        s_found[0] = top - i;
        s_found[1] = above;
      }
      __syncthreads();
      prefix = prefix << (pass == 0 ? 12 : 10) | (uint32_t)s_found[0];
      want -= s_found[1];
    }
    threshold = prefix;
    ties = want;
  }
  // Ranks in order of position: of equal keys, then of holes and of what fills them.
  int total;
  int equal = 0;
  each([&](int, uint32_t key, bool real) { equal += __popcll(__ballot(real && key == threshold)); });
  int tie = block_scan(lane == 0 ? equal : 0, s_sums, &total);
  tie = __builtin_amdgcn_readfirstlane(tie);
  const uint64_t below = (1ull << lane) - 1;
  auto stays = [&](uint32_t key, bool real, int& rank) {
    const bool is_tie = real && front > 0 && key == threshold;
    const uint64_t all = __ballot(is_tie);
    const bool yes = real && front > 0 && (key > threshold || (is_tie && rank + __popcll(all & below) < ties));
    rank += __popcll(all);
    return yes;
  };
  int holes = 0, fills = 0, rank = tie;
  each([&](int p, uint32_t key, bool real) {
    const bool yes = stays(key, real, rank);
    holes += __popcll(__ballot(real && !yes && p < front));
    fills += __popcll(__ballot(yes && p >= front));
  });
  int hole = block_scan(lane == 0 ? holes : 0, s_sums, &total);
  int fill = block_scan(lane == 0 ? fills : 0, s_sums, &total);
  hole = __builtin_amdgcn_readfirstlane(hole);
  fill = __builtin_amdgcn_readfirstlane(fill);
  rank = tie;
  each([&](int p, uint32_t key, bool real) {
    const bool yes = stays(key, real, rank);
    const bool is_hole = real && !yes && p < front, is_fill = yes && p >= front;
    const uint64_t hs = __ballot(is_hole), fs = __ballot(is_fill);
    if (is_hole) to[hole + __popcll(hs & below)] = p;
    if (is_fill) from[fill + __popcll(fs & below)] = p;
    hole += __popcll(hs);
    fill += __popcll(fs);
  });
  const int moves = total;
  if (tid == 0) {
    head[0] = moves;
    head[1] = C;
    head[2] = front;
  }
  // The weights: what stays where it is, what moves, the window, zeros.  (out may
  // be w: nothing is written before all that lies there has been read.)
  if (out != w)
    for (int i = tid; i < front; i += kSelectThreads) out[i] = w[i];
  __syncthreads();
  for (int i = tid; i < moves; i += kSelectThreads) out[to[i]] = w[from[i]];
  __syncthreads();
  for (int i0 = 0; i0 < window; i0 += kSelectThreads) {
    const float x = i0 + tid < window ? w[C + i0 + tid] : 0.f;
    __syncthreads();
    if (i0 + tid < window) out[front + i0 + tid] = x;
  }
  __syncthreads();
  for (int i = keep + tid; i < e.weights_width; i += kSelectThreads) out[i] = 0.f;
}

// ---------------------------------------------------------------------------
// A token's key, value and scales, 16 lanes each: a lane takes 1 / 16 of the
// key's bytes and every 16th dimension of the value.
// ---------------------------------------------------------------------------
template <int D, bool I8>
struct Token {
  static constexpr int U = I8 ? 16 : 8;
  static constexpr int kWords = D * (I8 ? 1 : 2) / (4 * kRowLanes);
  typedef uint32_t Words __attribute__((ext_vector_type(kWords)));
  Words k;
  uint32_t v[D / kRowLanes];
  float ks, vs;

  __device__ __forceinline__ void read(const CacheView& c, int64_t slot, int h, int l) {
    const int off = (int)slot & ((1 << c.page_shift) - 1);
    const int64_t blk = block_of(c, slot >> c.page_shift, h);
    k = *((const Words*)(c.k + (blk + off * D) * (I8 ? 1 : 2)) + l);
    const int64_t va = blk + (off & ~(U - 1)) * D + (off & (U - 1));
#pragma unroll
    for (int j = 0; j < D / kRowLanes; ++j) {
      const int64_t at = va + (l + kRowLanes * j) * U;
      v[j] = I8 ? c.v[at] : ((const uint16_t*)c.v)[at];
    }
    if (I8 && l == 0) {
      ks = c.k_scales[scale_of(c, slot, h)];
      vs = c.v_scales[scale_of(c, slot, h)];
    }
  }
  __device__ __forceinline__ void write(const CacheView& c, int64_t slot, int h, int l) const {
    const int off = (int)slot & ((1 << c.page_shift) - 1);
    const int64_t blk = block_of(c, slot >> c.page_shift, h);
    *((Words*)(c.k + (blk + off * D) * (I8 ? 1 : 2)) + l) = k;
    const int64_t va = blk + (off & ~(U - 1)) * D + (off & (U - 1));
#pragma unroll
    for (int j = 0; j < D / kRowLanes; ++j) {
      const int64_t at = va + (l + kRowLanes * j) * U;
      if (I8)
        c.v[at] = (uint8_t)v[j];
      else
        ((uint16_t*)c.v)[at] = (uint16_t)v[j];
    }
    if (I8 && l == 0) {
      c.k_scales[scale_of(c, slot, h)] = ks;
      c.v_scales[scale_of(c, slot, h)] = vs;
    }
  }
};

__device__ __forceinline__ int64_t slot_at(const CacheView& c, const EvictArgs& e, int b, int p) {
  const int64_t page = e.table[(int64_t)b * e.width + (p >> c.page_shift)];
  if (page < 0 || page >= c.num_pages) {
    report(c.status, kBadPage);
    return -1;
  }
  return (page << c.page_shift) | (p & ((1 << c.page_shift) - 1));
}

// Fills the places of evicted tokens: destinations lie before `front`, sources at
// or past it, so the moves are independent of each other.
template <int D, bool I8>
__global__ __launch_bounds__(kMoveThreads) void fill_kernel(CacheView c, EvictArgs e, int groups) {
  const int pair = (int)(blockIdx.x / (unsigned)groups), group = (int)(blockIdx.x % (unsigned)groups);
  const int b = (int)((unsigned)pair / (unsigned)c.kv_heads), h = (int)((unsigned)pair % (unsigned)c.kv_heads);
  const int32_t* head = e.moves + pair * moves_row(e.max_len);
  const int moves = head[0];
  const int32_t* from = head + kHead;
  const int32_t* to = from + most_moves(e.max_len);
  constexpr int kMoves = kMoveThreads / kRowLanes;
  const int l = (int)threadIdx.x % kRowLanes;
  for (int i = group * kMoves + (int)threadIdx.x / kRowLanes; i < moves; i += groups * kMoves) {
    const int64_t src = slot_at(c, e, b, from[i]), dst = slot_at(c, e, b, to[i]);
    if (src < 0 || dst < 0) continue;
    Token<D, I8> t;
    t.read(c, src, h, l);
    t.write(c, dst, h, l);
  }
}

// The window, behind the rest: it only moves towards the front, so a token still to
// be read lies past every one written before it.  Chunks of 64 tokens, each read
// whole before any of it is written.
template <int D, bool I8>
__global__ __launch_bounds__(1024) void window_kernel(CacheView c, EvictArgs e) {
  const int b = (int)(blockIdx.x / (unsigned)c.kv_heads), h = (int)(blockIdx.x % (unsigned)c.kv_heads);
  const int32_t* head = e.moves + (int64_t)blockIdx.x * moves_row(e.max_len);
  const int C = head[1], front = head[2];
  if (C == front) return;
  const int keep = e.lens_out[b];
  const int window = keep - front;
  const int l = (int)threadIdx.x % kRowLanes, g = (int)threadIdx.x / kRowLanes;
  for (int i0 = 0; i0 < window; i0 += 1024 / kRowLanes) {
    const int i = i0 + g;
    int64_t src = -1, dst = -1;
    if (i < window) {
      src = slot_at(c, e, b, C + i);
      dst = slot_at(c, e, b, front + i);
    }
    const bool moves = src >= 0 && dst >= 0;
    Token<D, I8> t;
    if (moves) t.read(c, src, h, l);
    __syncthreads();
    if (moves) t.write(c, dst, h, l);
  }
}

}  // namespace

size_t evict_workspace_bytes(const CacheView& c, int seqs, int max_len) {
  return (size_t)seqs * c.kv_heads * moves_row(max_len) * sizeof(int32_t);
}

hipError_t launch_evict(const CacheView& c, const EvictArgs& e, hipStream_t stream) {
  const unsigned pairs = (unsigned)e.seqs * c.kv_heads;
  auto select = [&](auto n) {
    hipLaunchKernelGGL((select_kernel<decltype(n)::value>), dim3(pairs), dim3(kSelectThreads), 0, stream, c, e);
  };
  if (e.max_len <= 4 * kSelectThreads)
    select(std::integral_constant<int, 4>{});
  else if (e.max_len <= 16 * kSelectThreads)
    select(std::integral_constant<int, 16>{});
  else
    select(std::integral_constant<int, 0>{});
  // about 2048 workgroups, each with 16 moves at a time
  int64_t groups = (most_moves(e.max_len) + 15) / 16;
  const int64_t share = (2048 + pairs - 1) / pairs;
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
