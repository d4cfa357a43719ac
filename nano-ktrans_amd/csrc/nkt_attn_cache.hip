// The paged key / value cache: head norms, rotation and the write in one
// launch, reading rows back, and moving accepted drafted tokens.
#include "nkt_attn_device.h"

namespace nkt {

namespace {

constexpr int kThreads = 256;
constexpr int kLanes = 64;

// Tokens per 16-byte piece of the value layout.
template <bool I8>
constexpr int kUnit = I8 ? 16 : 8;

// Maximum over groups of N lanes of |x| as ordered bits: a NaN is above
// every number, so it is not lost.
template <int N>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
#pragma unroll
  for (int off = N / 2; off >= 1; off >>= 1) {
    const uint32_t o = (uint32_t)__shfl_xor((int)v, off);
    v = o > v ? o : v;
  }
  return v;
}
template <int N>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int off = N / 2; off >= 1; off >>= 1) v += __shfl_xor(v, off);
  return v;
}

// The scale of a row with this maximum; NaN for a row with a NaN or an
// infinity, whose codes then do not matter.
__device__ __forceinline__ float scale_from_max(uint32_t max_bits) {
  const float s = __uint_as_float(max_bits) / 127.0f;
  return max_bits >= 0x7f800000u ? __builtin_nanf("") : s == 0.0f ? 1.0f : s;
}
// round-half-even(x / scale): the quotient by the scale's reciprocal and one
// correction step, |x| <= 127 scale.  Both are taken 2^64 times as large for a
// scale whose reciprocal could pass fp32's range.
struct Quantizer {
  float up, scale, inverse;
  __device__ __forceinline__ explicit Quantizer(float s)
      : up(s < 0x1p-64f ? 0x1p64f : 1.0f), scale(s * up), inverse(1.0f / scale) {}
  __device__ __forceinline__ uint32_t code(float x) const {
    x *= up;
    const float q = x * inverse;
    const float r = __builtin_rintf(__builtin_fmaf(__builtin_fmaf(-q, scale, x), inverse, q));
    return (uint32_t)(int)fminf(fmaxf(r, -127.0f), 127.0f) & 0xffu;
  }
};

__device__ __forceinline__ float lo_f32(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_f32(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// Pieces and single tokens of a window of up to 64 tokens: lane l holds token l's slot
// (-1: none).  Returns the tokens at which a run of U consecutive slots fills
// one 16-byte piece of the value layout (bit l); *single: the other stored ones.
template <int U>
__device__ __forceinline__ uint64_t whole_pieces(int64_t slot, int lane, uint64_t* single) {
  const int64_t before = ((int64_t)__shfl_up((int)(slot >> 32), 1) << 32) | (uint32_t)__shfl_up((int)slot, 1);
  const bool stored = slot >= 0;
  const uint64_t valid = __ballot(stored);
  const uint64_t follows = __ballot(lane > 0 && stored && slot == before + 1);
  constexpr uint64_t kRun = (1ull << (U - 1)) - 1;
  const uint64_t next = lane < 63 ? follows >> (lane + 1) : 0;
  const bool whole = stored && lane + U <= 64 && (slot & (U - 1)) == 0 && (next & kRun) == kRun;
  const uint64_t pieces = __ballot(whole);
  uint64_t covered = 0;
#pragma unroll
  for (int j = 0; j < U; ++j) covered |= pieces << j;
  *single = valid & ~covered;
  return pieces;
}

__device__ __forceinline__ int next_bit(uint64_t& bits) {
  const int i = __builtin_ctzll(bits);
  bits &= bits - 1;
  return i;
}

__device__ __forceinline__ int64_t uniform64(int64_t v) {
  return ((int64_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32) |
         (uint32_t)__builtin_amdgcn_readfirstlane((int)v);
}

// ---------------------------------------------------------------------------
// Write.  The first rope_blocks workgroups take the query and key rows: D / 8
// lanes per row, four values from each half of the head, so that a rotation's
// two values sit in one lane; HEADS rows of a token in turn, on one read of its
// cosines and sines.  The others take windows of W tokens of one head's
// values, which they turn in LDS so that runs of consecutive slots go out as
// whole 16-byte pieces of the value layout (one token alone is D stores of one
// value each, 16 bytes apart: what a decode step pays for the prompt's layout).
// Bound by HBM: 16384 tokens of 16 + 16 heads, D = 128, bf16 403 MB in 77 us, 5.2
// TB/s; one token of 16 sequences, 32 / 4 heads, int8: 4.5 us, a launch's latency.
// ---------------------------------------------------------------------------
template <int D, bool I8, int HEADS, int W>
__global__ __launch_bounds__(kThreads) void write_kernel(CacheView c, WriteArgs a, int rope_blocks) {
  constexpr int LR = D / 8;
  constexpr int kRows = kThreads / LR;
  const int tid = threadIdx.x;
  const int l = tid % LR, g = tid / LR;
  const int HK = c.kv_heads;
  __shared__ int64_t s_slot[kLanes];
  __shared__ __align__(16) uint8_t s_rows[W * D * (I8 ? 1 : 2)];

  if ((int)blockIdx.x < rope_blocks) {
    const int H = a.heads + HK;
    const int sets = (H + HEADS - 1) / HEADS;
    const int set = (int)blockIdx.x * kRows + g;
    if (set >= a.tokens * sets) return;  // (whole groups of D / 8 lanes)
    const int t = set / sets;
    const int h0 = (set - t * sets) * HEADS;
    u32x2 w1[HEADS], w2[HEADS];
#pragma unroll
    for (int j = 0; j < HEADS; ++j) {
      const int h = h0 + j < H ? h0 + j : H - 1;
      const uint16_t* src = h >= a.heads ? a.k + t * a.k_stride + (h - a.heads) * D : a.q + t * a.q_stride + h * D;
      w1[j] = *(const u32x2*)(src + 4 * l);
      w2[j] = *(const u32x2*)(src + D / 2 + 4 * l);
    }
    const int64_t pos = a.positions[t];
    const int64_t given = a.slots[t];
    const bool pos_ok = pos >= 0 && pos < a.rope_rows;
    if (!pos_ok && given >= 0 && l == 0) report(c.status, kBadPosition);  // (padding may have any)
    const float* rp = a.rope + (pos_ok ? pos : 0) * D;
    const f32x4 cs = *(const f32x4*)(rp + 4 * l);
    const f32x4 sn = *(const f32x4*)(rp + D / 2 + 4 * l);
#pragma unroll
    for (int j = 0; j < HEADS; ++j) {
      const int h = h0 + j;
      if (h >= H) return;
      const bool is_k = h >= a.heads;
      float x1[4] = {lo_f32(w1[j][0]), hi_f32(w1[j][0]), lo_f32(w1[j][1]), hi_f32(w1[j][1])};
      float x2[4] = {lo_f32(w2[j][0]), hi_f32(w2[j][0]), lo_f32(w2[j][1]), hi_f32(w2[j][1])};
      const uint16_t* nw = is_k ? a.k_norm : a.q_norm;
      if (nw) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) ss += x1[i] * x1[i] + x2[i] * x2[i];
        ss = group_sum<LR>(ss);
        const float inv = __builtin_amdgcn_rsqf(ss * (1.0f / D) + a.eps);
        const u32x2 n1 = *(const u32x2*)(nw + 4 * l);
        const u32x2 n2 = *(const u32x2*)(nw + D / 2 + 4 * l);
        const float m1[4] = {lo_f32(n1[0]), hi_f32(n1[0]), lo_f32(n1[1]), hi_f32(n1[1])};
        const float m2[4] = {lo_f32(n2[0]), hi_f32(n2[0]), lo_f32(n2[1]), hi_f32(n2[1])};
#pragma unroll
        for (int i = 0; i < 4; ++i) x1[i] *= inv * m1[i], x2[i] *= inv * m2[i];
      }
      float y1[4], y2[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        y1[i] = pos_ok ? x1[i] * cs[i] - x2[i] * sn[i] : 0.f;
        y2[i] = pos_ok ? x2[i] * cs[i] + x1[i] * sn[i] : 0.f;
      }
      const u32x2 b1 = {pack_pair(y1[0], y1[1]), pack_pair(y1[2], y1[3])};
      const u32x2 b2 = {pack_pair(y2[0], y2[1]), pack_pair(y2[2], y2[3])};
      if (!is_k) {
        uint16_t* dst = a.q_out + ((int64_t)t * a.heads + h) * D;
        *(u32x2*)(dst + 4 * l) = b1;
        *(u32x2*)(dst + D / 2 + 4 * l) = b2;
        continue;
      }
      const int64_t slot = pos_ok ? checked_slot(c, given) : -1;
      if (slot < 0) return;  // (nothing but keys follows)
      const int off = (int)slot & ((1 << c.page_shift) - 1);
      const int64_t at = block_of(c, slot >> c.page_shift, h - a.heads) + off * D;
      if (!I8) {
        uint16_t* dst = (uint16_t*)c.k + at;
        *(u32x2*)(dst + 4 * l) = b1;
        *(u32x2*)(dst + D / 2 + 4 * l) = b2;
      } else {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t a1 = __float_as_uint(y1[i]) & 0x7fffffffu, a2 = __float_as_uint(y2[i]) & 0x7fffffffu;
          top = a1 > top ? a1 : top;
          top = a2 > top ? a2 : top;
        }
        const float s = scale_from_max(group_max<LR>(top));
        const Quantizer q(s);
        uint32_t p1 = 0, p2 = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) p1 |= q.code(y1[i]) << (8 * i), p2 |= q.code(y2[i]) << (8 * i);
        *(uint32_t*)(c.k + at + 4 * l) = p1;
        *(uint32_t*)(c.k + at + D / 2 + 4 * l) = p2;
        if (l == 0) c.k_scales[scale_of(c, slot, h - a.heads)] = s;
      }
    }
    return;
  }

  const int item = (int)blockIdx.x - rope_blocks;
  const int h = item % HK;
  const int t0 = item / HK * W;
  if (tid < kLanes) {
    int64_t slot = -1;
    if (tid < W && t0 + tid < a.tokens) {
      const int64_t pos = a.positions[t0 + tid];
      if (pos >= 0 && pos < a.rope_rows) slot = checked_slot(c, a.slots[t0 + tid]);
    }
    s_slot[tid] = slot;
  }
  __syncthreads();
  constexpr int kMine = (W + kRows - 1) / kRows;  // rows per thread
  u32x2 w1[kMine], w2[kMine];
#pragma unroll
  for (int j = 0; j < kMine; ++j) {
    if (t0 + j * kRows >= a.tokens) break;
    const int t = t0 + j * kRows + g;
    const uint16_t* src = a.v + (t < a.tokens ? t : a.tokens - 1) * a.v_stride + h * D + 8 * l;
    w1[j] = *(const u32x2*)src;
    w2[j] = *(const u32x2*)(src + 4);
  }
#pragma unroll
  for (int j = 0; j < kMine; ++j) {
    if (t0 + j * kRows >= a.tokens) break;
    const int r = j * kRows + g;
    if (r >= W) break;  // (whole groups of D / 8 lanes)
    if (!I8) {
      *(u32x4*)(s_rows + (r * D + 8 * l) * 2) = u32x4{w1[j][0], w1[j][1], w2[j][0], w2[j][1]};
    } else {
      const float x[8] = {lo_f32(w1[j][0]), hi_f32(w1[j][0]), lo_f32(w1[j][1]), hi_f32(w1[j][1]),
                          lo_f32(w2[j][0]), hi_f32(w2[j][0]), lo_f32(w2[j][1]), hi_f32(w2[j][1])};
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t b = __float_as_uint(x[i]) & 0x7fffffffu;
        top = b > top ? b : top;
      }
      const float s = scale_from_max(group_max<LR>(top));
      const Quantizer q(s);
      uint32_t p[2] = {0, 0};
#pragma unroll
      for (int i = 0; i < 8; ++i) p[i >> 2] |= q.code(x[i]) << (8 * (i & 3));
      *(u32x2*)(s_rows + r * D + 8 * l) = u32x2{p[0], p[1]};
      const int64_t slot = s_slot[r];
      if (l == 0 && slot >= 0) c.v_scales[scale_of(c, slot, h)] = s;
    }
  }
  __syncthreads();
  constexpr int U = kUnit<I8>;
  const int lane = tid & 63, wave = tid >> 6;
  uint64_t single;
  uint64_t pieces = whole_pieces<U>(s_slot[lane], lane, &single);
  const int mask = (1 << c.page_shift) - 1;
  for (int n = 0; pieces; ++n) {
    const int t = next_bit(pieces);
    if ((n & 3) != wave) continue;
    const int64_t slot = uniform64(s_slot[t]);
    uint8_t* dst = c.v + (block_of(c, slot >> c.page_shift, h) + ((int)slot & mask) * D) * (I8 ? 1 : 2);
    for (int d = lane; d < D; d += 64) {
      u32x4 w;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (!I8) {
          const uint16_t* s = (const uint16_t*)s_rows + (t + 2 * i) * D + d;
          w[i] = s[0] | (uint32_t)s[D] << 16;
        } else {
          const uint8_t* s = s_rows + (t + 4 * i) * D + d;
          w[i] = s[0] | (uint32_t)s[D] << 8 | (uint32_t)s[2 * D] << 16 | (uint32_t)s[3 * D] << 24;
        }
      }
      *(u32x4*)(dst + d * 16) = w;
    }
  }
  for (int n = 0; single; ++n) {
    const int t = next_bit(single);
    if ((n & 3) != wave) continue;
    const int64_t slot = uniform64(s_slot[t]);
    const int off = (int)slot & mask;
    const int64_t at = block_of(c, slot >> c.page_shift, h) + (off & ~(U - 1)) * D + (off & (U - 1));
    for (int d = lane; d < D; d += 64) {
      if (!I8)
        ((uint16_t*)c.v)[at + d * U] = ((const uint16_t*)s_rows)[t * D + d];
      else
        c.v[at + d * U] = s_rows[t * D + d];
    }
  }
}

// ---------------------------------------------------------------------------
// Read: one workgroup per window of W slots of one head.  Keys are rows;
// values come out of their layout through LDS, whole pieces for runs of
// consecutive slots.  Bound by HBM: 8 sequences of up to 8100 tokens, 8 heads, D =
// 128, bf16 372 MB in 77 us, 4.8 TB/s; 777 tokens of 4 heads 3.6 us.
// ---------------------------------------------------------------------------
template <int D, bool I8, int W>
__global__ __launch_bounds__(kThreads) void read_kernel(CacheView c, const int64_t* __restrict__ slots, int n,
                                                        uint16_t* __restrict__ k_out, uint16_t* __restrict__ v_out) {
  constexpr int LR = D / 8;
  constexpr int kRows = kThreads / LR;
  constexpr int U = kUnit<I8>;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int l = tid % LR, g = tid / LR;
  const int HK = c.kv_heads;
  const int h = (int)(blockIdx.x % (unsigned)HK);
  const int t0 = (int)(blockIdx.x / (unsigned)HK) * W;
  const int mask = (1 << c.page_shift) - 1;
  __shared__ int64_t s_slot[kLanes];
  __shared__ __align__(16) uint8_t s_rows[W * D * (I8 ? 1 : 2)];
  if (tid < kLanes) s_slot[tid] = tid < W && t0 + tid < n ? checked_slot(c, slots[t0 + tid]) : -1;
  __syncthreads();
  // this thread's keys (and scales), asked for before the values are turned
  constexpr int kMine = (W + kRows - 1) / kRows;
  typedef uint32_t KeyWords __attribute__((ext_vector_type(I8 ? 2 : 4)));
  KeyWords keys[kMine];
  float ks[kMine], vs[kMine];
#pragma unroll
  for (int j = 0; j < kMine; ++j) {
    if (t0 + j * kRows >= n) break;
    const int64_t slot = s_slot[j * kRows + g] < 0 ? 0 : s_slot[j * kRows + g];
    const int64_t at = block_of(c, slot >> c.page_shift, h) + ((int)slot & mask) * D + 8 * l;
    keys[j] = *(const KeyWords*)(c.k + at * (I8 ? 1 : 2));
    if (I8) {
      ks[j] = c.k_scales[scale_of(c, slot, h)];
      vs[j] = c.v_scales[scale_of(c, slot, h)];
    }
  }
  uint64_t single;
  uint64_t pieces = whole_pieces<U>(s_slot[lane], lane, &single);
  for (int i = 0; pieces; ++i) {
    const int t = next_bit(pieces);
    if ((i & 3) != wave) continue;
    const int64_t slot = uniform64(s_slot[t]);
    const uint8_t* src = c.v + (block_of(c, slot >> c.page_shift, h) + ((int)slot & mask) * D) * (I8 ? 1 : 2);
    for (int d = lane; d < D; d += 64) {
      const u32x4 w = *(const u32x4*)(src + d * 16);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (!I8) {
          uint16_t* s = (uint16_t*)s_rows + (t + 2 * j) * D + d;
          s[0] = (uint16_t)w[j];
          s[D] = (uint16_t)(w[j] >> 16);
        } else {
          uint8_t* s = s_rows + (t + 4 * j) * D + d;
          s[0] = (uint8_t)w[j];
          s[D] = (uint8_t)(w[j] >> 8);
          s[2 * D] = (uint8_t)(w[j] >> 16);
          s[3 * D] = (uint8_t)(w[j] >> 24);
        }
      }
    }
  }
  // single tokens: every fourth token is this wave's, four of them at a time
  for (uint64_t mine = single & (0x1111111111111111ull << wave); mine;) {
    int t[4];
    uint32_t x[4][D / 64];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      t[i] = mine ? next_bit(mine) : -1;
      const int64_t slot = uniform64(s_slot[t[i] < 0 ? t[0] : t[i]]);
      const int off = (int)slot & mask;
      const int64_t at = block_of(c, slot >> c.page_shift, h) + (off & ~(U - 1)) * D + (off & (U - 1));
#pragma unroll
      for (int j = 0; j < D / 64; ++j) {
        const int64_t e = at + (lane + 64 * j) * U;
        x[i][j] = I8 ? c.v[e] : ((const uint16_t*)c.v)[e];
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < D / 64; ++j) {
        if (t[i] < 0) continue;
        const int e = t[i] * D + lane + 64 * j;
        if (I8)
          s_rows[e] = (uint8_t)x[i][j];
        else
          ((uint16_t*)s_rows)[e] = (uint16_t)x[i][j];
      }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kMine; ++j) {
    const int r = j * kRows + g;
    if (r >= W || t0 + r >= n) return;
    u32x4 kw = {0, 0, 0, 0}, vw = {0, 0, 0, 0};
    if (s_slot[r] >= 0) {
      if constexpr (!I8) {
        kw = keys[j];
        vw = *(const u32x4*)(s_rows + (r * D + 8 * l) * 2);
      } else {
        const u32x2 vc = *(const u32x2*)(s_rows + r * D + 8 * l);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int sh = 16 * (i & 1);
          const uint32_t kc = keys[j][i >> 1] >> sh, v2 = vc[i >> 1] >> sh;
          kw[i] = pack_pair((float)(int8_t)kc * ks[j], (float)(int8_t)(kc >> 8) * ks[j]);
          vw[i] = pack_pair((float)(int8_t)v2 * vs[j], (float)(int8_t)(v2 >> 8) * vs[j]);
        }
      }
    }
    const int64_t to = ((int64_t)(t0 + r) * HK + h) * D + 8 * l;
    *(u32x4*)(k_out + to) = kw;
    *(u32x4*)(v_out + to) = vw;
  }
}

// ---------------------------------------------------------------------------
// Keep: one workgroup per (sequence, head).  A token only ever moves towards
// the context (kept[i] >= i), so a row still to be read (kept[j] >= j) lies
// past every row written for an earlier i < j: rows are taken in chunks, each
// read whole before any of it is written.  Latency: 2.7 us for one draft of 12,
// 5 for 64 drafts of up to 64 tokens, 8 heads, int8.
// ---------------------------------------------------------------------------
constexpr int kKeepChunk = 16;

template <int D, bool I8>
__global__ __launch_bounds__(kThreads) void keep_kernel(CacheView c, const int32_t* __restrict__ table, int width,
                                                        const int32_t* __restrict__ context,
                                                        const int32_t* __restrict__ kept, int kept_width,
                                                        const int32_t* __restrict__ counts) {
  constexpr int U = kUnit<I8>;
  constexpr int LR = 16;  // lanes per row
  const int b = (int)(blockIdx.x / (unsigned)c.kv_heads), h = (int)(blockIdx.x % (unsigned)c.kv_heads);
  const int l = threadIdx.x % LR, g = threadIdx.x / LR;  // 16 rows of a chunk
  const int mask = (1 << c.page_shift) - 1;
  const int64_t most = (int64_t)width << c.page_shift;
  const int64_t base = context[b];
  int count = counts[b];
  if (count > kept_width || (base < 0 && count > 0)) {  // (a sequence that keeps nothing may be padding)
    if (threadIdx.x == 0) report(c.status, kBadKept);
    count = base < 0 ? 0 : kept_width;
  }
  auto slot_of = [&](int64_t pos) -> int64_t {
    const int64_t page = table[(int64_t)b * width + (pos >> c.page_shift)];
    if (page < 0 || page >= c.num_pages) {
      report(c.status, kBadPage);
      return -1;
    }
    return (page << c.page_shift) | (pos & mask);
  };
  for (int i0 = 0; i0 < count; i0 += kKeepChunk) {
    const int i = i0 + g;
    int64_t from = -1, to = -1;
    if (i < count) {
      const int64_t src = kept[(int64_t)b * kept_width + i];
      if (src < i || base + src >= most) {
        if (l == 0) report(c.status, kBadKept);
      } else if (src != i) {
        from = slot_of(base + src);
        to = slot_of(base + i);
      }
    }
    const bool moves = from >= 0 && to >= 0;
    uint16_t kr[D / LR], vr[D / LR];
    float ks = 0.f, vs = 0.f;
    if (moves) {
      const int off = (int)from & mask;
      const int64_t blk = block_of(c, from >> c.page_shift, h);
      const int64_t va = blk + (off & ~(U - 1)) * D + (off & (U - 1));
#pragma unroll
      for (int j = 0; j < D / LR; ++j) {
        const int d = l + LR * j;
        kr[j] = I8 ? c.k[blk + off * D + d] : ((const uint16_t*)c.k)[blk + off * D + d];
        vr[j] = I8 ? c.v[va + d * U] : ((const uint16_t*)c.v)[va + d * U];
      }
      if (I8 && l == 0) {
        ks = c.k_scales[scale_of(c, from, h)];
        vs = c.v_scales[scale_of(c, from, h)];
      }
    }
    __syncthreads();
    if (moves) {
      const int off = (int)to & mask;
      const int64_t blk = block_of(c, to >> c.page_shift, h);
      const int64_t va = blk + (off & ~(U - 1)) * D + (off & (U - 1));
#pragma unroll
      for (int j = 0; j < D / LR; ++j) {
        const int d = l + LR * j;
        if (I8) {
          c.k[blk + off * D + d] = (uint8_t)kr[j];
          c.v[va + d * U] = (uint8_t)vr[j];
        } else {
          ((uint16_t*)c.k)[blk + off * D + d] = kr[j];
          ((uint16_t*)c.v)[va + d * U] = vr[j];
        }
      }
      if (I8 && l == 0) {
        c.k_scales[scale_of(c, to, h)] = ks;
        c.v_scales[scale_of(c, to, h)] = vs;
      }
    }
  }
}

// Windows of 64 tokens (and four heads at a time), or of 16 (and one) for a few,
// which would leave most CUs idle.  In us, 16 and 64: write, 16 + 16 heads, bf16,
// 256 tokens 4.1 and 4.4, 1024 8.5 and 7.7, 2048 12.9 and 11.6, 8192 48 and 38;
// 32 + 4, int8, 1024 9.5 and 10.7, 2048 13.4 and 14.3, 4096 22.2 and 22.2, 8192 46
// and 38.  read, 16 heads, 512 4.8 and 5.3, 1024 6.5 and 6.5, 4096 16.4 and 13.4; 4
// heads, 1024 3.7 and 5.1, 2048 4.8 and 5.5, 4096 6.9 and 6.7.
int window_of(int tokens) { return tokens > 1024 ? 64 : 16; }

}  // namespace

hipError_t launch_cache_write(const CacheView& c, const WriteArgs& a, hipStream_t stream) {
  by_layout(c, [&](auto dim, auto int8) {
    constexpr int D = decltype(dim)::value;
    constexpr bool I8 = decltype(int8)::value;
    auto launch = [&](auto heads, auto window) {
      constexpr int HEADS = decltype(heads)::value, W = decltype(window)::value;
      constexpr int kRows = kThreads / (D / 8);
      const int value_blocks = (a.tokens + W - 1) / W * c.kv_heads;
      const int sets = (a.heads + c.kv_heads + HEADS - 1) / HEADS;
      const int rope_blocks = (a.tokens * sets + kRows - 1) / kRows;
      hipLaunchKernelGGL((write_kernel<D, I8, HEADS, W>), dim3(rope_blocks + value_blocks), dim3(kThreads), 0, stream,
                         c, a, rope_blocks);
    };
    // Four heads per group where there are enough rows for it (16384 tokens,
    // 16 + 16 heads: 77 us bf16, 69 int8; one head per group 85 and 89).
    if (window_of(a.tokens) == 64)
      launch(std::integral_constant<int, 4>{}, std::integral_constant<int, 64>{});
    else
      launch(std::integral_constant<int, 1>{}, std::integral_constant<int, 16>{});
  });
  return hipGetLastError();
}

hipError_t launch_cache_read(const CacheView& c, const int64_t* slots, int n, uint16_t* k_out, uint16_t* v_out,
                             hipStream_t stream) {
  by_layout(c, [&](auto dim, auto int8) {
    constexpr int D = decltype(dim)::value;
    constexpr bool I8 = decltype(int8)::value;
    auto launch = [&](auto window) {
      constexpr int W = decltype(window)::value;
      hipLaunchKernelGGL((read_kernel<D, I8, W>), dim3((n + W - 1) / W * c.kv_heads), dim3(kThreads), 0, stream, c, slots,
                         n, k_out, v_out);
    };
    if (window_of(n) == 64)
      launch(std::integral_constant<int, 64>{});
    else
      launch(std::integral_constant<int, 16>{});
  });
  return hipGetLastError();
}

hipError_t launch_cache_keep(const CacheView& c, const int32_t* table, int width, const int32_t* context,
                             const int32_t* kept, int kept_width, const int32_t* counts, int seqs,
                             hipStream_t stream) {
  by_layout(c, [&](auto dim, auto int8) {
    hipLaunchKernelGGL((keep_kernel<decltype(dim)::value, decltype(int8)::value>), dim3(seqs * c.kv_heads),
                       dim3(kThreads), 0, stream, c, table, width, context, kept, kept_width, counts);
  });
  return hipGetLastError();
}

}  // namespace nkt
