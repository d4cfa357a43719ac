// Low-rank adapters of many requests beside a shared projection.
#include <type_traits>

#include "nkt_common.h"
#include "nkt_lora_internal.h"

namespace nkt {

namespace {

constexpr int kTile = 32;  // tokens of a workgroup: the columns of a 32x32x16 product

typedef float f32x16 __attribute__((ext_vector_type(16)));

// 32x32x16 bf16: lane l supplies A[l%32][8*(l/32) .. +7] and B[8*(l/32) ..
// +7][l%32]; D[(v&3) + 8*(v>>2) + 4*(l/32)][l%32] lands in register v.  With the
// rows of A in the order of the buffers' layout, register v is row 16 (l/32) + v.
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

constexpr int kNone = -1, kPast = -2;

// The adapter of the tile's token in this lane (lanes l and l + 32 have the same
// one): kNone without one, kPast behind the last token.
__device__ __forceinline__ int adapter_of(const LoraView& v, const LoraArgs& a, int tile, int col, bool reports) {
  const int t = tile * kTile + col;
  if (t >= a.tokens) return kPast;
  const int64_t i = a.index[t];
  if (i >= v.adapters) {
    if (reports && v.status) __hip_atomic_fetch_or(v.status, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
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

// ---------------------------------------------------------------------------
// low = scale x A^T: one workgroup per tile of 32 tokens and slot (the tile's
// slot-th, slot + slots-th, ... distinct adapter), MB blocks of 32 rows of A.  The
// waves share the input's features, 64 at a time, and add up in LDS in order.
// ---------------------------------------------------------------------------
template <int MB, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void shrink_kernel(LoraView v, LoraArgs a, int slots) {
  __shared__ float s_sum[WAVES][64][17];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int half = lane >> 5, col = lane & 31;
  const int slot0 = (int)(blockIdx.x % (unsigned)slots);
  const int tile = (int)(blockIdx.x / (unsigned)slots);
  const int m0 = (int)blockIdx.y * MB;
  const int mine = adapter_of(v, a, tile, col, tid < 32 && slot0 == 0 && m0 == 0);
  const int t = tile * kTile + col < a.tokens ? tile * kTile + col : a.tokens - 1;
  const uint16_t* x = a.x + t * a.x_stride + half * 32;
  const int groups = v.in / 64;
  const int64_t block = (int64_t)v.in * 32;  // values of a block of A
  for (int slot = slot0;; slot += slots) {
    const int adapter = distinct(mine, slot, false);
    if (adapter < 0) return;
    const uint16_t* w = v.a + ((int64_t)adapter * v.row_blocks + m0) * block + lane * 8;
    f32x16 acc[MB];
#pragma unroll
    for (int m = 0; m < MB; ++m) acc[m] = zeros();
    for (int k = wave; k < groups; k += WAVES) {
      u32x4 xf[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) xf[j] = *(const u32x4*)(x + k * 64 + j * 8);
#pragma unroll
      for (int m = 0; m < MB; ++m) {
        if (m0 + m < v.row_blocks) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            acc[m] = mfma32(*(const u32x4*)(w + m * block + (k * 4 + j) * 512), xf[j], acc[m]);
        }
      }
    }
#pragma unroll
    for (int m = 0; m < MB; ++m) {
      if (m0 + m >= v.row_blocks) break;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 16; ++i) s_sum[wave][lane][i] = acc[m][i];
      __syncthreads();
#pragma unroll
      for (int e0 = 0; e0 < 1024; e0 += WAVES * 64) {
        const int e = e0 + tid, i = e & 15, l = e >> 4;
        float sum = 0.f;
#pragma unroll
        for (int u = 0; u < WAVES; ++u) sum += s_sum[u][l][i];
        const int row = (m0 + m) * 32 + (l >> 5) * 16 + i;
        const int part = row / v.rank;
        const int token = tile * kTile + (l & 31);
        if (__builtin_amdgcn_ds_bpermute((l & 31) * 4, mine) != adapter || part >= v.parts) continue;
        // (a rank that the adapter does not have is zero whatever x holds)
        const int at = adapter * v.parts + part;
        a.low[(int64_t)token * (v.row_blocks * 32) + row] = row - part * v.rank < v.ranks[at] ? sum * v.scales[at] : 0.f;
      }
    }
  }
}

// Eight fp32 values as two bf16 operands whose sum they are to 2^-16 of them: the
// upper 16 bits, and the rest rounded.  (An infinity has no rest.)
__device__ __forceinline__ void split_operand(const float* src, u32x4* high, u32x4* rest) {
  const f32x4 a = *(const f32x4*)src, b = *(const f32x4*)(src + 4);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t h[2];
    float r[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float x = i < 2 ? a[2 * i + j] : b[2 * i + j - 4];
      const uint32_t u = __float_as_uint(x);
      h[j] = x != x ? 0x7fc00000u : u & 0xffff0000u;
      r[j] = (u & 0x7f800000u) == 0x7f800000u ? 0.f : x - __uint_as_float(h[j]);
    }
    (*high)[i] = h[0] >> 16 | h[1];
    (*rest)[i] = pair_of(r[0], r[1]);
  }
}

// ---------------------------------------------------------------------------
// out = base + low B^T: one workgroup per tile of 32 tokens, slot and run of
// column blocks; a wave computes 32 tokens x 32 columns at a time.  low enters
// as two bf16 operands, so that its rounding stays far below the result's.
// KS = R / 16.
// ---------------------------------------------------------------------------
template <int KS>
__global__ __launch_bounds__(256) void expand_kernel(LoraView v, LoraArgs a, int slots, int per_wave) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int half = lane >> 5, col = lane & 31;
  const int slot0 = (int)(blockIdx.x % (unsigned)slots);
  const int tile = (int)(blockIdx.x / (unsigned)slots);
  const int blocks = v.columns / 32;
  const int first = (int)blockIdx.y * per_wave * 4;
  const int mine = adapter_of(v, a, tile, col, false);
  const int t = tile * kTile + col < a.tokens ? tile * kTile + col : a.tokens - 1;
  const uint16_t* base = a.base + t * a.base_stride + half * 16;
  uint16_t* out = a.out + t * a.out_stride + half * 16;
  const bool same = a.base == a.out;
  for (int slot = slot0;; slot += slots) {
    const int adapter = distinct(mine, slot, !same);
    if (adapter == kPast) return;
    int loaded = -1;
    u32x4 high[KS], rest[KS];
    for (int i = 0; i < per_wave; ++i) {
      const int c = first + i * 4 + wave;
      if (c >= blocks) break;
      const u32x4 b0 = *(const u32x4*)(base + c * 32), b1 = *(const u32x4*)(base + c * 32 + 8);
      u32x4 y[2] = {b0, b1};
      if (adapter >= 0) {
        int part = 0;
        while (c >= v.part_end[part]) ++part;
        if (part != loaded) {
          const float* low = a.low + (int64_t)t * (v.row_blocks * 32) + part * v.rank + half * 8;
#pragma unroll
          for (int s = 0; s < KS; ++s) split_operand(low + s * 16, &high[s], &rest[s]);
          loaded = part;
        }
        const uint16_t* w = v.b + (((int64_t)adapter * blocks + c) * KS * 64 + lane) * 8;
        f32x16 acc = zeros();
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          const u32x4 wf = *(const u32x4*)(w + s * 512);
          acc = mfma32(wf, rest[s], acc);
          acc = mfma32(wf, high[s], acc);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t z = y[j >> 2][j & 3];
          y[j >> 2][j & 3] = pair_of(__uint_as_float(z << 16) + acc[2 * j], __uint_as_float(z & 0xffff0000u) + acc[2 * j + 1]);
        }
      }
      if (mine == adapter) {
        *(u32x4*)(out + c * 32) = y[0];
        *(u32x4*)(out + c * 32 + 8) = y[1];
      }
    }
  }
}

}  // namespace

hipError_t launch_lora(const LoraView& v, const LoraArgs& a, hipStream_t stream) {
  const unsigned tiles = (unsigned)(a.tokens + kTile - 1) / kTile;
  // distinct adapters side by side while there are few tiles, in turn for many
  const int most = v.adapters < kTile ? v.adapters : kTile;
  int slots = tiles <= 16 ? (a.tokens < most ? a.tokens : most) : 1;
  if (slots < 1) slots = 1;
  auto shrink = [&](auto mb, auto waves) {
    constexpr int MB = decltype(mb)::value, WAVES = decltype(waves)::value;
    hipLaunchKernelGGL((shrink_kernel<MB, WAVES>), dim3(tiles * slots, (v.row_blocks + MB - 1) / MB), dim3(WAVES * 64),
                       0, stream, v, a, slots);
  };
  auto by_blocks = [&](auto waves) {
    if (v.row_blocks == 1)
      shrink(std::integral_constant<int, 1>{}, waves);
    else if (v.row_blocks == 2)
      shrink(std::integral_constant<int, 2>{}, waves);
    else
      shrink(std::integral_constant<int, 3>{}, waves);
  };
  if (tiles <= 16)
    by_blocks(std::integral_constant<int, 16>{});
  else
    by_blocks(std::integral_constant<int, 4>{});
  const int blocks = v.columns / 32;
  const int per_wave = tiles <= 16 ? 1 : 4;
  const int more = slots + (a.base != a.out && slots > 1 ? 1 : 0);
  const dim3 grid(tiles * more, (blocks + 4 * per_wave - 1) / (4 * per_wave));
  auto expand = [&](auto ks) {
    hipLaunchKernelGGL((expand_kernel<decltype(ks)::value>), grid, dim3(256), 0, stream, v, a, more, per_wave);
  };
  if (v.rank == 16)
    expand(std::integral_constant<int, 1>{});
  else if (v.rank == 32)
    expand(std::integral_constant<int, 2>{});
  else if (v.rank == 64)
    expand(std::integral_constant<int, 4>{});
  else
    expand(std::integral_constant<int, 8>{});
  return hipGetLastError();
}

}  // namespace nkt
