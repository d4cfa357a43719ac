// Device helpers of the attention kernels: the paged cache's addresses and
// the status word.
#pragma once

#include <type_traits>

#include "nkt_attn_internal.h"
#include "nkt_common.h"

namespace nkt {

__device__ __forceinline__ void report(uint32_t* status, uint32_t bit) {
  if (status) __hip_atomic_fetch_or(status, bit, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

constexpr uint32_t kBadSlot = 1, kBadPosition = 2, kBadPage = 4, kBadLength = 8, kBadKept = 16;

// A slot as the kernels use it: the slot, or -1 where nothing is stored.
__device__ __forceinline__ int64_t checked_slot(const CacheView& c, int64_t slot) {
  if (slot < 0) return -1;
  if ((slot >> c.page_shift) >= c.num_pages) {
    report(c.status, kBadSlot);
    return -1;
  }
  return slot;
}

// First value of (page, head) block, in values from the start of the cache.
__device__ __forceinline__ int64_t block_of(const CacheView& c, int64_t page, int head) {
  return ((page * c.kv_heads + head) << c.page_shift) * c.dim;
}
__device__ __forceinline__ int64_t scale_of(const CacheView& c, int64_t slot, int head) {
  const int64_t page = slot >> c.page_shift;
  const int off = (int)slot & ((1 << c.page_shift) - 1);
  return ((page * c.kv_heads + head) << c.page_shift) + off;
}

// Two floats -> packed bf16 pair (lo = first), round to nearest even.
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
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

// int8 codes of one 32-bit word -> two words of bf16 (exact)
__device__ __forceinline__ void bf16_of_codes(uint32_t w, uint32_t* lo, uint32_t* hi) {
  const float f0 = (float)(int8_t)w, f1 = (float)(int8_t)(w >> 8), f2 = (float)(int8_t)(w >> 16),
              f3 = (float)(int8_t)(w >> 24);
  *lo = __builtin_amdgcn_perm(__float_as_uint(f1), __float_as_uint(f0), 0x07060302u);
  *hi = __builtin_amdgcn_perm(__float_as_uint(f3), __float_as_uint(f2), 0x07060302u);
}

constexpr float kLog2e = 1.4426950408889634f;

// A product that is rounded before the maximum is taken off it.  Contracted with
// the subtraction it would keep bits that the maximum has lost: from 2^31 on, a
// score less the maximum that it is itself could reach 2^7, its weight infinity.
__device__ __forceinline__ float rounded_product(float a, float b) {
#pragma clang fp contract(off)
  return a * b;
}

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

// What the sequence is made from, asked for together (b is the same in all
// lanes): one round trip, and the caller's own loads may go beside it.
struct SeqWords {
  int start, next, len;
};
__device__ __forceinline__ SeqWords sequence_words(const AttnArgs& a, int b) {
  const int32_t* at = a.starts ? a.starts + b : a.lens + b;
  return {at[0], at[a.starts ? 1 : 0], a.lens[b]};
}

// (the result is held in scalar registers)
__device__ __forceinline__ Seq sequence(const CacheView& c, const AttnArgs& a, int b, const SeqWords& w, bool reports) {
  Seq s;
  s.first = b;
  s.n = 1;
  bool bad = false;
  if (a.starts) {
    const int s0 = __builtin_amdgcn_readfirstlane(w.start);
    const int s1 = __builtin_amdgcn_readfirstlane(w.next);
    s.first = s0 < 0 ? 0 : s0 > a.tokens ? a.tokens : s0;
    const int end = s1 > a.tokens ? a.tokens : s1;
    s.n = end > s.first ? end - s.first : 0;
    bad = s.n > a.max_queries;
  }
  const int len = __builtin_amdgcn_readfirstlane(w.len);
  s.context = (len < 0 ? 0 : len) - s.n;
  if (s.n > a.max_queries) s.n = a.max_queries;
  const int64_t table = (int64_t)a.width << c.page_shift;
  const int most = table < a.max_len ? (int)table : a.max_len;
  s.len = len < 0 ? 0 : len > most ? most : len;
  if (reports && (bad || len < 0 || len > most)) report(c.status, kBadLength);
  return s;
}

// 64 entries of sequence b's page table from entry i on, one per lane
__device__ __forceinline__ int table_entries(const AttnArgs& a, int b, int i, int lane) {
  return i + lane < a.width ? a.table[(int64_t)b * a.width + i + lane] : -1;
}

// fn(dim, int8) as constants: the cache's two head sizes and formats
template <typename Fn>
void by_layout(const CacheView& c, Fn fn) {
  if (c.dim == 64)
    c.int8 ? fn(std::integral_constant<int, 64>{}, std::true_type{})
           : fn(std::integral_constant<int, 64>{}, std::false_type{});
  else
    c.int8 ? fn(std::integral_constant<int, 128>{}, std::true_type{})
           : fn(std::integral_constant<int, 128>{}, std::false_type{});
}

}  // namespace nkt
