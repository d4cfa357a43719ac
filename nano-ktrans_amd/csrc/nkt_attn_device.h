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
