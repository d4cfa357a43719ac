// Attention over the paged cache.
#include "nkt_attn_device.h"

namespace nkt {

namespace {

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
    const dim3 grid((unsigned)a.tokens * a.heads);
    if (a.tree)
      hipLaunchKernelGGL((attn_row_kernel<D, I8, true>), grid, dim3(64), 0, stream, c, a);
    else
      hipLaunchKernelGGL((attn_row_kernel<D, I8, false>), grid, dim3(64), 0, stream, c, a);
  });
  return hipGetLastError();
}

}  // namespace nkt
