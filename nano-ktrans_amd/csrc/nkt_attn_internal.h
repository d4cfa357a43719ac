// Launch wrappers of the attention kernels, shared with their C ABI
// (include/nkt_attn.h).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace nkt {

// One layer's paged cache as the kernels address it (layouts in
// include/nkt_attn.h).  A (page, head) block holds page_size x D values of
// keys and as many of values; blocks are addressed with 64-bit offsets, the
// inside of one with 32-bit ones.
struct CacheView {
  uint8_t* k;
  uint8_t* v;
  float* k_scales;  // int8 only
  float* v_scales;
  uint32_t* status;
  int64_t num_pages;
  int kv_heads;
  int page_shift;  // log2 of the page size
  int int8;
  int dim;
};

struct WriteArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  int64_t q_stride, k_stride, v_stride;  // elements between tokens
  const int64_t* positions;
  const int64_t* slots;
  const float* rope;  // [rope_rows, D]: cos, then sin
  int64_t rope_rows;
  const uint16_t* q_norm;  // [D] or nullptr
  const uint16_t* k_norm;
  float eps;
  int tokens, heads;
  uint16_t* q_out;
  // several axes of positions: [num_axes, tokens], two bits for each frequency's axis
  int num_axes;
  uint32_t axis_of[4];
};

hipError_t launch_cache_write(const CacheView& c, const WriteArgs& a, hipStream_t stream);
hipError_t launch_cache_read(const CacheView& c, const int64_t* slots, int n, uint16_t* k_out, uint16_t* v_out,
                             hipStream_t stream);
hipError_t launch_cache_keep(const CacheView& c, const int32_t* table, int width, const int32_t* context,
                             const int32_t* kept, int kept_width, const int32_t* counts, int seqs,
                             hipStream_t stream);

struct AttnArgs {
  const uint16_t* q;  // [tokens, heads, D]
  uint16_t* out;
  const int32_t* table;  // [seqs, width]
  const int32_t* lens;
  const int32_t* starts;  // nullptr: row b is sequence b
  const int64_t* tree;    // [tokens, words] or nullptr (causal)
  int words;
  int width;
  int tokens, seqs, heads;
  int max_queries, max_len;
  float scale;
  // For the weights of the cached tokens, or nullptr: each row's maximum (log2) and sum
  // of weights, [tokens, heads, 2]; in the row form, its scores instead, [seqs,
  // kv_heads, rows, score_row] with the sequence's rows (the statistics lie with the parts).
  float* stats;
  float* scores;
  int score_row;
};

// Workgroups of the call's largest launch.
int64_t attn_workgroups(const CacheView& c, int heads, int tokens, int seqs, int max_queries, int max_len);
size_t attn_workspace_bytes(const CacheView& c, int heads, int tokens, int seqs, int max_queries, int max_len);
hipError_t launch_attn(const CacheView& c, const AttnArgs& a, void* workspace, hipStream_t stream);

// What cached tokens got of a forward call's weights (which kept attn.stats, the
// first tokens x heads x 2 floats of the workspace).
struct WeighArgs {
  AttnArgs attn;
  float* weights;  // of sequence b, head h, position p at b seq_stride + h head_stride + p
  int64_t seq_stride, head_stride;
  int last;  // rows of a sequence's last so many tokens count
  // set by the launch
  int blocks, chunks, chunk_rows, row_blocks;
  int32_t* extreme;  // [seqs, kv_heads, row_blocks] of 256 rows: whether some maximum is extreme
  float* parts;  // [chunks, seqs, kv_heads, blocks of tokens]
};
int64_t weigh_workgroups(const CacheView& c, int heads, int seqs, int max_queries, int max_len, int last);
size_t weigh_workspace_floats(const CacheView& c, int heads, int tokens, int seqs, int max_queries, int max_len,
                              int last);
hipError_t launch_weigh(const CacheView& c, WeighArgs w, float* workspace, hipStream_t stream);

// Both in the row form, by scores kept in the workspace: while these take no more than
// 1 GiB.  (0 bytes: not so.)
size_t attn_scores_workspace_bytes(const CacheView& c, int heads, int tokens, int seqs, int max_queries, int max_len);
hipError_t launch_attn_scores(const CacheView& c, WeighArgs w, void* workspace, hipStream_t stream);

// Eviction: every pointer as in nkt_attn_evict.
struct EvictArgs {
  const int32_t* table;
  int width, seqs, max_len, recent;
  const int32_t* lens;
  const int32_t* budgets;
  const float* weights;
  float* out;  // may be weights, with its strides
  int64_t seq_stride, head_stride, out_seq_stride, out_head_stride;
  int weights_width;
  int32_t* lens_out;
  int32_t* moves;  // workspace
};
size_t evict_workspace_bytes(const CacheView& c, int seqs, int max_len);
hipError_t launch_evict(const CacheView& c, const EvictArgs& e, hipStream_t stream);

}  // namespace nkt
