// C ABI of the attention half (declared in include/nkt_attn.h).
#include <stdarg.h>
#include <stdio.h>

#include <new>

#include "../../include/nkt_attn.h"
#include "nkt_attn_internal.h"

namespace {

using namespace nkt;

struct AttnHandle {
  int heads;
  CacheView cache;
  bool bound;
};

void set_err(char* err, size_t len, const char* fmt, ...) {
  if (!err || len == 0) return;
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(err, len, fmt, ap);
  va_end(ap);
}

bool check_hip(hipError_t e, const char* what, char* err, size_t len) {
  if (e == hipSuccess) return true;
  set_err(err, len, "%s: %s", what, hipGetErrorString(e));
  return false;
}

bool aligned(const void* p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

// the handle, with its cache bound
AttnHandle* bound_handle(void* handle, char* err, size_t len) {
  AttnHandle* h = (AttnHandle*)handle;
  if (!h) {
    set_err(err, len, "null handle");
    return nullptr;
  }
  if (!h->bound) {
    set_err(err, len, "no cache bound (nkt_attn_bind_cache)");
    return nullptr;
  }
  return h;
}

// Rows x heads of a call, tokens of a sequence, and workgroups of a launch
// (whose threads HIP counts in 32 bits).
constexpr int64_t kMaxRows = (int64_t)1 << 27;
constexpr int64_t kMaxTokens = (int64_t)1 << 30;
constexpr int64_t kMaxGroups = ((int64_t)1 << 24) - 1;

// the sizes of a forward call
bool check_sizes(const AttnHandle* h, int num_tokens, int num_seqs, int max_queries, int max_seq_len, char* err,
                 size_t len) {
  if (num_tokens < 0 || num_seqs < 0) {
    set_err(err, len, "num_tokens=%d, num_seqs=%d: negative", num_tokens, num_seqs);
    return false;
  }
  if ((int64_t)num_tokens * h->heads > kMaxRows || (int64_t)num_seqs * h->heads > kMaxRows) {
    set_err(err, len, "num_tokens=%d, num_seqs=%d: over 2^27 rows of %d heads", num_tokens, num_seqs, h->heads);
    return false;
  }
  if (max_queries < 0 || max_seq_len < 0 || max_seq_len > kMaxTokens) {
    set_err(err, len, "max_queries=%d, max_seq_len=%d: outside [0, 2^30]", max_queries, max_seq_len);
    return false;
  }
  if (attn_workgroups(h->cache, h->heads, num_tokens, num_seqs, max_queries, max_seq_len) > kMaxGroups) {
    set_err(err, len, "num_seqs=%d of up to max_seq_len=%d tokens: over 2^24 workgroups", num_seqs, max_seq_len);
    return false;
  }
  return true;
}

int forward(void* handle, const void* q, const int64_t* tree_mask, int mask_words, const int32_t* page_table,
            int table_width, const int32_t* seq_lens, const int32_t* query_starts, int num_tokens, int num_seqs,
            int max_queries, int max_seq_len, float scale, void* out, void* workspace, size_t workspace_bytes,
            void* stream, char* err, size_t len) {
  AttnHandle* h = bound_handle(handle, err, len);
  if (!query_starts) max_queries = 1;
  if (!h || !check_sizes(h, num_tokens, num_seqs, max_queries, max_seq_len, err, len)) return NKT_ATTN_ERR;
  if (table_width < 0 || ((int64_t)table_width << h->cache.page_shift) > kMaxTokens) {
    set_err(err, len, "table_width=%d: outside [0, 2^30 tokens]", table_width);
    return NKT_ATTN_ERR;
  }
  if (!query_starts && num_tokens != num_seqs) {
    set_err(err, len, "no query_starts: num_tokens=%d and num_seqs=%d differ", num_tokens, num_seqs);
    return NKT_ATTN_ERR;
  }
  if (num_tokens == 0 || num_seqs == 0) return NKT_ATTN_OK;
  if (!q || !out || !seq_lens || (!page_table && table_width > 0)) {
    set_err(err, len, "null q, out, seq_lens or page_table");
    return NKT_ATTN_ERR;
  }
  if (!(scale > 0.f) || !(scale < 1e30f)) {
    set_err(err, len, "scale=%g: a positive number wanted", (double)scale);
    return NKT_ATTN_ERR;
  }
  if (!aligned(q, 16) || !aligned(out, 16)) {
    set_err(err, len, "q and out must be 16-byte aligned");
    return NKT_ATTN_ERR;
  }
  const size_t need = attn_workspace_bytes(h->cache, h->heads, num_tokens, num_seqs, max_queries, max_seq_len);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned(workspace, 16))) {
    set_err(err, len, "workspace of %zu bytes, 16-byte aligned, needed; got %zu", need, workspace_bytes);
    return NKT_ATTN_ERR;
  }
  AttnArgs a = {};
  a.q = (const uint16_t*)q;
  a.out = (uint16_t*)out;
  a.table = page_table;
  a.lens = seq_lens;
  a.starts = query_starts;
  a.tree = tree_mask;
  a.words = mask_words;
  a.width = table_width;
  a.tokens = num_tokens;
  a.seqs = num_seqs;
  a.heads = h->heads;
  a.max_queries = max_queries;
  a.max_len = max_seq_len;
  a.scale = scale;
  if (!check_hip(launch_attn(h->cache, a, workspace, (hipStream_t)stream), "attention kernel", err, len))
    return NKT_ATTN_ERR;
  return NKT_ATTN_OK;
}

}  // namespace

extern "C" {

void* nkt_attn_create(int num_heads, int num_kv_heads, int head_dim, int cache_format, int page_size,
                      int64_t num_pages, char* err, size_t err_len) {
  if (num_kv_heads < 1 || num_heads < num_kv_heads || num_heads % num_kv_heads || num_heads > 1024) {
    set_err(err, err_len, "num_heads=%d: a multiple of num_kv_heads=%d up to 1024 wanted", num_heads, num_kv_heads);
    return nullptr;
  }
  if (head_dim != 64 && head_dim != 128) {
    set_err(err, err_len, "head_dim=%d: 64 or 128 supported", head_dim);
    return nullptr;
  }
  if (cache_format != NKT_ATTN_CACHE_BF16 && cache_format != NKT_ATTN_CACHE_INT8) {
    set_err(err, err_len, "unknown cache_format %d", cache_format);
    return nullptr;
  }
  if (page_size != 64 && page_size != 128 && page_size != 256) {
    set_err(err, err_len, "page_size=%d: 64, 128 or 256 supported", page_size);
    return nullptr;
  }
  if (num_pages < 1 || num_pages > INT32_MAX) {
    set_err(err, err_len, "num_pages=%lld outside [1, 2^31)", (long long)num_pages);
    return nullptr;
  }
  AttnHandle* h = new (std::nothrow) AttnHandle();
  if (!h) {
    set_err(err, err_len, "out of host memory");
    return nullptr;
  }
  h->heads = num_heads;
  h->cache.num_pages = num_pages;
  h->cache.kv_heads = num_kv_heads;
  h->cache.page_shift = page_size == 64 ? 6 : page_size == 128 ? 7 : 8;
  h->cache.int8 = cache_format == NKT_ATTN_CACHE_INT8;
  h->cache.dim = head_dim;
  return h;
}

void nkt_attn_destroy(void* handle) { delete (AttnHandle*)handle; }

int nkt_attn_cache_bytes(void* handle, int buffer, size_t* bytes, char* err, size_t err_len) {
  AttnHandle* h = (AttnHandle*)handle;
  if (!h || !bytes) {
    set_err(err, err_len, "null handle or output pointer");
    return NKT_ATTN_ERR;
  }
  if (buffer < 0 || buffer >= NKT_ATTN_NUM_BUFS) {
    set_err(err, err_len, "buffer=%d outside [0, %d)", buffer, NKT_ATTN_NUM_BUFS);
    return NKT_ATTN_ERR;
  }
  const CacheView& c = h->cache;
  const size_t rows = ((size_t)c.num_pages * c.kv_heads) << c.page_shift;
  if (buffer == NKT_ATTN_BUF_STATUS)
    *bytes = 4;
  else if (buffer == NKT_ATTN_BUF_K || buffer == NKT_ATTN_BUF_V)
    *bytes = rows * c.dim * (c.int8 ? 1 : 2);
  else
    *bytes = c.int8 ? rows * 4 : 0;
  return NKT_ATTN_OK;
}

int nkt_attn_bind_cache(void* handle, void* const* ptrs, char* err, size_t err_len) {
  AttnHandle* h = (AttnHandle*)handle;
  if (!h || !ptrs) {
    set_err(err, err_len, "bad arguments");
    return NKT_ATTN_ERR;
  }
  for (int i = 0; i < NKT_ATTN_NUM_BUFS; ++i) {
    const bool scales = i == NKT_ATTN_BUF_K_SCALES || i == NKT_ATTN_BUF_V_SCALES;
    if (scales && !h->cache.int8) continue;
    if (!ptrs[i] || !aligned(ptrs[i], i == NKT_ATTN_BUF_STATUS ? 4 : 16)) {
      set_err(err, err_len, "buffer %d: null or not 16-byte aligned", i);
      return NKT_ATTN_ERR;
    }
  }
  h->cache.k = (uint8_t*)ptrs[NKT_ATTN_BUF_K];
  h->cache.v = (uint8_t*)ptrs[NKT_ATTN_BUF_V];
  h->cache.k_scales = (float*)ptrs[NKT_ATTN_BUF_K_SCALES];
  h->cache.v_scales = (float*)ptrs[NKT_ATTN_BUF_V_SCALES];
  h->cache.status = (uint32_t*)ptrs[NKT_ATTN_BUF_STATUS];
  h->bound = true;
  return NKT_ATTN_OK;
}

int nkt_attn_write(void* handle, const void* q, int64_t q_stride, const void* k, int64_t k_stride, const void* v,
                   int64_t v_stride, const int64_t* positions, const int64_t* slots, const float* rope,
                   int64_t rope_rows, const void* q_norm, const void* k_norm, float eps, int num_tokens, void* q_out,
                   void* stream, char* err, size_t err_len) {
  AttnHandle* h = bound_handle(handle, err, err_len);
  if (!h) return NKT_ATTN_ERR;
  if (num_tokens < 0 || (int64_t)num_tokens * (h->heads + 2 * h->cache.kv_heads) > kMaxRows) {
    set_err(err, err_len, "num_tokens=%d: negative, or over 2^27 rows of all heads", num_tokens);
    return NKT_ATTN_ERR;
  }
  if (rope_rows < 1) {
    set_err(err, err_len, "rope_rows=%lld: at least one row wanted", (long long)rope_rows);
    return NKT_ATTN_ERR;
  }
  if (num_tokens == 0) return NKT_ATTN_OK;
  if (!q || !k || !v || !positions || !slots || !rope || !q_out) {
    set_err(err, err_len, "null q, k, v, positions, slots, rope or q_out");
    return NKT_ATTN_ERR;
  }
  if (!aligned(q, 8) || !aligned(k, 8) || !aligned(v, 8) || !aligned(q_out, 8) || !aligned(q_norm, 8) ||
      !aligned(k_norm, 8) || !aligned(rope, 16) || q_stride % 4 || k_stride % 4 || v_stride % 4) {
    set_err(err, err_len, "q, k, v, q_out and norm weights (and strides) must be 8-byte aligned, rope 16-byte");
    return NKT_ATTN_ERR;
  }
  WriteArgs a = {};
  a.q = (const uint16_t*)q;
  a.k = (const uint16_t*)k;
  a.v = (const uint16_t*)v;
  a.q_stride = q_stride;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.positions = positions;
  a.slots = slots;
  a.rope = rope;
  a.rope_rows = rope_rows;
  a.q_norm = (const uint16_t*)q_norm;
  a.k_norm = (const uint16_t*)k_norm;
  a.eps = eps;
  a.tokens = num_tokens;
  a.heads = h->heads;
  a.q_out = (uint16_t*)q_out;
  if (!check_hip(launch_cache_write(h->cache, a, (hipStream_t)stream), "cache write kernel", err, err_len))
    return NKT_ATTN_ERR;
  return NKT_ATTN_OK;
}

int nkt_attn_read(void* handle, const int64_t* slots, int num_slots, void* k_out, void* v_out, void* stream, char* err,
                  size_t err_len) {
  AttnHandle* h = bound_handle(handle, err, err_len);
  if (!h) return NKT_ATTN_ERR;
  if (num_slots < 0 || (int64_t)num_slots * h->cache.kv_heads > kMaxRows) {
    set_err(err, err_len, "num_slots=%d: negative, or over 2^27 rows of all heads", num_slots);
    return NKT_ATTN_ERR;
  }
  if (num_slots == 0) return NKT_ATTN_OK;
  if (!slots || !k_out || !v_out || !aligned(k_out, 16) || !aligned(v_out, 16)) {
    set_err(err, err_len, "slots, k_out and v_out must be given, the outputs 16-byte aligned");
    return NKT_ATTN_ERR;
  }
  if (!check_hip(launch_cache_read(h->cache, slots, num_slots, (uint16_t*)k_out, (uint16_t*)v_out,
                                   (hipStream_t)stream),
                 "cache read kernel", err, err_len))
    return NKT_ATTN_ERR;
  return NKT_ATTN_OK;
}

int nkt_attn_keep(void* handle, const int32_t* page_table, int table_width, const int32_t* context,
                  const int32_t* kept, int kept_width, const int32_t* counts, int num_seqs, void* stream, char* err,
                  size_t err_len) {
  AttnHandle* h = bound_handle(handle, err, err_len);
  if (!h) return NKT_ATTN_ERR;
  if (num_seqs < 0 || (int64_t)num_seqs * h->cache.kv_heads > kMaxGroups) {
    set_err(err, err_len, "num_seqs=%d: negative, or over 2^24 workgroups", num_seqs);
    return NKT_ATTN_ERR;
  }
  if (table_width < 0 || kept_width < 0 || ((int64_t)table_width << h->cache.page_shift) > kMaxTokens) {
    set_err(err, err_len, "table_width=%d, kept_width=%d: negative, or over 2^30 tokens", table_width, kept_width);
    return NKT_ATTN_ERR;
  }
  if (num_seqs == 0 || table_width == 0 || kept_width == 0) return NKT_ATTN_OK;
  if (!page_table || !context || !kept || !counts) {
    set_err(err, err_len, "null page_table, context, kept or counts");
    return NKT_ATTN_ERR;
  }
  if (!check_hip(launch_cache_keep(h->cache, page_table, table_width, context, kept, kept_width, counts, num_seqs,
                                   (hipStream_t)stream),
                 "cache keep kernel", err, err_len))
    return NKT_ATTN_ERR;
  return NKT_ATTN_OK;
}

int nkt_attn_workspace_bytes(void* handle, int num_tokens, int num_seqs, int max_queries, int max_seq_len,
                             size_t* bytes, char* err, size_t err_len) {
  AttnHandle* h = (AttnHandle*)handle;
  if (!h || !bytes) {
    set_err(err, err_len, "null handle or output pointer");
    return NKT_ATTN_ERR;
  }
  if (!check_sizes(h, num_tokens, num_seqs, max_queries, max_seq_len, err, err_len)) return NKT_ATTN_ERR;
  *bytes = attn_workspace_bytes(h->cache, h->heads, num_tokens, num_seqs, max_queries, max_seq_len);
  return NKT_ATTN_OK;
}

int nkt_attn_forward(void* handle, const void* q, const int32_t* page_table, int table_width, const int32_t* seq_lens,
                     const int32_t* query_starts, int num_tokens, int num_seqs, int max_queries, int max_seq_len,
                     float scale, void* out, void* workspace, size_t workspace_bytes, void* stream, char* err,
                     size_t err_len) {
  return forward(handle, q, nullptr, 0, page_table, table_width, seq_lens, query_starts, num_tokens, num_seqs,
                 max_queries, max_seq_len, scale, out, workspace, workspace_bytes, stream, err, err_len);
}

int nkt_attn_forward_tree(void* handle, const void* q, const int64_t* tree_mask, int mask_words,
                          const int32_t* page_table, int table_width, const int32_t* seq_lens,
                          const int32_t* query_starts, int num_tokens, int num_seqs, int max_queries, int max_seq_len,
                          float scale, void* out, void* workspace, size_t workspace_bytes, void* stream, char* err,
                          size_t err_len) {
  if ((num_tokens > 0 && !tree_mask) || mask_words < 1 || (int64_t)num_tokens * mask_words > kMaxTokens) {
    set_err(err, err_len, "tree_mask of at least one word per row (and at most 2^30 in all) wanted, got %d", mask_words);
    return NKT_ATTN_ERR;
  }
  return forward(handle, q, tree_mask, mask_words, page_table, table_width, seq_lens, query_starts, num_tokens,
                 num_seqs, max_queries, max_seq_len, scale, out, workspace, workspace_bytes, stream, err, err_len);
}

}  // extern "C"
