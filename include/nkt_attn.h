/*
 * nkt_attn.h -- C ABI of the MI355X (gfx950) attention half of a decoder layer:
 * head norms and rotation, the paged key / value cache, attention over it.
 *
 * Same conventions as nkt_moe.h: one handle per layer shape, device buffers
 * owned by the caller, every entry point enqueues on the given HIP stream and
 * returns without synchronising the host; NKT_ATTN_OK (0) or NKT_ATTN_ERR (-1)
 * with a message in err[0..err_len).  Activations are bf16.
 *
 * The cache of one layer is num_pages pages of page_size tokens for num_kv_heads
 * heads of head_dim (D) values.  Slot s is token s % page_size of page
 * s / page_size.  Device layouts (es: 2 bytes bf16, 1 byte int8; U = 16 / es):
 *   keys    [num_pages, num_kv_heads, page_size, D]
 *   values  [num_pages, num_kv_heads, page_size / U, D, U]: 16 bytes hold one
 *           dimension of U consecutive tokens, the operand that one lane of a
 *           matrix instruction takes (tokens are the inner dimension of P . V)
 *   scales  int8 only: fp32 [num_pages, num_kv_heads, page_size], one for keys
 *           and one for values; a value is code * scale, scale = max|row| / 127
 *           (1 for a row of zeros), code = round-half-even(value / scale).  A
 *           row with a NaN or an infinity gets a NaN scale: it reads back as
 *           NaN.
 *
 * Sequences: page_table int32 [num_seqs, table_width] holds each sequence's
 * pages in order; seq_lens int32 [num_seqs] the tokens of it in the cache, this
 * call's included; query_starts int32 [num_seqs + 1], ascending from 0, the
 * rows of q of each sequence (NULL: one row per sequence).  The n rows of a
 * sequence are its last n tokens.
 *
 * What a kernel finds out of range on the device it leaves out and reports as a
 * bit of the status word (NKT_ATTN_STATUS_*), which no entry point clears.
 */
#ifndef NKT_ATTN_H
#define NKT_ATTN_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define NKT_ATTN_OK 0
#define NKT_ATTN_ERR (-1)

/* cache formats */
#define NKT_ATTN_CACHE_BF16 0
#define NKT_ATTN_CACHE_INT8 1

/* device buffers for nkt_attn_cache_bytes / nkt_attn_bind_cache */
#define NKT_ATTN_BUF_K 0
#define NKT_ATTN_BUF_V 1
#define NKT_ATTN_BUF_K_SCALES 2
#define NKT_ATTN_BUF_V_SCALES 3
#define NKT_ATTN_BUF_STATUS 4 /* one uint32, zeroed by the caller */
#define NKT_ATTN_NUM_BUFS 5

/* bits of the status word */
#define NKT_ATTN_STATUS_BAD_SLOT 1u     /* a slot past the cache: not stored, read as zeros */
#define NKT_ATTN_STATUS_BAD_POSITION 2u /* a position outside the rotation table, of a token that is not padding:
                                           queries zero, nothing stored */
#define NKT_ATTN_STATUS_BAD_PAGE 4u     /* a page outside the cache: its tokens are not seen, not moved */
#define NKT_ATTN_STATUS_BAD_LENGTH 8u   /* a length past max_seq_len or the table (cut), negative (0), or a sequence
                                           with more than max_queries rows (the rest left as they were) */
#define NKT_ATTN_STATUS_BAD_KEPT 16u    /* a kept index smaller than its place or past the table, a
                                           count past kept_width, a negative context: not moved */

/* A handle for one layer shape: num_heads a multiple of num_kv_heads (query
 * head i reads key / value head i / (num_heads / num_kv_heads)), head_dim 64 or
 * 128, page_size 64, 128 or 256.  NULL on failure. */
void* nkt_attn_create(int num_heads, int num_kv_heads, int head_dim, int cache_format, int page_size,
                      int64_t num_pages, char* err, size_t err_len);
void nkt_attn_destroy(void* handle);

/* Bytes of a device buffer (0: the handle has none). */
int nkt_attn_cache_bytes(void* handle, int buffer, size_t* bytes, char* err, size_t err_len);

/* Bind the buffers (NKT_ATTN_NUM_BUFS pointers, 16-byte aligned, NULL where
 * nkt_attn_cache_bytes is 0).  Calls made before bind_cache fail. */
int nkt_attn_bind_cache(void* handle, void* const* ptrs, char* err, size_t err_len);

/* Head norms, rotation and the cache write in one launch, for num_tokens new
 * tokens.  q [T, num_heads, D], k and v [T, num_kv_heads, D]: heads contiguous,
 * tokens *_stride elements apart (so the three may be parts of one projection's
 * output), pointers and strides multiples of 8 bytes.
 *   y = x / sqrt(mean(x^2) + eps) * w  per head, where q_norm / k_norm (bf16
 *   [D]) are not NULL;
 *   (y1, y2) -> (y1 cos - y2 sin, y2 cos + y1 sin) on the two halves of a head,
 *   cos | sin = row positions[t] of rope fp32 [rope_rows, D];
 * in fp32 with one rounding, to bf16 for q_out [T, num_heads, D] (which may be
 * q itself if its tokens are dense) and to the cache's format for the keys;
 * values are stored as they are.  slots int64 [T]: where each token's key and value go; a negative slot
 * stores nothing (padding, whose position may be anything: outside the table
 * its queries are zero).  The slots of one call are distinct: what a slot
 * given twice holds is undefined. */
int nkt_attn_write(void* handle, const void* q, int64_t q_stride, const void* k, int64_t k_stride, const void* v,
                   int64_t v_stride, const int64_t* positions, const int64_t* slots, const float* rope,
                   int64_t rope_rows, const void* q_norm, const void* k_norm, float eps, int num_tokens, void* q_out,
                   void* stream, char* err, size_t err_len);

/* The cache read back: keys and values of num_slots slots (int64, in any order,
 * repeated ones too) to k_out and v_out, bf16 [num_slots, num_kv_heads, D].  A
 * negative slot reads as zeros. */
int nkt_attn_read(void* handle, const int64_t* slots, int num_slots, void* k_out, void* v_out, void* stream, char* err,
                  size_t err_len);

/* Keep the accepted tokens of a draft: in each sequence b the key and value at
 * position context[b] + kept[b, i] move to position context[b] + i, for i <
 * counts[b].  context int32 [num_seqs]: the tokens before the draft; kept int32
 * [num_seqs, kept_width], ascending in each row up to its count; counts int32
 * [num_seqs] (0: padding, whose context may be anything).  No two sequences may
 * share a page that a draft reaches into. */
int nkt_attn_keep(void* handle, const int32_t* page_table, int table_width, const int32_t* context,
                  const int32_t* kept, int kept_width, const int32_t* counts, int num_seqs, void* stream, char* err,
                  size_t err_len);

/* Workspace of a forward call (may be 0) of the same sizes.  max_queries: at
 * least the most rows of one sequence (1 for calls without query_starts);
 * max_seq_len: at least the longest sequence.  They choose the launch, so bounds
 * far above what comes cost time.  Refused: over 2^27 rows x heads, 2^30 tokens
 * of a sequence, or 2^24 workgroups of a launch. */
int nkt_attn_workspace_bytes(void* handle, int num_tokens, int num_seqs, int max_queries, int max_seq_len,
                             size_t* bytes, char* err, size_t err_len);

/* Causal attention over the cache (scale > 0): out[i] = sum_j softmax_j(scale q_i . k_j) v_j
 * over the positions j <= seq_len - n + i of the sequence's i-th row (i < n).
 * q and out (which may be q itself) bf16 [num_tokens, num_heads, D], contiguous,
 * 16-byte aligned.  A row that sees nothing, or whose scores are all -infinity,
 * is zero; rows behind the last sequence are left as they were.  A token that a
 * row does not see does not reach it, whatever the cache holds there.  Scores
 * (and scale q . k log2(e)) are fp32: those past its range, and a row's that lie
 * more than 2^127 apart, count as infinite. */
int nkt_attn_forward(void* handle, const void* q, const int32_t* page_table, int table_width, const int32_t* seq_lens,
                     const int32_t* query_starts, int num_tokens, int num_seqs, int max_queries, int max_seq_len,
                     float scale, void* out, void* workspace, size_t workspace_bytes, void* stream, char* err,
                     size_t err_len);

/* The same for drafted tokens: a row sees the seq_len - n tokens before the
 * draft, and the draft's j-th token where bit j % 64 of word j / 64 of its row
 * of tree_mask (int64 [num_tokens, mask_words]) is set; its own bit included,
 * nothing is implied, and tokens past the last word are not seen. */
int nkt_attn_forward_tree(void* handle, const void* q, const int64_t* tree_mask, int mask_words,
                          const int32_t* page_table, int table_width, const int32_t* seq_lens,
                          const int32_t* query_starts, int num_tokens, int num_seqs, int max_queries, int max_seq_len,
                          float scale, void* out, void* workspace, size_t workspace_bytes, void* stream, char* err,
                          size_t err_len);

#ifdef __cplusplus
}
#endif

#endif /* NKT_ATTN_H */
