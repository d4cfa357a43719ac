/*
 * nkt_lora.h -- C ABI of low-rank adapters of many requests beside a shared
 * projection (MI355X, gfx950).
 *
 * Same conventions as nkt_moe.h: one handle per projection, device buffers owned
 * by the caller, every entry point enqueues on the given HIP stream and returns
 * without synchronising the host; NKT_LORA_OK (0) or NKT_LORA_ERR (-1) with a
 * message in err[0..err_len).  Activations and adapters are bf16.
 *
 * A projection may be several of one input side by side (queries, keys and
 * values): parts, each with its own A and B.  For token t with adapter a = index[t]
 * and the columns of part p:
 *   out[t] = base[t] + scale[a, p] (x[t] A[a, p]^T) B[a, p]^T
 * A [rank, in_features], B [columns of p, rank], in fp32 but for the operands of
 * the matrix products and with one rounding of the result.
 *
 * Device buffers, for n adapters, P parts, N columns in all, R the largest rank
 * rounded up to 16, 32, 64 or 128, M = P R rounded up to 32; the ranks that an
 * adapter does not have are zero:
 *   A       bf16 [n, M / 32, in_features / 64, 4, 2, 32, 8]: value [i, m, k, j, h, r, e]
 *           is A row 32 m + r, column 64 k + 32 h + 8 j + e, row p R + q being rank q
 *           of part p;
 *   B       bf16 [n, N / 64, R / 16, 2, 2, 32, 8]: value [i, c, s, o, h, r, e] is column
 *           64 c + 2 r + o, rank 16 s + 8 h + e
 *           (so 64 lanes load the operand of a matrix instruction as 1 KB in one
 *           piece, and a lane's results are pairs of columns side by side);
 *   scales  fp32 [n, P];
 *   ranks   int32 [n, P]: ranks past R count as R, negative ones as 0;
 *   status  one uint32, zeroed by the caller.
 */
#ifndef NKT_LORA_H
#define NKT_LORA_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define NKT_LORA_OK 0
#define NKT_LORA_ERR (-1)

#define NKT_LORA_MAX_PARTS 4
#define NKT_LORA_MAX_RANK 128

/* device buffers for nkt_lora_buffer_bytes / nkt_lora_bind */
#define NKT_LORA_BUF_A 0
#define NKT_LORA_BUF_B 1
#define NKT_LORA_BUF_SCALES 2
#define NKT_LORA_BUF_RANKS 3
#define NKT_LORA_BUF_STATUS 4
#define NKT_LORA_NUM_BUFS 5

/* bits of the status word, which no entry point clears */
#define NKT_LORA_STATUS_BAD_ADAPTER 1u /* an index past the adapters: the token has none */

/* A handle for a projection: in_features a multiple of 64, num_parts parts (1 to
 * NKT_LORA_MAX_PARTS) of out_features[p] columns (multiples of 64), up to
 * num_adapters (4096) adapters of ranks up to max_rank (1 to NKT_LORA_MAX_RANK).  NULL on
 * failure. */
void* nkt_lora_create(int num_adapters, int in_features, const int* out_features, int num_parts, int max_rank,
                      char* err, size_t err_len);
void nkt_lora_destroy(void* handle);

/* Bytes of a device buffer. */
int nkt_lora_buffer_bytes(void* handle, int buffer, size_t* bytes, char* err, size_t err_len);

/* Bind the buffers (NKT_LORA_NUM_BUFS pointers, 16-byte aligned).  What they hold
 * may change between calls (adapters that come and go), ordered by the stream. */
int nkt_lora_bind(void* handle, void* const* ptrs, char* err, size_t err_len);

/* Workspace of a call on num_tokens tokens, up to 2^22 (may be 0). */
int nkt_lora_workspace_bytes(void* handle, int num_tokens, size_t* bytes, char* err, size_t err_len);

/* The adapters' part added to a projection's output.  x bf16 [num_tokens,
 * in_features], base and out bf16 [num_tokens, N], tokens *_stride elements apart
 * (up to 2^27), pointers and strides multiples of 16 bytes; out may be base (with its stride),
 * else it overlaps neither base nor x.  index int64 [num_tokens]: each token's
 * adapter, in any order; negative: none, its output is base bit for bit.  If another
 * stream changes index while the call runs, which adapter a token gets is undefined, and
 * nothing else is written.  Sums are taken in the same order at every call of the same
 * number of tokens. */
int nkt_lora_forward(void* handle, const void* x, int64_t x_stride, const void* base, int64_t base_stride,
                     const int64_t* index, int num_tokens, void* out, int64_t out_stride, void* workspace,
                     size_t workspace_bytes, void* stream, char* err, size_t err_len);

#ifdef __cplusplus
}
#endif

#endif /* NKT_LORA_H */
