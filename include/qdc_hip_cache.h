/* qdc_hip_cache.h -- entry points of libqdc_hip.so for decoding from a cache: keys
 * and values in pages that rows of the cache share, and the state of the linear
 * attention layers, one token at a time.  Types, status codes, dtype codes and
 * stream rules are those of qdc_hip.h: nothing is allocated or kept, everything is
 * enqueued on `stream`, and a negative status is returned before anything is
 * enqueued.  The reference recomputes a sequence for every call and has no
 * counterpart of these.
 *
 * A cache of `rows` rows (sequences) and `pages` pages of page_size positions each
 * (16, 32, 64, 128 or 256) holds, all on the device:
 *   k_pages, v_pages  [pages, kv_heads, page_size, head_dim], per layer;
 *   table   int32 [rows, width]: entry j the page of positions j*page_size .. , -1
 *           behind a row's last page;
 *   lengths int32 [rows]: positions that a row holds;
 *   refs    int32 [pages]: rows that share a page;
 *   free    int32 [1 + pages]: a count c, then the free pages as a stack, its top at c.
 * A page that is not full belongs to one row alone.  pages and rows * width are at most
 * 2^31 - 1024, width * page_size below 2^31 (QDC_ERR_SHAPE otherwise).
 *
 * A call's tokens are named by `index` (the row of the cache, int32 [n]) and
 * `positions` (int32 [n]).  An entry whose row or position is negative is no token:
 * its outputs are as said below, nothing of the cache is read or written for it.
 * What the device holds cannot be checked on the host: a row, position or page
 * outside its table is never followed; the kernel then does as each entry point says
 * and, when error_flag is not NULL, sets *error_flag = 1 (device int32, cleared by
 * the caller).
 */
#ifndef QDC_HIP_CACHE_H
#define QDC_HIP_CACHE_H

#include "qdc_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Version of this header, and of the library that was built with it; the minor number
 * changes with a signature, the patch number with added entry points. */
#define QDC_HIP_CACHE_VERSION "qdc_hip_cache 0.1.0"
const char *qdc_cache_version(void);

/* Per-head zero-centred RMSNorm and half-split partial RoPE of q and k heads, as
 * qdc_qk_norm_rope, each token at its own position, with k and v stored into the
 * cache in the same pass: K row (t, g) to place positions[t] % page_size of head g of
 * page table[index[t], positions[t] / page_size], V row (t, g) likewise.  q_out is
 * [tokens, heads, head_dim] contiguous; k_out, where not NULL, takes the K rows too
 * ([tokens, kv_heads, head_dim] contiguous: keys for attention within the prompt).
 * An entry that is no token is normalised, not rotated and not stored; so is one
 * whose position is not below table_len and width * page_size, whose row is not below
 * `rows` or whose page is not one (error_flag).  Two tokens of one row and position
 * leave one of them or a mixture of their 16-byte pieces.
 * Inputs are views with rows of head_dim contiguous elements (strides between tokens
 * and heads in elements); head_dim 64, 128 or 256; pointers and strides of 16 bytes,
 * tokens * (heads + 2 kv_heads) below 2^26 (QDC_ERR_SHAPE otherwise).
 * cos_table and sin_table fp32 [table_len, rotary_dim / 2], unused when rotary_dim is 0.
 * Outputs overlap neither each other nor an input. */
int32_t qdc_prepare_paged(void *q_out, void *k_out, void *k_pages, void *v_pages, const void *q,
                          const void *k, const void *v, const void *q_norm, const void *k_norm,
                          const float *cos_table, const float *sin_table, const int32_t *index,
                          const int32_t *positions, const int32_t *table, int64_t tokens,
                          int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t rotary_dim,
                          int64_t table_len, int64_t rows, int64_t width, int64_t pages,
                          int64_t page_size, int64_t q_tok, int64_t q_head, int64_t k_tok,
                          int64_t k_head, int64_t v_tok, int64_t v_head, float eps, int32_t dtype,
                          int32_t *error_flag, hipStream_t stream);

/* Bytes of 16-byte aligned device scratch that qdc_paged_attention needs (0: none, for
 * short rows), -1 when it does not take the sizes. */
int64_t qdc_paged_attention_workspace(int64_t n, int64_t heads, int64_t kv_heads,
                                      int64_t head_dim, int64_t width, int64_t page_size,
                                      int32_t dtype);

/* Attention of one token's queries over its row of the cache:
 *     out[i, h*head_dim + r] = sigmoid(gate[i, h, r]) *
 *         sum_j softmax_j(scale * q[i, h] . k_j) v_j[r],  j = 0 .. positions[i],
 * k_j and v_j the rows of KV head h / (heads / kv_heads) at position j of cache row
 * index[i]; gate NULL: no gate.  Scores, exponentials, sums and the product with V in
 * fp32 (for bf16 pages the exponentials as two bf16 terms).  An entry that is no
 * token, or whose row is not below `rows`, gives zeros.  Positions behind the table's
 * width, and pages that are not one, are left out as if masked (error_flag); a head that
 * sees no key, or scores of -inf alone, gives zeros.  What a page holds behind the last
 * position, NaN too, is not used.
 * `dtype` is the type of q, gate and the pages; out_dtype may also be QDC_BF16X2.
 * Strides in elements; pointers and strides of 16 bytes; head_dim 64, 128 or 256;
 * scale positive and scale * log2(e) finite (QDC_ERR_RANGE otherwise).  `workspace`
 * is scratch of this call alone.  out may not overlap any other argument. */
int32_t qdc_paged_attention(void *out, int32_t out_dtype, const void *q, const void *k_pages,
                            const void *v_pages, const void *gate, const int32_t *table,
                            const int32_t *index, const int32_t *positions, int64_t n,
                            int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t rows,
                            int64_t width, int64_t pages, int64_t page_size, int64_t q_tok,
                            int64_t q_head, int64_t gate_tok, int64_t gate_head, int64_t out_tok,
                            float scale, int32_t dtype, void *workspace, int64_t workspace_bytes,
                            int32_t *error_flag, hipStream_t stream);

/* counts[i] more positions (counts NULL: one) for row index[i]: lengths grow, and
 * pages come off the stack, in the order of the entries, where a row's last page is
 * full.  positions[i] is the first of them, the row's length before.  An entry with a
 * negative row is left out (position -1).  A call that cannot be done whole is not
 * done at all -- a row twice or not below `rows`, a negative count, a length past
 * width * page_size, more pages than are free: every positions[i] is -1 then
 * (error_flag).  rows < 2^18, n < 2^24. */
int32_t qdc_pages_extend(int32_t *positions, int32_t *table, int32_t *lengths, int32_t *refs,
                         int32_t *free_pages, const int32_t *index, const int32_t *counts,
                         int64_t n, int64_t rows, int64_t width, int64_t pages, int64_t page_size,
                         int32_t *error_flag, hipStream_t stream);

/* Rows index[i] give up their pages and are empty after it.  A page that no row holds
 * any more goes on the stack: of the pages that the rows in their order list, the
 * first is on top (a page that several list counts where it is listed last), so rows
 * freed right after they got their pages leave the stack as it was.  Negative rows
 * are left out; a row twice or not below `rows`: nothing is done (error_flag). */
int32_t qdc_pages_free(int32_t *table, int32_t *lengths, int32_t *refs, int32_t *free_pages,
                       const int32_t *index, int64_t n, int64_t rows, int64_t width,
                       int64_t pages, int64_t page_size, int32_t *error_flag, hipStream_t stream);

/* Row children[i], empty before, becomes a copy of row parents[i]: full pages are
 * shared, a page that is not full is copied into one from the stack, in the order of
 * the entries: of each of the `planes` planes of `pool` ([planes, pages, heads,
 * page_size, token_bytes], NULL with planes 0: no copies) the places that hold a
 * token.  An entry with a negative parent or child is left out.  A child that is not
 * empty, named twice or a parent too, a row not below `rows`, or more pages than are
 * free: nothing is done (error_flag).  `workspace`: qdc_pages_fork_workspace bytes of
 * device scratch (0 where little is copied).  token_bytes a multiple of 16 below 2^20,
 * pool 16-byte aligned. */
int64_t qdc_pages_fork_workspace(int64_t n, int64_t page_size, int64_t planes, int64_t heads,
                                 int64_t token_bytes);
int32_t qdc_pages_fork(int32_t *table, int32_t *lengths, int32_t *refs, int32_t *free_pages,
                       const int32_t *parents, const int32_t *children, int64_t n, int64_t rows,
                       int64_t width, int64_t pages, int64_t page_size, void *pool,
                       int64_t planes, int64_t heads, int64_t token_bytes, void *workspace,
                       int64_t workspace_bytes, int32_t *error_flag, hipStream_t stream);

/* The pages in use move to the low end: with m of them, the k-th page below m that is
 * free takes the data, in every plane of `pool` ([planes, pages, page_bytes]), and the
 * place in tables and refs of the k-th page in use from m on.  The stack then holds
 * the pages from m on, the lowest on top, zeros above it.  `workspace`:
 * qdc_pages_compact_workspace(pages) bytes of device scratch.  page_bytes a multiple
 * of 16. */
int64_t qdc_pages_compact_workspace(int64_t pages);
int32_t qdc_pages_compact(int32_t *table, int32_t *refs, int32_t *free_pages, int64_t rows,
                          int64_t width, int64_t pages, void *pool, int64_t planes,
                          int64_t page_bytes, void *workspace, int64_t workspace_bytes,
                          hipStream_t stream);

/* Items src[i] -> dst[i] in each plane of `pool` ([planes, items, item_bytes]): pages,
 * or whatever a row of the cache holds beside them.  A pair with a negative index is
 * left out.  A pair whose dst is an earlier pair's dst or any pair's src, or that is
 * out of range, is not copied (error_flag).  item_bytes a multiple of 16, pool 16-byte
 * aligned, n at most 4096 (every pair is held against all others). */
int32_t qdc_copy_pages(void *pool, const int32_t *src, const int32_t *dst, int64_t n,
                       int64_t planes, int64_t items, int64_t item_bytes, int32_t *error_flag,
                       hipStream_t stream);

/* One token of a linear attention layer for each entry: what qdc_delta_prologue,
 * qdc_delta_scan and qdc_gated_rmsnorm give for the last of the tokens seen, from
 * what a cache row keeps of those before:
 *   ring  [rows, taps, channels] in proj's type: the qkv block of the token at
 *         position p in slot p % taps (this call writes the new token's);
 *   state fp32 [rows, value_heads, value_dim, key_dim] (read and rewritten).
 * `proj` [n, ld] holds the packed projections [q | k | v | z | a | b].  At position 0
 * a row starts from an empty state, whatever ring and state hold, and taps that reach
 * before position 0 read zero.  out [n, value_heads * value_dim] in out_dtype (proj's
 * type, or QDC_BF16X2 for bf16): the gated norm's result.  An entry that is no token
 * gives zeros and leaves ring and state; so does one whose row is not below `rows` or
 * is that of an earlier token of the call (error_flag).  key_dim 32, 64 or 128,
 * value_dim a multiple of 16 up to 256, taps up to 8, n * value_heads below 2^22; state
 * 16-byte aligned (QDC_ERR_SHAPE otherwise). */
int32_t qdc_delta_step(void *out, int32_t out_dtype, const void *proj, int32_t proj_dtype,
                       int64_t ld, const float *conv, int64_t taps, const float *a_decay,
                       const float *dt_bias, const void *norm, void *ring, float *state,
                       const int32_t *index, const int32_t *positions, int64_t n, int64_t rows,
                       int64_t key_heads, int64_t key_dim, int64_t value_heads, int64_t value_dim,
                       float eps, int32_t *error_flag, hipStream_t stream);

/* qdc_delta_scan_ws that also writes the state after the last token, fp32 [batch,
 * heads, value_dim, key_dim] (16-byte aligned, no overlap with another argument). */
int32_t qdc_delta_scan_state(void *out, int32_t out_dtype, float *state, const float *q,
                             const float *k, const float *v, const float *beta,
                             const float *decay, int64_t batch, int64_t seq, int64_t heads,
                             int64_t key_heads, int64_t key_dim, int64_t value_dim, int64_t ld_qk,
                             int64_t ld_v, void *workspace, int64_t workspace_bytes,
                             hipStream_t stream);

#ifdef __cplusplus
}
#endif
#endif
