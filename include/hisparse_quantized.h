/*
 * hisparse_quantized.h — C ABI of libhisparse.so, third part: a cache whose rows
 * are held in 8 bits.
 *
 *   (9)  append: rows quantised as they are written, with the page's metadata
 *   (10) reading rows back
 *   (11) decode attention over physical rows
 *
 * A row (one token's K, or its V) is held as a record of
 * hs_quantized_row_bytes(kv_heads, head_dim) bytes: kv_heads * head_dim e4m3
 * codes, kv_heads bytes with the heads' scales, zeros up to a multiple of 32.
 * With x a head's head_dim elements and a the largest |x_d| of the finite ones,
 *   e        = the smallest whole number with a <= 448 * 2^e, at least -100
 *   code_d   = x_d * 2^-e rounded to e4m3 (to nearest, ties to even); an
 *              element that is not finite is held as NaN
 *   scale    = e + 127, one byte; the value held is code_d * 2^e
 * A floating-point code gains nothing from a scale between powers of two but up
 * to one bit of its smallest numbers, and these make every result exact: the
 * scaled element in fp32, the value held in bf16 and fp32. Rows have scales of
 * their own because the resolver moves them alone between host and pool. No scale is 0:
 * a record of zeros, as in cleared memory, holds nothing; attention does not see
 * such a row, and reading it gives zeros.
 *
 *   pool   [pool_blocks, 2 (K|V), page_size, record]   bytes, 16-byte aligned
 *   host   [host_blocks, 2 (K|V), page_size, record]
 * hs_gather_rows moves such rows with row_bytes = the record's; hs_resolve_rows
 * does not look at them; hs_quest_* reads metadata in bf16, which holds every
 * bound exactly.
 *
 * The conventions are those of hisparse.h: borrowed pointers on the current
 * device, caller-provided workspace, everything enqueued on `stream` without a
 * host synchronisation, an hs_status returned and hs_last_error() set, HS_DEV_*
 * bits ORed into the optional `device_status`. None of these operators keeps
 * state between calls, and all of them can be captured in a CUDA graph.
 * head_dim is at most 256.
 */
#ifndef HISPARSE_QUANTIZED_H
#define HISPARSE_QUANTIZED_H

#include "hisparse.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Bytes of a row's record; 0 for invalid sizes. */
HS_API int64_t hs_quantized_row_bytes(int kv_heads, int head_dim);

/* ---- (9) append ------------------------------------------------------------------
 * As hs_append_rows (hisparse.h), with k and v of dtype kv_dtype quantised on
 * their way into pool and host records (host_block NULL: no host mirror), and with the metadata taken from the
 * values that are held: minimum_ptrs / maximum_ptrs point to bf16 bounds
 * (torch.minimum / torch.maximum semantics), summary_ptrs to the fp32 mean of the
 * page's rows so far; all three NULL: no metadata. A row of k or v is kv_heads * head_dim adjacent elements,
 * rows of a chunk follow one another, chunks are kv_batch_stride elements apart
 * and have `tokens` rows each; a count above that is refused like one that leaves
 * its page.
 */
HS_API int hs_append_quantized(int batch, int64_t tokens, const void *k, const void *v,
                               int64_t kv_batch_stride, int kv_dtype, const int32_t *within,
                               const int32_t *count,
                               const int64_t *pool_block, void *pool, int64_t pool_blocks,
                               const int64_t *host_block, void *host_alias, int64_t host_blocks,
                               const uint64_t *minimum_ptrs, const uint64_t *maximum_ptrs,
                               const uint64_t *summary_ptrs, int kv_heads, int head_dim,
                               int page_size, int32_t *device_status, hs_stream stream);

/* ---- (10) reading rows back --------------------------------------------------------
 * out [2 (K|V), count, kv_heads, head_dim] of `dtype` takes the values of
 * physical rows rows[0 .. count-1], rounded to nearest once (exact in bf16 and
 * fp32; fp16 overflows to infinity as any conversion does); zeros for a negative
 * row (padding) and for one beyond the pool, which raises
 * HS_DEV_ROW_OUT_OF_RANGE.
 */
HS_API int hs_read_quantized(const void *pool, int64_t pool_blocks, const int64_t *rows,
                             int64_t count, void *out, int dtype, int kv_heads, int head_dim,
                             int page_size, int32_t *device_status, hs_stream stream);

/* ---- (11) decode attention -----------------------------------------------------------
 * out[b,h] = softmax_i(q[b,h] . K_i / sqrt(head_dim)) V_i over the rows i of
 * request b: rows[b, (h,) i] >= 0 with i < counts[b] (NULL: count), whose K and V
 * are the values held; query head h reads KV head h / (q_heads / kv_heads). fp32
 * sums; zeros where nothing is seen. rows int64: head h of request b starts at
 * b * rows_batch_stride + h * rows_head_stride (0: the heads share their rows,
 * which is the fast form, where head_dim is also a multiple of 16 and query and its
 * stride are multiples of four elements; other calls run on CUDA cores). query
 * [batch, q_heads, head_dim] with heads adjacent
 * and requests query_batch_stride elements apart, out contiguous, both of `dtype`.
 * counts below 0 or above `count` are clamped. A row beyond the pool is skipped
 * and raises HS_DEV_ROW_OUT_OF_RANGE.
 *
 * The phase form leaves partial results of one list of rows in the workspace, for
 * the merge to join (rows that need no gather first, gathered rows later): request
 * b has the sum of counts[b * counts_stride + counts_first .. + counts_n) rows
 * (counts NULL: count). phase is 0 or 1 and a merge of `phases` joins phases
 * 0 .. phases - 1, all of one batch, dtype, sizes and `count`.
 *
 * The workspace (phases: 1 for the plain form, 2 for the phase form and its merge, however
 * many phases that joins) is 16-byte aligned and needs no initialisation; calls that may
 * overlap on the GPU need separate ones.
 */
HS_API size_t hs_attend_quantized_workspace_bytes(int batch, int phases, int dtype,
                                                  int q_heads, int kv_heads, int head_dim,
                                                  int64_t count);

HS_API int hs_attend_quantized(int batch, const void *query, int64_t query_batch_stride,
                               int dtype, const void *pool, int64_t pool_blocks,
                               const int64_t *rows, int64_t rows_batch_stride,
                               int64_t rows_head_stride, int64_t count, const int32_t *counts,
                               void *out, int q_heads, int kv_heads, int head_dim, int page_size,
                               void *workspace, size_t workspace_bytes, int32_t *device_status,
                               hs_stream stream);

HS_API int hs_attend_quantized_phase(int batch, const void *query, int64_t query_batch_stride,
                                     int dtype, const void *pool, int64_t pool_blocks,
                                     const int64_t *rows, int64_t rows_batch_stride,
                                     int64_t count, const int64_t *counts, int counts_stride,
                                     int counts_first, int counts_n, int phase, int q_heads,
                                     int kv_heads, int head_dim, int page_size, void *workspace,
                                     size_t workspace_bytes, int32_t *device_status,
                                     hs_stream stream);

HS_API int hs_attend_quantized_merge(int batch, int phases, void *out, int dtype, int q_heads,
                                     int kv_heads, int head_dim, int64_t count, void *workspace,
                                     size_t workspace_bytes, hs_stream stream);

#ifdef __cplusplus
}
#endif

#endif /* HISPARSE_QUANTIZED_H */
