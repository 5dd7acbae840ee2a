/*
 * hisparse_verify.h — C ABI of libhisparse.so, second part: the operators of a
 * verification step, which checks several drafted tokens of every request in
 * one forward pass.
 *
 *   (6) per-head norms of queries and keys with the position rotation
 *   (7) attention of a tree of drafted tokens over cache rows and the tree
 *   (8) log probabilities of given tokens, entropy and top alternatives
 *
 * The conventions are those of hisparse.h: borrowed pointers on the current
 * device, caller-provided workspace, everything enqueued on `stream` without a
 * host synchronisation, an hs_status returned and hs_last_error() set, HS_DEV_*
 * bits ORed into the optional `device_status`. None of these operators keeps
 * state between calls, and all of them can be captured in a CUDA graph.
 */
#ifndef HISPARSE_VERIFY_H
#define HISPARSE_VERIFY_H

#include "hisparse.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- (6) per-head norms and rotation ------------------------------------------
 * For every token n and head h of the query (q_heads) and the key (kv_heads),
 * with x the head's head_dim elements, R = head_dim / 2 and w the query or key
 * weight (NULL leaves the norm out: y = x):
 *   y_d       = x_d / sqrt(mean(x^2) + eps) * w_d
 *   a_i       = positions[n] * inv_freq[i]                        (i < R)
 *   out_i     = y_i * cos(a_i) - y_{i+R} * sin(a_i)
 *   out_{i+R} = y_{i+R} * cos(a_i) + y_i * sin(a_i)
 * in fp32 with one rounding at the end; the angle is reduced to a fraction of
 * a turn in fp64. Element d of head h of token n is at n * token_stride + h *
 * head_stride + d. Outputs are contiguous [tokens, heads, head_dim].
 * head_dim is even and at most 256; positions are HS_INT32 or HS_INT64.
 */
HS_API int hs_qk_norm_rope(int64_t tokens, const void *query, int64_t query_token_stride,
                           int64_t query_head_stride, int q_heads, const void *key,
                           int64_t key_token_stride, int64_t key_head_stride, int kv_heads,
                           int head_dim, int dtype, const void *positions, int positions_dtype,
                           const double *inv_freq, const void *query_weight,
                           const void *key_weight, float eps, void *query_out, void *key_out,
                           hs_stream stream);

/* ---- (7) attention of a tree of drafted tokens ----------------------------------
 * Request b has node_counts[b] (NULL: `nodes`) drafted tokens and counts[b]
 * (NULL: `count`) selected cache rows. Node t of it sees every valid row
 * (rows[b, i] >= 0, i < counts[b]) of the pool and the nodes j whose bit is
 * set in mask[b, t] (j < node_counts[b]); query head h reads KV head
 * h / (q_heads / kv_heads). With S the K/V pairs seen:
 *   out[b,t,h] = softmax_S(q[b,t,h] . K / sqrt(head_dim)) V
 * in fp32, zero when S is empty and for nodes t >= node_counts[b]. Values of
 * pairs that are not seen take no part, whatever they hold. query is
 * [batch, nodes, q_heads, head_dim], key and value [batch, nodes, kv_heads,
 * head_dim] with heads adjacent and the given batch and node strides (elements);
 * the pool layout is hisparse.h's. All tensors have one dtype; nodes <= 64,
 * head_dim <= 256. rows int64 [batch, count] (rows_batch_stride between
 * requests), mask int64 [batch, nodes], counts and node_counts int32 [batch];
 * counts below 0 or above their limit are clamped. out is contiguous
 * [batch, nodes, q_heads, head_dim]. A row beyond the pool is skipped and
 * raises HS_DEV_ROW_OUT_OF_RANGE. The workspace is 16-byte aligned and
 * needs no initialisation; calls that may overlap on the GPU need separate ones.
 * Every other address has its element's alignment; 16-bit calls are an order of
 * magnitude faster where all of them, out included, are multiples of 16 bytes.
 */
HS_API size_t hs_attend_tree_workspace_bytes(int batch, int nodes, int q_heads, int kv_heads,
                                             int head_dim, int64_t count, int dtype);

HS_API int hs_attend_tree(int batch, int nodes, const void *query, int64_t query_batch_stride,
                          int64_t query_node_stride, const void *key, const void *value,
                          int64_t kv_batch_stride, int64_t kv_node_stride, int dtype,
                          const int64_t *mask, const int32_t *node_counts, const void *pool,
                          int64_t pool_blocks, const int64_t *rows, int64_t rows_batch_stride,
                          int64_t count, const int32_t *counts, void *out, int q_heads,
                          int kv_heads, int head_dim, int page_size, void *workspace,
                          size_t workspace_bytes, int32_t *device_status, hs_stream stream);

/* ---- (8) log probabilities, entropy, alternatives --------------------------------
 * For every row x of logits [rows, vocab] (row_stride elements apart), in fp32:
 *   lse            = log sum_v exp(x_v)
 *   out_logprobs   [rows, given]: x[tokens[r, c]] - lse; 0 for a negative token
 *                  (padding); NaN and HS_DEV_TOKEN_OUT_OF_RANGE for one >= vocab
 *   out_entropy    [rows]: lse - sum_v p_v x_v, p_v = exp(x_v - lse), in nats
 *   out_top_tokens [rows, top] int64: the `top` largest entries, equal values by
 *                  the lower index; out_top_logprobs the same entries' x - lse
 * An entry of -inf has probability 0 and log probability -inf; a row with
 * nothing above -inf has log probabilities -inf and entropy 0. A row that holds
 * NaN or +inf gives NaN log probabilities and entropy; its top entries rank
 * NaN above all numbers. top <= 32 and top <= vocab; vocab < 2^31. tokens are
 * HS_INT32 or HS_INT64 (ignored when given = 0). out_entropy may be NULL.
 */
HS_API int hs_token_logprobs(int64_t rows, const void *logits, int64_t row_stride, int dtype,
                             int64_t vocab, const void *tokens, int tokens_dtype, int given,
                             float *out_logprobs, float *out_entropy, int top,
                             float *out_top_logprobs, int64_t *out_top_tokens,
                             int32_t *device_status, hs_stream stream);

#ifdef __cplusplus
}
#endif

#endif /* HISPARSE_VERIFY_H */
