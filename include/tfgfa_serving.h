/*
 * tfgfa_serving.h - C ABI of the serving operators beside the attention (MI355X, gfx950): one decode
 * step over a paged key-value cache, the attention weight each key has received, eviction from the
 * cache by that weight, and penalties, biases and grammar masks on the logits.
 *
 * The reference's generate() keeps no cache and samples from unmodified logits
 * (src/py/model_inference.py:199-228); there is nothing of this in it.
 *
 * Conventions as in tfgfa.h: device pointers, the caller owns every buffer, launches are asynchronous
 * on `hip_stream`, arguments are checked before any HIP call; 0 on success, > 0 an invalid argument
 * (TFGFA_ERR_*), < 0 a negated hipError_t.  Strides are in elements.  dtype: TFGFA_DTYPE_BF16 or
 * TFGFA_DTYPE_F16; scores, softmax, weights and sums are float32.
 */
#ifndef TFGFA_SERVING_H
#define TFGFA_SERVING_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/*
 * A paged cache: k_pages and v_pages are (P, H_kv, page, D), strides [p, h, n, d] as the caches of
 * tfgfa_decode (last dimension dense, the others non-negative multiples of 8 elements, n >= D).  Row j
 * of sequence b is row j % page of page page_table[b * table_stride + j / page]; page_table is int32
 * (B, M), cache_seqlens B int32, both in device memory, so a sequence holds at most N_max = M * page
 * rows.  Entries of the table past a sequence's last row are not used.  H is a multiple of H_kv: query
 * head h reads key-value head h / (H / H_kv).
 *
 * One decode step, attention of one new query per (batch, head):
 *   L_b = cache_seqlens[b] (+1 when appending)
 *   O[b,h,:] = sum_{j < L_b} softmax_j(scale * q[b,h,:] . K[b,h',j,:]) * V[b,h',j,:]
 *   LSE[b,h] = log sum_{j < L_b} exp(scale * q[b,h,:] . K[b,h',j,:])
 * q, o: (B, H, D) strides [b, h, d]; k_new, v_new: (B, H_kv, D), both NULL or both set: they become row
 * cache_seqlens[b] of the sequence first (the caller advances cache_seqlens afterwards, and gives no
 * two sequences one page for their new rows; a pool whose strides put rows over one another is
 * refused).  lse: (B, H) contiguous or NULL.
 * key_weights: NULL, or float32 (B, H_kv, N >= N_max), strides [b, h] in weights_strides, last dimension
 * dense:
 *   key_weights[b,h',j] += sum over the heads h of h' of softmax_j(...)     j < L_b
 * and, when appending, the new row's entry is set to that sum (whatever it held).  Entries at or past
 * L_b are left alone.  A head whose LSE is not finite adds nothing.
 * A row whose scores are all -inf, and L_b = 0, give O = 0 and LSE = -inf.
 * Visible on the device only: a length that does not fit (cache_seqlens[b] < 0 or + append > N_max)
 * gives NaN in O and LSE for that batch row, which is otherwise left alone; a page id outside [0, P)
 * among a sequence's rows gives NaN in O and LSE too, and nothing is written through it.
 * Values of rows at or past the length never reach the result.
 * Sums of weighted values are float32 before the sum of weights, up to e^8 L, divides them: bf16 values past
 * 3.4e38 / (2981 L_b) can make them infinite.
 *
 * workspace (16-byte aligned, device memory, no initialisation): tfserve_decode_paged_workspace bytes let
 * the step divide the rows of long sequences over several workgroups; fewer (or NULL) is correct but
 * slower, except that key_weights needs the whole of it (TFGFA_ERR_SCRATCH).  Calls sharing a workspace
 * must be ordered on one stream, and a call with key_weights, which may be two launches, must not have
 * another thread's between them.
 */
int tfserve_decode_paged(const void* q, const int64_t* q_strides,
                         void* k_pages, const int64_t* k_strides,
                         void* v_pages, const int64_t* v_strides,
                         const int* page_table, int64_t table_stride, const int* cache_seqlens,
                         const void* k_new, const int64_t* k_new_strides,
                         const void* v_new, const int64_t* v_new_strides,
                         void* o, const int64_t* o_strides, float* lse,
                         float* key_weights, const int64_t* weights_strides,
                         int B, int H, int H_kv, int P, int page, int M, int D, int dtype,
                         float softmax_scale, void* workspace, size_t workspace_bytes,
                         void* hip_stream);

/* Workspace bytes for the above (0 for sizes out of range); with_weights: 1 when key_weights is given. */
size_t tfserve_decode_paged_workspace(int B, int H, int H_kv, int page, int M, int D,
                                      int with_weights);

/*
 * The attention weight each key receives from given queries:
 *   out[b,h',j] = sum over the heads h of h', over the queries i that see key j, of
 *                 exp(scale * q[b,h,i,:] . k[b,h',j,:] - lse[b,h,i])
 * Query i sees key j when causal == 0, or j <= first_query + i.
 * q: (B, H, N_q, D), k: (B, H_kv, N_k, D), strides [b, h, n, d] as for tfgfa_fwd; lse: float32
 * (B, H, N_q), strides [b, h], last dimension dense, the log-sum-exp the attention returned; out: float32
 * (B, H_kv, N_k), strides [b, h], last dimension dense, written whole.  A query whose lse is -inf (or
 * past 2^127 in magnitude) adds nothing; hidden pairs add nothing whatever they hold.  The result does
 * not depend on the device's scheduling: sums are added in a fixed order.
 *
 * workspace (16-byte aligned, device memory, no initialisation): tfserve_key_weights_workspace bytes let the
 * queries of a block of keys be divided over several workgroups where there are few keys; fewer (or NULL) is
 * correct but slower.  Calls sharing a workspace must be ordered on one stream.
 */
int tfserve_key_weights(const void* q, const int64_t* q_strides, const void* k,
                        const int64_t* k_strides, const float* lse, const int64_t* lse_strides,
                        float* out, const int64_t* out_strides, int B, int H, int H_kv, int N_q,
                        int N_k, int D, int dtype, float softmax_scale, int causal,
                        int64_t first_query, void* workspace, size_t workspace_bytes, void* hip_stream);

/* Workspace bytes for the above (0 where nothing is divided, and for sizes out of range). */
size_t tfserve_key_weights_workspace(int B, int H, int H_kv, int N_q, int N_k, int causal);

/*
 * Eviction from a paged cache (laid out as above) by accumulated weight.  Of the L = cache_seqlens[b] rows
 * of each (sequence, key-value head) n = min(L, budget) are kept: the last min(L, recent), then those
 * of largest key_weights[b,h',j], ties to the lowest j, NaN below everything.  The kept rows, in their
 * order, are copied to rows 0 .. n - 1 of the pages in new_page_table (int32 (B, M_new), M_new * page >=
 * budget), and
 *   kept[b,h',i]        = the i-th kept row, -1 from n on       int32 (B, H_kv, budget) contiguous
 *   weights_out[b,h',i] = its key_weights, 0 from n on          float32, strides [b, h], i < budget
 * Pools whose strides put rows over one another are refused.
 * Table entries past a sequence's last row, old and new, are not read.  The pages of new_page_table must
 * be none that any row still reads, and each named once (the caller afterwards takes it for its
 * page_table and bounds cache_seqlens by budget); the old pages are left as they were.  weights_out may be key_weights
 * itself (same strides).
 * A row whose length does not fit (L < 0 or > M * page), or with a page id outside [0, P) among the
 * ones it needs, gets kept = -1 and weights_out = NaN, and nothing is copied for it.
 * recent in [0, budget].
 */
int tfserve_evict(void* k_pages, const int64_t* k_strides, void* v_pages, const int64_t* v_strides,
                  const int* page_table, int64_t table_stride, const int* cache_seqlens,
                  const float* key_weights, const int64_t* weights_strides,
                  const int* new_page_table, int64_t new_table_stride, int* kept,
                  float* weights_out, const int64_t* weights_out_strides, int B, int H_kv, int P,
                  int page, int M, int M_new, int D, int budget, int recent, void* hip_stream);

/* Element types of the logits. */
#define TFSERVE_LOGITS_BF16 0
#define TFSERVE_LOGITS_F16  1
#define TFSERVE_LOGITS_F32  2

/*
 * Penalties, biases and masks on logits (B, V), one rounding at the end:
 *   n   = how often v stands in tokens[b, 0 .. lengths[b])     (T without lengths; ids outside [0, V) count
 *                                                              for nothing; lengths are taken into [0, T])
 *   x   = logits[b,v];   n > 0:  x = (x > 0 ? x / repetition : x * repetition) - frequency * n - presence
 *   x  += bias[v]
 *   out = allowed bit ? x : -inf
 * logits, out: row strides, last dimension dense; out may be logits itself.  tokens: int32 or int64
 * (token_bytes 4 or 8), row stride, or NULL with T = 0.  Each of the three penalties is the scalar, or,
 * where its array is not NULL, a float32 value per row.  bias: float32, row stride (0: one for all
 * rows), or NULL.  allowed: int32 words, row stride (0: one for all), bit v % 32 of word v / 32, or NULL.
 */
int tfserve_penalize(const void* logits, int64_t logits_stride, void* out, int64_t out_stride,
                     int kind, const void* tokens, int token_bytes, int64_t tokens_stride,
                     const int* lengths, const float* repetitions, float repetition,
                     const float* presences, float presence, const float* frequencies,
                     float frequency, const float* bias, int64_t bias_stride, const int* allowed,
                     int64_t allowed_stride, int B, int V, int T, void* hip_stream);

#ifdef __cplusplus
}
#endif

#endif /* TFGFA_SERVING_H */
