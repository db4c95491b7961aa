/*
 * tfgfa_pages.h - C ABI of the operators around a paged key-value cache (MI355X, gfx950): rotary positions, new
 * tokens' keys and values into the pages, attention of several new tokens over them, and a decode step for
 * sequences that share a prefix.
 *
 * The reference's model has learned positions and keeps no cache (src/py/model_inference.py:166-228); there is
 * nothing of this in it.
 *
 * Conventions and paged caches as in tfgfa_serving.h: device pointers, the caller owns every buffer, launches are
 * asynchronous on `hip_stream`, arguments are checked before any HIP call; 0 on success, > 0 an invalid argument
 * (TFGFA_ERR_*), < 0 a negated hipError_t.  Strides are in elements.
 */
#ifndef TFGFA_PAGES_H
#define TFGFA_PAGES_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of tfpages_rotate: TFGFA_DTYPE_BF16, TFGFA_DTYPE_F16 and this one. */
#define TFPAGES_DTYPE_F32 2

/*
 * Rotary positions.  Of each head vector x the first `rot` dims (even, at most D) are rotated in pairs (a, b), the
 * others copied:
 *   y_a = m (x_a cos t - x_b sin t),  y_b = m (x_b cos t + x_a sin t),  t = 2 pi position turns_i / 2^64
 * Pair i is (i, i + rot / 2), or with interleaved (2i, 2i + 1).  turns: rot / 2 uint64 in device memory, turns of a
 * position in 2^-64 (position * turns_i is exact modulo a turn, so far positions keep their angles).  transposed: -t
 * for t, which turns the gradient of y into that of x.
 * q, q_out: (B, H, N, D), k, k_out: (B, H_kv, N, D) or all NULL with H_kv 0; strides [b, h, n, d], last dimension
 * dense, the others not negative; what is written must not overlap.  q_out may be q itself with its strides, and k_out
 * k.  positions: int32 or int64 (position_bytes 4 or 8), element [b, n] at b * position_strides[0] + n *
 * position_strides[1]; or NULL: first + n.  D at most 128, B * N at most 2^27 (TFGFA_ERR_TOO_LARGE).
 */
int tfpages_rotate(const void* q, const int64_t* q_strides, void* q_out, const int64_t* q_out_strides, int H,
                   const void* k, const int64_t* k_strides, void* k_out, const int64_t* k_out_strides, int H_kv,
                   const void* positions, int position_bytes, const int64_t* position_strides, int64_t first,
                   const uint64_t* turns, int rot, int interleaved, float magnitude, int transposed, int B, int N,
                   int D, int dtype, void* hip_stream);

/*
 * New tokens into a paged cache (laid out as for tfserve_decode_paged, rows in places of their own): with n_b =
 * lengths[b] (N without lengths), token i < n_b of k and v (B, H_kv, N, D) becomes row cache_seqlens[b] + i of
 * sequence b.  The caller advances cache_seqlens afterwards, and gives no two sequences one page for new rows.
 * With turns (rot > 0) k is rotated on the way as by tfpages_rotate, token i at position positions[b] + i (int32 (B,);
 * cache_seqlens[b] + i without); and so is q (B, H, N, D) into q_out, if given (q_out may be q with its strides).
 * Tokens past n_b: their rows of q_out become zeros with pad != 0, and are left as they were otherwise.
 * Visible on the device only: where cache_seqlens[b] < 0, n_b is not in [0, N] or their sum is past M * page, nothing
 * is written to the cache for the sequence and its rows of q_out are NaN; a page id outside [0, P) gets no row.
 * dtype: TFGFA_DTYPE_BF16 or TFGFA_DTYPE_F16; D a multiple of 8 up to 128; strides of k, v, q and q_out as for
 * tfserve_key_weights (multiples of 8, rows apart), pointers to 16 bytes; B * N at most 2^27.
 */
int tfpages_append(const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides, void* k_pages,
                   const int64_t* k_pages_strides, void* v_pages, const int64_t* v_pages_strides,
                   const int* page_table, int64_t table_stride, const int* cache_seqlens, const int* lengths,
                   const int* positions, const void* q, const int64_t* q_strides, void* q_out,
                   const int64_t* q_out_strides, int pad, const uint64_t* turns, int rot, int interleaved,
                   float magnitude, int B, int H, int H_kv, int N, int P, int page, int M, int D, int dtype,
                   void* hip_stream);

/*
 * Attention of N new tokens over a paged cache that holds their keys already:
 *   O[b,h,i,:] = sum_{j < L_bi} softmax_j(scale * q[b,h,i,:] . K[b,h',j,:]) * V[b,h',j,:],   LSE likewise
 * with h' = h / (H / H_kv) and L_bi = cache_seqlens[b] + i + 1 (causal: the rows before the tokens, and the tokens up
 * to this one) or cache_seqlens[b] (not causal: all rows).  cache_seqlens counts the rows before the new tokens when
 * causal, and all rows when not.  Tokens i >= n_b = lengths[b] (N without lengths) have no output: their rows of o
 * and lse become 0 and -inf with pad != 0, and are left as they were otherwise.
 * q, o: (B, H, N, D), strides [b, h, n, d] (multiples of 8, rows apart); lse: (B, H, N) contiguous or NULL.
 * softmax_scale: positive, log2(e) times it finite.
 * A row whose scores are all -inf, or that sees no key, gives O = 0 and LSE = -inf.  Hidden rows and rows past the
 * cache's never reach a result.  Visible on the device only: where cache_seqlens[b] < 0, n_b is not in [0, N] or the
 * rows do not fit M * page, O and LSE of the sequence's N tokens are NaN; a page id outside [0, P) among the rows that a
 * token sees gives it NaN.
 * Weights are rounded to the element type for the product with V where there are more than 64 query rows (tokens x H /
 * H_kv), as tfgfa_fwd does, and divided by the sum of the rounded ones; with fewer they go through the product in two parts
 * (all but 2^-16 of a weight in bf16, 2^-22 in fp16).  LSE takes the unrounded ones.
 * workspace (16-byte aligned, device memory, no initialisation): tfpages_attend_workspace bytes let the rows of long
 * caches be divided over several workgroups; fewer (or NULL) is correct but slower.  Calls sharing a workspace must be
 * ordered on one stream, without another thread's call between the launches of one.
 */
int tfpages_attend(const void* q, const int64_t* q_strides, const void* k_pages, const int64_t* k_strides,
                   const void* v_pages, const int64_t* v_strides, const int* page_table, int64_t table_stride,
                   const int* cache_seqlens, const int* lengths, void* o, const int64_t* o_strides, float* lse,
                   int pad, int causal, int B, int H, int H_kv, int N, int P, int page, int M, int D, int dtype,
                   float softmax_scale, void* workspace, size_t workspace_bytes, void* hip_stream);

/* Workspace bytes for the above (0 where nothing is divided, and for sizes out of range). */
size_t tfpages_attend_workspace(int B, int H, int H_kv, int N, int page, int M, int D);

/*
 * One decode step of B sequences in R groups of B / R (sequence b in group b / (B / R)) that share their first rows:
 * sequence b attends to the prefix_lens[r] rows of its group's prefix, whose pages prefix_table (int32 (R, M_prefix))
 * names, and then to its own cache_seqlens[b] (+1 when appending) rows of page_table (int32 (B, M)); the prefix's rows
 * are read once for the group.  The pools, k_new and v_new (row cache_seqlens[b] of the sequence's own), o, lse and
 * empty rows are as for tfserve_decode_paged.  B is a multiple of R.
 * Visible on the device only: a length that does not fit, or a page id outside [0, P) among the rows, gives NaN to
 * the sequence, or to the whole group if it is the prefix's.
 * Weights of a prefix are rounded to the element type for the product with V, as tfpages_attend does, where a group has
 * more than 64 query rows (B / R x H / H_kv).
 * workspace (16-byte aligned, device memory, no initialisation): tfpages_decode_shared_workspace bytes, which the call
 * needs (TFGFA_ERR_SCRATCH otherwise).  Calls sharing a workspace must be ordered on one stream, without another
 * thread's call between the launches of one.
 */
int tfpages_decode_shared(const void* q, const int64_t* q_strides, void* k_pages, const int64_t* k_strides,
                          void* v_pages, const int64_t* v_strides, const int* prefix_table, int64_t prefix_stride,
                          const int* prefix_lens, const int* page_table, int64_t table_stride,
                          const int* cache_seqlens, const void* k_new, const int64_t* k_new_strides,
                          const void* v_new, const int64_t* v_new_strides, void* o, const int64_t* o_strides,
                          float* lse, int R, int B, int H, int H_kv, int P, int page, int M_prefix, int M, int D,
                          int dtype, float softmax_scale, void* workspace, size_t workspace_bytes, void* hip_stream);

/* Workspace bytes for the above (0 for sizes out of range). */
size_t tfpages_decode_shared_workspace(int R, int B, int H, int H_kv, int page, int M_prefix, int M, int D);

#ifdef __cplusplus
}
#endif

#endif /* TFGFA_PAGES_H */
