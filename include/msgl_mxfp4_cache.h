/*
 * msgl_mxfp4_cache.h -- a K/V pool held in 4 bits: what writes it, what reads it back and what attends over it.
 *
 * The pool of msgl_paged_attention.h with 4.25 bits to a value in place of 16.  Per layer two arrays:
 *   kv_codes  (num_slots, num_kv_heads, 2, head_dim / 2)   bytes: K's codes, then V's
 *   kv_scales (num_slots, num_kv_heads, 2, head_dim / 32)  bytes: one to each block of 32 dims
 * A code is a 4-bit float (0, 0.5, 1, 1.5, 2, 3, 4, 6; bit 3 is the sign), dim 2i in the low half of byte i; a block byte b
 * stands for the factor 2^(b - 127).  The writers choose the smallest b with which no value of the block lies beyond 6,
 * held to [2, 252], and round to the nearest code, halfway to the even one.  A row whose K or V of a head has a NaN or an infinity
 * leaves 255 in that head's block bytes of K and zeros in its codes of K and V: the key's score is then NaN for whoever sees it, and
 * nothing for whom the mask hides it from.  (V's block bytes are never 255.)
 *
 * The reference has no such pool; the conventions are those of msgl_paged_attention.h: device pointers, nothing
 * allocated, retained or synchronised, errors as MSGL_ERR_* codes, slot ids outside the pool written nowhere by the writers and
 * clamped to the pool by the readers.  `codes_stride0` and `scales_stride0` are the BYTES from one slot to the next (the rest is
 * contiguous): multiples of 16 and of 8, below 2^32 (MSGL_ERR_SHAPE).  head_dim is 128 or 256.
 */
#ifndef MSGL_MXFP4_CACHE_H
#define MSGL_MXFP4_CACHE_H

#include "msgl_paged_attention.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Rows r of k and v (length, num_kv_heads, head_dim), bf16 or half by `dtype`, leading strides free, into slots indices[r], which are
 * distinct: the counterpart of msgl_store_kv_cache. */
MSGL_API int msgl_store_kv_cache_mxfp4(void* kv_codes, void* kv_scales, const int32_t* indices, const void* k, const void* v,
                                       int64_t length, int64_t num_kv_heads, int64_t head_dim, int64_t num_slots,
                                       int64_t codes_stride0, int64_t scales_stride0, int64_t k_stride0, int64_t v_stride0,
                                       int32_t dtype, void* stream);

/* What slots indices[r] hold, as contiguous rows of k and v.  Exact in bf16; in half what it cannot hold is rounded. */
MSGL_API int msgl_load_kv_cache_mxfp4(const void* kv_codes, const void* kv_scales, const int32_t* indices, void* k, void* v,
                                      int64_t length, int64_t num_kv_heads, int64_t head_dim, int64_t num_slots,
                                      int64_t codes_stride0, int64_t scales_stride0, int32_t dtype, void* stream);

/* Per-head RMS norm of q and k, rotary embedding of both, and the store of k and v, with q as q_out (n_tokens, num_q_heads, head_dim):
 * the counterpart of msgl_qk_norm_rope_store (bf16).  Between the inputs and q_out, or the codes of k, nothing is rounded to
 * bf16, and angles are those of 64 bits. */
MSGL_API int msgl_qk_norm_rope_store_mxfp4(const void* q, const void* k, const void* v, int64_t q_stride0, int64_t k_stride0,
                                           int64_t v_stride0, const void* q_weight, const void* k_weight,
                                           const int32_t* positions, const int32_t* out_loc, void* q_out, void* kv_codes,
                                           void* kv_scales, int64_t codes_stride0, int64_t scales_stride0, int64_t num_slots,
                                           int64_t n_tokens, int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim,
                                           double rms_norm_eps, double rope_base, int32_t dtype, void* stream);

/* One query per request over the slots listed for it: the counterpart of msgl_paged_decode_attention.  q and out
 * (batch, num_q_heads, head_dim) contiguous, bf16 or half; at most 16 q heads to a kv head.  A request without keys gets zeros.
 * With q in bf16 the pool's values are taken exactly.  Half takes them at half their size: those of blocks whose factor is below 2^-22 are off
 * by 2^-24 at most, and values beyond 98304 are infinities.
 * total_kv is the length of kv_indices, at least kv_indptr[batch].  Both kinds of attention take total_kv up to 2^30 and up to 2^15 kv heads. */
MSGL_API size_t msgl_paged_decode_mxfp4_workspace_bytes(int64_t batch, int64_t total_kv, int64_t num_q_heads,
                                                        int64_t num_kv_heads, int64_t head_dim);
MSGL_API int msgl_paged_decode_attention_mxfp4(const void* q, const void* kv_codes, const void* kv_scales,
                                               const int32_t* kv_indptr, const int32_t* kv_indices, void* out, void* workspace,
                                               size_t workspace_bytes, int64_t batch, int64_t total_kv, int64_t num_q_heads,
                                               int64_t num_kv_heads, int64_t head_dim, int64_t num_slots, int64_t codes_stride0,
                                               int64_t scales_stride0, float sm_scale, int32_t dtype, void* stream);

/* Several queries per request under the four masks of msgl_paged_prefill_attention, which this is the counterpart of (bf16).
 * Short query blocks read the pool as it is.  Longer ones have the listed rows unpacked into the workspace first, once for all their
 * queries (total_kv rows of K and V in bf16 at most; total_kv * num_kv_heads below 2^31), and go through the tile kernels of the 16-bit pool. */
MSGL_API size_t msgl_paged_prefill_mxfp4_workspace_bytes(int64_t batch, int64_t total_q, int64_t total_kv, int64_t num_q_heads,
                                                         int64_t num_kv_heads, int64_t head_dim, int64_t max_len_extend);
MSGL_API int msgl_paged_prefill_attention_mxfp4(const void* q, const void* kv_codes, const void* kv_scales,
                                                const int32_t* qo_indptr, const int32_t* kv_indptr, const int32_t* kv_indices,
                                                const int32_t* prefix_lens, void* out, void* workspace, size_t workspace_bytes,
                                                int64_t batch, int64_t total_q, int64_t total_kv, int64_t num_q_heads,
                                                int64_t num_kv_heads, int64_t head_dim, int64_t num_slots,
                                                int64_t codes_stride0, int64_t scales_stride0, float sm_scale,
                                                int32_t max_len_extend, int32_t is_cross_attention,
                                                int32_t sliding_window_size, int32_t dtype, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MSGL_MXFP4_CACHE_H */
