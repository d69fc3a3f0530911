/*
 * dwa_decode.h — the serving operators of this library's DWA language model:
 * a paged key/value cache (written, read back, attended to) and the
 * verification of drafted tokens.  Same conventions as dwa_retrieval.h:
 * stream-ordered and asynchronous, arguments validated on the host (non-zero
 * status, nothing launched, when invalid), no allocation, bf16 buffers as
 * uint16 bit patterns, e4m3 buffers as bytes.
 *
 * The cache holds n_pages pages of page_size tokens, head-major:
 *   k_cache, v_cache [n_pages][H][page_size][d]   bf16, or e4m3 with
 *   k_scale, v_scale [n_pages][H][page_size]      one f32 scale per vector.
 * Pages may lie ld_page elements (scales: ld_scale_page) apart; everything
 * inside a page is contiguous.  Slot s is token s % page_size of page
 * s / page_size.  page_size is 16, 32, 64 or 128; d is a multiple of 16 in
 * [16, 128].  NULL scales mean a bf16 cache.  Pages and their scales are 16-byte
 * aligned (ld_page a multiple of d, ld_scale_page of 4).  Codes are numbers
 * (dwa_kv_write makes no NaN code: what it cannot store has a NaN scale).
 *
 * What only the device can see is checked there: a bad slot, page number,
 * length or row range never leads to an access; it writes DWA_ERR_DEVICE_CHECK
 * to *status (device int32, may be NULL) and NaN to the rows concerned.  (A row
 * range that is none, descending or outside q, says of no row whose it is: rows that
 * no other sequence has stay as they were.)
 */
#ifndef DWA_DECODE_H_
#define DWA_DECODE_H_

#include "dwa_retrieval.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Writes T tokens' keys and values into the cache: token t's head h,
 * k + t ld_tok + h ld_head (elements; k and v bf16 when src_bf16 else f32),
 * goes to slot slots[t].  An e4m3 cache stores
 *   scale = max(amax / 448, 2^-126),  code = e4m3(x / scale)
 * (f32 divisions, round to nearest even); a vector with a value that is not
 * finite gets the scale NaN and zero codes, so that it reads back as NaN.
 * Slot -1 skips the token; where slots repeat, the last token stays; any other
 * slot outside [0, n_pages page_size) is skipped and reported in *status.
 * Rows 16-byte aligned: every stride times the element size a multiple of 16.
 */
DWA_API dwa_status dwa_kv_write(const void* k, const void* v, int32_t src_bf16, int64_t T, int32_t H,
                                int32_t d, int64_t k_ld_tok, int64_t k_ld_head, int64_t v_ld_tok,
                                int64_t v_ld_head, const int64_t* slots, void* k_cache,
                                void* v_cache, float* k_scale, float* v_scale, int64_t n_pages,
                                int32_t page_size, int64_t ld_page, int64_t ld_scale_page,
                                int32_t* status, dwa_stream_t stream);

/*
 * Reads T tokens back: k_out, v_out bf16 [T][H][d] contiguous, code * scale
 * rounded once (f32 product).  Slot -1 leaves the token's rows as they were, or
 * with clear_skipped zeroes them; any other slot outside the cache gives NaN and
 * is reported in *status.
 */
DWA_API dwa_status dwa_kv_read(const void* k_cache, const void* v_cache, const float* k_scale,
                               const float* v_scale, const int64_t* slots, int64_t T, int32_t H,
                               int32_t d, int64_t n_pages, int32_t page_size, int64_t ld_page,
                               int64_t ld_scale_page, void* k_out, void* v_out,
                               int32_t clear_skipped, int32_t* status, dwa_stream_t stream);

/*
 * Attention of every sequence's newest tokens over its pages.  Sequence b has
 * lengths[b] cached tokens (the new ones written already) on the pages
 * block_table[b ld_table + i] (int32, i < ceil(length / page_size)), and its
 * new tokens are rows q_start[b] .. q_start[b + 1] - 1 of q (q_start NULL: T / B
 * rows each, which B has to divide).  For new token i of n and query head h,
 *   out = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q . k_j - max),
 *   j < length - n + i + 1,
 * with the key and value head h / (H / H_kv); no key, or no score above -inf,
 * gives zeros.  q, out bf16 [T][H][d] with row strides q_ld / out_ld (elements;
 * heads contiguous).  Rows of no sequence are left as they were.  max_q
 * bounds every sequence's new tokens; a sequence may have 2^30 tokens.  Keys that
 * a row may not see do not reach it, whatever their bits and sizes.  A new token's
 * value that is not finite makes the rows that do see it not finite in its channel (an
 * infinity may become NaN).
 * Rounding, beside f32 sums and the result's: up to 16 rows per key/value head
 * (max_q H / H_kv), bf16 caches none (p_j as the sum of two bf16), e4m3 caches p_j
 * times its value's scale to 11 bits; more rows, bf16 caches p_j to 8 bits, e4m3
 * caches p_j, k_j and v_j to 11 bits each.  (What p_j times its value's scale is below
 * 2^-20 of the row's largest has fewer bits, below 2^-31 none.)
 */
DWA_API dwa_status dwa_paged_attention(const void* q, int64_t T, int32_t H, int32_t d, int64_t q_ld,
                                       const void* k_cache, const void* v_cache,
                                       const float* k_scale, const float* v_scale, int32_t H_kv,
                                       int64_t n_pages, int32_t page_size, int64_t ld_page,
                                       int64_t ld_scale_page, const int32_t* block_table,
                                       int64_t ld_table, int32_t max_pages, const int32_t* lengths,
                                       const int32_t* q_start, int32_t B, int32_t max_q, float scale,
                                       void* out, int64_t out_ld, int32_t* status,
                                       dwa_stream_t stream);

/*
 * Verification of drafted tokens (probabilities f32, or bf16 when probs_bf16):
 * target [B][K + 1][V], draft [B][K][V] (NULL: the drafter was certain, q = 1
 * at its token), tokens int32 [B][K], accept_u f32 [B][K] and sample_u f32 [B]
 * uniform in [0, 1).  Draft i of sequence b stands while
 *   accept_u q_i(x_i) < p_i(x_i)  and  i < draft_lengths[b]  (NULL: K),
 * products and sums in 64 bits.  With n standing drafts the next token is the
 * lowest index whose running sum of w exceeds sample_u times the sum of w:
 * w = max(p_n - q_n, 0) where draft n fell, p_n where none did or where that
 * leaves nothing.  Entries that are not positive finite numbers count as 0, so
 * a drafted token outside the vocabulary falls.  n_accepted int32 [B];
 * out_tokens int32 [B][K + 1]: the standing drafts, the next token (-1 where p_n
 * sums to nothing), then -1.
 */
DWA_API dwa_status dwa_verify_drafts(const void* target, const void* draft, int32_t probs_bf16,
                                     const int32_t* tokens, const float* accept_u,
                                     const float* sample_u, const int32_t* draft_lengths, int64_t B,
                                     int32_t K, int32_t V, int32_t* n_accepted, int32_t* out_tokens,
                                     dwa_stream_t stream);

#ifdef __cplusplus
}  /* extern "C" */
#endif

#endif /* DWA_DECODE_H_ */
