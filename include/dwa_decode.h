/*
 * dwa_decode.h — the serving operators of this library's DWA language model:
 * a paged key/value cache (written, read back, attended to) and the
 * verification of drafted tokens, in chains or trees.  Same conventions as dwa_retrieval.h:
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
 * aligned (ld_page a multiple of d, ld_scale_page of 4).  Codes are numbers, scales finite or NaN
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

/*
 * Writes T tokens' keys and values into the cache as dwa_kv_write does, the keys rotated
 * for their positions, and their queries' rotation into q_out (bf16 [T][H][d] contiguous;
 * q NULL: no queries, H and q_out are not looked at).  For a vector x with x1 = x[0::2], x2 = x[1::2]
 * and row p = positions[t] (int64; NULL: t) of cos and sin ([n_positions][ld_table], d / 2
 * used; both bf16 when tables_bf16 else f32)
 *   [x1 cos - x2 sin, x1 sin + x2 cos].
 * With bf16 q, k, v (src_bf16) and bf16 tables every product, sum and difference is rounded to bf16,
 * as dwa_lm_rope_qk does; otherwise they are f32, and the result is rounded once where it is
 * stored (an e4m3 key from its f32 values).  A position outside the tables makes its
 * token's query and keys NaN (its values stay) and is reported in *status.
 * Tables' rows 16-byte aligned; everything else as dwa_kv_write wants it.
 */
DWA_API dwa_status dwa_kv_append(const void* q, const void* k, const void* v, int32_t src_bf16, int64_t T,
                                 int32_t H, int32_t H_kv, int32_t d, int64_t q_ld_tok, int64_t q_ld_head,
                                 int64_t k_ld_tok, int64_t k_ld_head, int64_t v_ld_tok, int64_t v_ld_head,
                                 const void* cos_t, const void* sin_t, int32_t tables_bf16, int64_t ld_table,
                                 int64_t n_positions, const int64_t* positions, const int64_t* slots,
                                 void* k_cache, void* v_cache, float* k_scale, float* v_scale,
                                 int64_t n_pages, int32_t page_size, int64_t ld_page, int64_t ld_scale_page,
                                 void* q_out, int32_t* status, dwa_stream_t stream);

/*
 * Trees of drafted tokens.  Sequence b's tree is its new tokens, rows q_start[b] ..
 * q_start[b + 1] - 1 of T packed ones (q_start NULL: T / B each): nodes 0, 1, ..., parents before
 * children, parents[row] a node's parent's number (-1: none).
 *
 * dwa_tree_masks: mask (uint64 [T][mask_words]) gets in every node's row its own bit and its
 * ancestors' (node j: bit j % 64 of word j / 64), depth (int32 [T]) the number of its ancestors.
 * max_q (4096 at most) bounds the nodes of a tree; mask_words >= max_q / 64.  A node whose parent
 * is not before it counts as one without a parent and is reported in *status; a tree of more than max_q
 * nodes is reported and its rows are zeros, as rows of no sequence are (those too that only a bad
 * range covers).
 */
DWA_API dwa_status dwa_tree_masks(const int32_t* parents, const int32_t* q_start, int64_t T, int32_t B,
                                  int32_t max_q, int64_t* mask, int32_t mask_words, int32_t* depth,
                                  int32_t* status, dwa_stream_t stream);

/*
 * dwa_paged_attention for new tokens that are a tree's nodes: node i of n attends to the first
 * length - n tokens, and to node j (token length - n + j) where bit j of its row of tree_mask
 * (uint64 [T][mask_words], 8-byte aligned) is set.  Any bits may be; those from n on count for nothing.
 * max_q is 64 mask_words at most.  All else as there, but the rounding of 17 to 32 rows per
 * key/value head, and of up to 64 over narrow tables: bf16 caches none (p_j as
 * the sum of two bf16), e4m3 caches p_j times its value's scale to 11 bits, and q to 2^-18 of its
 * row's largest value.  workspace: 16-byte aligned, of
 * dwa_paged_tree_attention_workspace bytes (0: none) for the current device; it holds nothing between calls.
 */
DWA_API dwa_status dwa_paged_tree_attention(const void* q, int64_t T, int32_t H, int32_t d, int64_t q_ld,
                                            const void* k_cache, const void* v_cache,
                                            const float* k_scale, const float* v_scale, int32_t H_kv,
                                            int64_t n_pages, int32_t page_size, int64_t ld_page,
                                            int64_t ld_scale_page, const int32_t* block_table,
                                            int64_t ld_table, int32_t max_pages, const int32_t* lengths,
                                            const int32_t* q_start, int32_t B, int32_t max_q,
                                            const int64_t* tree_mask, int32_t mask_words, float scale,
                                            void* out, int64_t out_ld, void* workspace,
                                            size_t workspace_bytes, int32_t* status, dwa_stream_t stream);
DWA_API size_t dwa_paged_tree_attention_workspace(int32_t H, int32_t d, int32_t H_kv, int32_t page_size,
                                                  int32_t max_pages, int32_t B, int32_t max_q);

/*
 * The walk through a verified tree: target [T][V] (f32, or bf16 when probs_bf16) holds the
 * target's probabilities behind every node, tokens int32 [T] the nodes' tokens (node 0's is not
 * looked at), sample_u f32 [B][steps] uniform numbers in [0, 1).  From node 0 on, step s draws the lowest
 * index whose running sum of the node's row exceeds sample_u[b][s] times the row's sum (64-bit sums;
 * entries that are not positive finite numbers count as 0).  Where a child of the node has that
 * token the walk goes on there (the first such child), as long as s + 1 < steps; else it ends.
 * n_accepted int32 [B]: the drafts passed; out_tokens int32 [B][steps]: the drawn tokens (the
 * last is no draft; -1 where a row sums to nothing), then -1; path int32 [B][steps]: the nodes that
 * were drawn from, 0 first, then -1.  A sequence without nodes has 0 and all -1.
 */
DWA_API dwa_status dwa_verify_tree(const void* target, int32_t probs_bf16, const int32_t* tokens,
                                   const int32_t* parents, const int32_t* q_start, const float* sample_u,
                                   int64_t T, int32_t B, int32_t steps, int32_t V, int32_t* n_accepted,
                                   int32_t* out_tokens, int32_t* path, dwa_stream_t stream);

/*
 * Moves the cached tokens of a path to where a sequence's tokens belong, in `layers` layers
 * (ld_layer elements and ld_scale_layer scales apart): sequence b's token start[b] + path[b][i] to
 * start[b] + i, for i = 0 .. n_accepted[b] (int32; path int32 [B][steps]), on the pages of
 * block_table.  Paths ascend from 0 or more, so every token moves as it was before the call.  n_accepted below
 * 0, or 0 with a negative path[b][0]: nothing.  A path that does not ascend, is longer than
 * steps, or leaves the pages is reported in *status, and its sequence stays as it was.
 */
DWA_API dwa_status dwa_kv_keep(void* k_cache, void* v_cache, float* k_scale, float* v_scale,
                               int32_t layers, int64_t ld_layer, int64_t ld_scale_layer, int32_t H,
                               int32_t d, int64_t n_pages, int32_t page_size, int64_t ld_page,
                               int64_t ld_scale_page, const int32_t* block_table, int64_t ld_table,
                               int32_t max_pages, const int32_t* start, const int32_t* path,
                               const int32_t* n_accepted, int32_t B, int32_t steps, int32_t* status,
                               dwa_stream_t stream);

#ifdef __cplusplus
}  /* extern "C" */
#endif

#endif /* DWA_DECODE_H_ */
