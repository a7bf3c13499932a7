/*
 * zonos3_attn.h -- C ABI of the attention sublayer that stands between gated-delta-rule layers, on MI355X (gfx950): norms
 * and position rotation of queries and keys with the cache's write, and causal attention with a sliding window and first
 * tokens that stay visible (sinks), over whole sequences and one token at a time over a paged cache. In the library of
 * zonos3_gdn.h and by the same rules.
 *
 * Every entry point takes plain device pointers, sizes and a HIP stream (as void*, NULL = the default stream),
 * launches asynchronously on that stream, allocates nothing, never synchronises the host and can be captured into a
 * HIP graph. Return value and messages: zgdn_status and zgdn_last_error() of zonos3_gdn.h. dtype: ZGDN_F32 or ZGDN_BF16.
 *
 * Heads: query head h reads key head h / (Hq / Hk). Head sizes D: 64 or 128. A token's heads are contiguous; *_ld are the
 * elements between tokens (at least a token's, multiples of 16 bytes from 16-byte aligned bases, at most 2^22).
 * Workspaces start on 16-byte boundaries; the bytes that they need go by the CUs of the current device, so they are asked for
 * with the launch's device current. scale and its product with log2(e) are finite in float32.
 * Sums are formed in float32. A head whose squares sum to 2^128 or more comes out of its norm as zeros; values of 2^120 (for
 * zattn_window_step 2^128) over the number of a row's keys and more may become infinities.
 * A query at position p sees key j where j <= p and (p - j < window or j < sinks); window 0: no window. A row that sees
 * nothing is zeros. What a row does not see has no part in it, infinities and NaN included.
 */
#ifndef ZONOS3_ATTN_H
#define ZONOS3_ATTN_H

#include "zonos3_gdn.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * y = x * rsqrt(mean(x^2) + eps) * weight for each head of q and k, then the first R of its D entries turned by pairs:
 * (a, b) -> (a cos t - b sin t, b cos t + a sin t), t = position * inv_freq[i], i < R / 2. Pairs: entries i and i + R / 2, or
 * 2 i and 2 i + 1 where `interleaved`. All in float32 (t reduced in float64), rounded once.
 *   q [n_tokens, Hq, D], k [n_tokens, Hk, D], v [n_tokens, Hk, D] or NULL. positions: int64, or int32 where positions_i32.
 *   inv_freq [R / 2]: float64, or float32 where inv_freq_f32. R: a multiple of 16, at most D (0: nothing is turned).
 *   q_weight, k_weight [D] in w_dtype, or NULL (ones). q_out [n_tokens, Hq, D] dense. k_out [n_tokens, Hk, D] dense, or NULL.
 *   k_cache, v_cache with `rows` (int64 [n_tokens]), or all NULL: token t's k (turned) and v go to rows[t] of the
 *   n_cache_rows rows, kc_ld and vc_ld elements apart; a row outside the cache is not written. k_cache alone: v is NULL.
 *   (A cache of no rows may be NULL.)
 *   Where two tokens name one row, it holds pieces of either. Outputs overlap no other operand.
 */
int zattn_qk_norm_rope(const void* q, long q_ld, const void* k, long k_ld, const void* v, long v_ld, int dtype,
                       const void* positions, int positions_i32, const void* inv_freq, int inv_freq_f32,
                       const void* q_weight, const void* k_weight, int w_dtype, float eps, int interleaved, void* q_out,
                       void* k_out, void* k_cache, long kc_ld, void* v_cache, long vc_ld, const int64_t* rows,
                       long n_cache_rows, int n_tokens, int Hq, int Hk, int D, int R, void* stream);

/*
 * Bytes of workspace that zattn_window_fwd needs for the same sizes (0 for sizes that it refuses, and where it needs none).
 * packed: 1 where cu_q and cu_k are given (n_seqs sequences in Tq and Tk rows), else 0 (n_seqs = B).
 */
size_t zattn_window_fwd_workspace_bytes(int packed, int n_seqs, int Tq, int Tk, int Hq, int Hk, int D, int window, int sinks,
                                        int dtype);

/*
 * Attention over whole sequences: o_i = sum_j softmax_j(scale q_i . k_j) v_j over the keys that i sees.
 *   q, o [B, Tq, Hq, D], k, v [B, Tk, Hk, D] in `dtype`; o is dense. Query i of a sequence of nq queries and nk keys stands at
 *   position nk - nq + i (negative: it sees nothing).
 *   cu_q, cu_k: int32 [n_seqs + 1] with B == 1, or both NULL (n_seqs is not read). Rows that belong to no sequence are left as
 *   they were. Bounds are clamped to the rows and to the bound before; where sequences overlap even so, what their rows get is
 *   not specified, and nothing else is written. o and the workspace overlap no other operand.
 */
int zattn_window_fwd(const void* q, long q_ld, const void* k, long k_ld, const void* v, long v_ld, int dtype, void* o,
                     const int32_t* cu_q, const int32_t* cu_k, int n_seqs, int B, int Tq, int Tk, int Hq, int Hk, int D,
                     int window, int sinks, float scale, void* workspace, size_t workspace_bytes, void* stream);

/*
 * Bytes of workspace that zattn_window_step needs for the same sizes (0 for sizes that it refuses, and where it needs none).
 * room: the positions that a stream can have, page_size * n_pages.
 */
size_t zattn_window_step_workspace_bytes(int B, long room, int Hq, int Hk, int D, int window, int sinks, int dtype);

/*
 * One query for each of B streams, at the last of its lengths[b] positions, over a cache.
 *   q, o [B, Hq, D] in `dtype`, o dense. k_cache, v_cache: n_rows rows [Hk, D] of `dtype`, kc_ld and vc_ld elements apart.
 *   Position p of stream b is row pages[b * n_pages + p / page_size] * page_size + p % page_size (page_size a power of two),
 *   or, where pages is NULL, row b * page_size + p (n_pages == 1). Positions on a page that is not in the cache are not seen.
 *   lengths: int32 [B], clamped to 0 .. room.
 *   o and the workspace overlap no other operand.
 */
int zattn_window_step(const void* q, long q_ld, const void* k_cache, long kc_ld, const void* v_cache, long vc_ld, int dtype,
                      const int32_t* lengths, const int32_t* pages, int page_size, int n_pages, long n_rows, void* o, int B,
                      int Hq, int Hk, int D, int window, int sinks, float scale, void* workspace, size_t workspace_bytes,
                      void* stream);

#ifdef __cplusplus
}
#endif

#endif /* ZONOS3_ATTN_H */
