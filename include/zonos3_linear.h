/*
 * zonos3_linear.h -- C ABI of linear attention with a decay per head and of the projections around it, on MI355X
 * (gfx950): the operators next to the gated delta rule's (zonos3_gdn.h), in the same library and by the same rules.
 *
 * Every entry point takes plain device pointers, sizes and a HIP stream (as void*, NULL = the default stream),
 * launches asynchronously on that stream, allocates nothing, never synchronises the host and can be captured into a
 * HIP graph. Return value and messages: zgdn_status and zgdn_last_error() of zonos3_gdn.h.
 *
 * The recurrence, for each sequence and value head, over the state S [V, K] (float32, value-major):
 *   S_t = exp(g_t) S_{t-1} + v_t k_t^T,   o_t = S_t (scale q_t)
 * Value head h reads key head h / (Hv / Hk). g is a log decay; -inf (exp = 0) forgets all that was before, but for what is
 * not finite: infinities and NaN leave an infinity or a NaN in every output and state that depends on them, and in no other.
 */
#ifndef ZONOS3_LINEAR_H
#define ZONOS3_LINEAR_H

#include "zonos3_gdn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* What the epilogue of zlin_gemm_act applies to x w^T + bias. */
enum zlin_act { ZLIN_NONE = 0, ZLIN_RELU = 1, ZLIN_SILU = 2, ZLIN_GELU = 3 /* erf */, ZLIN_GELU_TANH = 4 };

/*
 * Bytes of workspace that zlin_attn_fwd needs for the same sizes (0 for sizes that it refuses). packed: 1 where
 * cu_seqlens is given (n_seqs sequences in T rows), else 0 (n_seqs = B batches of T rows).
 */
size_t zlin_attn_workspace_bytes(int packed, int n_seqs, int T, int Hk, int Hv, int K, int V, int dtype);

/*
 * Linear attention over whole sequences (chunked).
 *   q, k [B, T, Hk, K], v [B, T, Hv, V], o [B, T, Hv, V] in `dtype` (F32 or BF16); K and V each 64 or 128. A token's
 *   heads are contiguous; q_ld, k_ld, v_ld are the elements between tokens (multiples of 16 bytes, from 16-byte
 *   aligned bases; at most 2^22). o is dense.
 *   g: g_ld == 0: float32 [Hv], one log decay a head. Else [B, T, Hv] in g_dtype, g_ld elements between tokens.
 *   initial_state [N, Hv, V, K] float32 or NULL (zeros); final_state likewise or NULL (not written). final_state may
 *   be initial_state itself (in place). Otherwise o, final_state and the workspace may overlap no operand.
 *   cu_seqlens: int32 [n_seqs + 1] with B == 1, or NULL. Rows that belong to no sequence are left as they were. Bounds are
 *   clamped to the rows 0 .. T and to the bound before; where sequences overlap even so (a table that decreases), what
 *   their rows and states get is not specified, and nothing else is written.
 */
int zlin_attn_fwd(const void* q, long q_ld, const void* k, long k_ld, const void* v, long v_ld, int dtype,
                  const void* g, long g_ld, int g_dtype, const float* initial_state, float* final_state, void* o,
                  const int32_t* cu_seqlens, int n_seqs, int B, int T, int Hk, int Hv, int K, int V, float scale,
                  void* workspace, size_t workspace_bytes, void* stream);

/*
 * One token for each of B streams, in place on their states.
 *   q, k [B, Hk, K], v [B, Hv, V], o [B, Hv, V] in `dtype`; strides, K and V as above. g: g_ld == 0: float32 [Hv]; else
 *   [B, Hv] in g_dtype, g_ld elements between streams.
 *   state [n_slots, Hv, V, K] float32. slots: NULL (stream b's state is row b; n_slots == B), or int64 [B]. A stream
 *   whose slot lies outside the table, or that an earlier stream of the call has, gets zeros in o and touches no state.
 *   o and state may overlap no other operand.
 */
int zlin_attn_step(const void* q, long q_ld, const void* k, long k_ld, const void* v, long v_ld, int dtype,
                   const void* g, long g_ld, int g_dtype, float* state, const int64_t* slots, int n_slots, void* o,
                   int B, int Hk, int Hv, int K, int V, float scale, void* stream);

/*
 * y = act(x w^T + bias) + residual: x [M, K], w [N, K] (both bf16, rows x_ld and w_ld elements apart), bias [N] in
 * bias_dtype or NULL, residual [M, N] bf16 or NULL, y [M, N] bf16; products summed and the epilogue computed in float32,
 * rounded once. Any M, N, K and strides; rows that start on 16-byte boundaries take wide loads. y may be the residual
 * itself (same pointer and stride); it may share no memory with another operand, but rows with it (columns beside its own).
 */
int zlin_gemm_act(const void* x, long x_ld, const void* w, long w_ld, const void* bias, int bias_dtype, int act,
                  const void* residual, long r_ld, void* y, long y_ld, int M, int N, int K, int dtype, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* ZONOS3_LINEAR_H */
