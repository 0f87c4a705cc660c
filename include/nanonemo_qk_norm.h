/*
 * nanonemo_qk_norm.h — C ABI of the MI355X (gfx950) kernel that normalises the queries and keys of every head and rotates them
 * by their positions, in one pass (libnanonemo_fa.so, built from nanonemo_amd/csrc/qk_norm.hip).
 *
 * For a head's vector x of D values at position p, with half = D/2, n = x / sqrt(mean(x^2) + eps) and v = w n (w: one weight of
 * D values for all query heads, one for all key heads):
 *   y[i] = v[i] cos[p][i] - v[i + half] sin[p][i],   y[i + half] = v[i] sin[p][i] + v[i + half] cos[p][i]   (i < half)
 * in fp32, rounded once to the tensors' type.
 *
 *   - q: [M][H][D], k: [M][KVH][D] for M tokens, views with element strides {token, head} (positive multiples of 8, unit D
 *     stride), 16-byte aligned; D a multiple of 16, up to 256. Weights: dense fp32 [D], 16-byte aligned.
 *   - Position of token m: positions[m % period] (position_bits 32 or 64), or m % period where positions is null. A position
 *     that is not a row of the tables (dense fp32 [table_rows][D/2], 16-byte aligned) makes its token's outputs NaN, and in the
 *     backward its gradients and the weights'.
 *   - dtype: 0 = fp16, 1 = bf16, 2 = fp32. An output may be its own input where their strides are the same.
 *   - Enqueued on `stream`; nothing is allocated, synchronised or read back. Returns 0, or non-zero with the message in
 *     nn_qk_norm_last_error() (thread-local).
 */
#ifndef NANONEMO_QK_NORM_H
#define NANONEMO_QK_NORM_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* strides: {token, head} of q, k, q_out and k_out (8 values). */
int nn_qk_norm_rope_fwd(const void* q, const void* k, const float* q_weight, const float* k_weight, const float* cos_table,
                        const float* sin_table, int64_t table_rows, const void* positions, int position_bits, int64_t period,
                        void* q_out, void* k_out, int64_t M, int64_t H, int64_t KVH, int64_t D, const int64_t* strides,
                        float eps, int dtype, void* stream);

/* Bytes of device workspace of the backward (16-byte aligned): partial sums of the weights' gradients. One call at a time. */
size_t nn_qk_norm_rope_bwd_workspace_size(int64_t M, int64_t H, int64_t KVH, int64_t D);

/* The gradients of q, k and both weights (fp32 [D], dense; zeros for M = 0) from those of the outputs. The weights' are sums
 * over all tokens and heads in an order that the sizes alone decide. strides: {token, head} of dq_out, dk_out, q, k, dq and dk
 * (12 values). */
int nn_qk_norm_rope_bwd(const void* dq_out, const void* dk_out, const void* q, const void* k, const float* q_weight,
                        const float* k_weight, const float* cos_table, const float* sin_table, int64_t table_rows,
                        const void* positions, int position_bits, int64_t period, void* dq, void* dk, float* dq_weight,
                        float* dk_weight, void* workspace, size_t workspace_bytes, int64_t M, int64_t H, int64_t KVH, int64_t D,
                        const int64_t* strides, float eps, int dtype, void* stream);

/* Message of the last failed call on this thread ("" if none). */
const char* nn_qk_norm_last_error(void);

#ifdef __cplusplus
}
#endif

#endif /* NANONEMO_QK_NORM_H */
