/* C ABI of the embedding kernels (gfx950). All pointers are device pointers; calls launch on `stream` and neither allocate
 * nor synchronise, and no memset is issued, so they may be captured into a HIP graph. dtype: 0 fp16, 1 bf16, 2 fp32.
 * idx_bits: 32 or 64, the width of a token. Functions returning int give 0, or nonzero with nn_embedding_last_error set.
 * Stands for nn.Embedding, the model's first layer (/root/reference/nanonemo/model/model.py:13-70), with a scale. */
#ifndef NANONEMO_EMBEDDING_H
#define NANONEMO_EMBEDDING_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* out[m] = scale * weight[idx[m]], rounded once. weight [V][N] and out [M][N] dense, of one dtype; idx [M]. A row whose
 * token is not in [0, V) is NaN. 0 <= M < 2^31, 1 <= V < 2^27, 1 <= N < 2^20; M N and V N below 2^42, and M N below 2^34
 * where rows are not whole units of 16 bytes. */
int nn_embedding_fwd(const void* weight, const void* idx, void* out, int64_t M, int64_t V, int64_t N, float scale, int dtype,
                     int idx_bits, void* stream);

/* Bytes of workspace of the backward (a multiple of 16; the workspace is 16-byte aligned and belongs to one call at a time). */
size_t nn_embedding_bwd_workspace_size(int64_t M, int64_t V, int64_t N);

/* dw[v] = scale * the sum of dy[m] over the m with idx[m] = v, summed in fp32 and rounded once: written, not accumulated; zero
 * for rows without a token and for padding_idx (negative: none). Tokens outside [0, V) take no part. The sum's order depends on
 * idx and the sizes alone (in order of m within pieces of up to 64, whose sums are joined in a fixed order), so the result is
 * bit-reproducible. dy [M][N] and dw [V][N] dense, of one dtype. */
int nn_embedding_bwd(const void* dy, const void* idx, void* dw, void* workspace, size_t workspace_bytes, int64_t M, int64_t V,
                     int64_t N, float scale, int64_t padding_idx, int dtype, int idx_bits, void* stream);

const char* nn_embedding_last_error(void);

#ifdef __cplusplus
}
#endif

#endif /* NANONEMO_EMBEDDING_H */
