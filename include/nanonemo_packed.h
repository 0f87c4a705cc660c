/*
 * nanonemo_packed.h — C ABI of the MI355X (gfx950) causal grouped-query attention over packed sequences
 * (libnanonemo_fa.so, built from nanonemo_amd/csrc/flash_attn.hip).
 *
 * n sequences of lengths[0 .. n - 1] >= 0 tokens lie one behind the other in tensors
 *   q, o, dO, dq   [tokens, H,   D]    k, v, dk, dv   [tokens, KVH, D]    lse   [H, tokens] fp32
 * with tokens their sum: row t of sequence i is row lengths[0] + .. + lengths[i - 1] + t. A query sees the keys of its own
 * sequence up to itself; otherwise everything is as in nanonemo_fa.h (types, head_dim 32 or 64, scale, lse, errors through
 * nn_fa_last_error, work only enqueued on `stream`, no atomics), and a sequence's o and lse are the same bits as nn_fa_fwd's on
 * it alone.
 *
 * rest: tokens * H * D bytes, or null. The forward writes into it what rounding o to 16 bits took off each value, in 8 bits, and
 * a backward that is given it computes D = rowsum(dO * o) from both: dq and dk then carry the rounding of dS and their own, and
 * none of o's. Without it dq is the same bits as nn_fa_bwd's. (Sequences that the plan gives to a wave as one tile of 32 rows need
 * none: their rests are left as they were, and D is formed in the backward.)
 *
 * The work is laid out once for a batch, on the host: nn_fa_packed_plan fills `plan` (int32 words, in host memory), which the
 * caller copies to the device as it is (16-byte aligned) and keeps while it uses it, in both places. Its layout is the
 * library's own, but for the last `tokens` words, from word plan[NN_FA_PACKED_POSITIONS] on, which hold every row's position
 * in its sequence. A call whose device copy differs from the host's computes other values, within the tensors' bounds.
 */
#ifndef NANONEMO_PACKED_H
#define NANONEMO_PACKED_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define NN_FA_PACKED_POSITIONS 15

/* int32 words of the plan of these sequences; 0 for arguments that have none (nn_fa_last_error says why). */
size_t nn_fa_packed_plan_words(const int64_t* lengths, int64_t n, int64_t H, int64_t KVH);

/* Fills plan[0 .. words - 1], words as nn_fa_packed_plan_words returned it. Host memory only; nothing touches the GPU. */
int nn_fa_packed_plan(const int64_t* lengths, int64_t n, int64_t H, int64_t KVH, int32_t* plan, size_t words);

/* What a plan is of. */
typedef struct {
    int64_t words, sequences, H, KVH, tokens, longest;
} nn_fa_packed_info;
int nn_fa_packed_plan_info(const int32_t* plan, nn_fa_packed_info* info);

/* Forward; lse may be null where no backward follows. strides: element strides {head, row} of q, of k and v, and of o (6 values;
 * positive multiples of 8, rows at least D apart), or null for dense tensors. */
int nn_fa_packed_fwd(const void* q, const void* k, const void* v, void* o, float* lse, void* rest, const int32_t* plan,
                     const int32_t* device_plan, int64_t D, const int64_t* strides, int dtype, float scale, void* stream);

/* Bytes of device workspace of the backward, 256-byte aligned: -rowsum(dO * o) and -lse / scale, and where pairs of 64-key
 * units are shared by several blocks (few or uneven sequences) their partial dk and dv. One call at a time. */
size_t nn_fa_packed_bwd_workspace_size(const int32_t* plan, int64_t D);

/* Backward. strides: {head, row} of q and dO, of k and v, of o, of dq, and of dk and dv (10 values), or null. */
int nn_fa_packed_bwd(const void* dO, const void* q, const void* k, const void* v, const void* o, const float* lse,
                     const void* rest, void* dq, void* dk, void* dv, void* workspace, size_t workspace_bytes, const int32_t* plan,
                     const int32_t* device_plan, int64_t D, const int64_t* strides, int dtype, float scale, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* NANONEMO_PACKED_H */
