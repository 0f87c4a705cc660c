/* C ABI of the distillation kernels (gfx950): a teacher's top logits, and the loss of a student's logits against them. All
 * pointers are device pointers; calls launch on `stream` and neither allocate nor synchronise, and no memset is issued, so
 * they may be captured into a HIP graph. dtype: 0 fp16, 1 bf16, 2 fp32. Functions returning int give 0, or nonzero with
 * nn_distill_last_error set.
 *
 * Logits are R rows of V values side by side: row r begins at element (r / T) * sb + (r % T) * st (sequences of T
 * positions in a larger buffer; a dense matrix has T = R, st = V), at any 2- or 4-byte boundary of its type.
 * 1 <= R < 2^22, 1 <= V <= 393216, 1 <= k <= min(V, 512), 1e-4 <= temperature <= 1e4. Everything else is dense. */
#ifndef NANONEMO_DISTILL_H
#define NANONEMO_DISTILL_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* The k largest of each row, descending, equal ones by index (NaN above +inf; -0 equals 0 and is given as 0, a NaN of any
 * bits as one of them): values [R][k] of the logits' dtype, indices int64 [R][k], and rest[R] = logsumexp(the other logits /
 * temperature) in fp32, -inf where there are none. Deterministic. */
int nn_top_logits(const void* logits, int64_t T, int64_t sb, int64_t st, void* values, int64_t* indices, float* rest, int64_t R,
                  int64_t V, int64_t k, double temperature, int dtype, void* stream);

/* Doubles of the statistics that the forward keeps for the backward. */
size_t nn_distill_stats_size(int64_t R);

/* loss[1] = the mean over the rows that count of weight * temperature^2 * KL(p || q) + (1 - weight) * CE, where
 *   p  the teacher's: softmax of values / temperature over the row's k indices; with rest (not NULL), rest is one class more;
 *   q  the student's: softmax of logits / temperature over all V; with rest, all logits outside the k are one class;
 *   CE logsumexp(logits) - logits[target], with targets (not NULL) and weight < 1.
 * A row counts unless its target is -100 (all do without targets). values [R][k] of value_dtype, indices int64 [R][k] in any
 * order (an index that is there twice adds up its probabilities), rest fp32 [R], targets int64 [R]. NaN where no row counts,
 * and where an index or target of a row that counts is out of range. 0 <= weight <= 1. Deterministic. */
int nn_distill_fwd(const void* logits, int64_t T, int64_t sb, int64_t st, const void* values, const int64_t* indices, const float* rest,
                   const int64_t* targets, float* loss, double* stats, int64_t R, int64_t V, int64_t k, double temperature,
                   double weight, int dtype, int value_dtype, void* stream);

/* dlogits [R][V] dense, of the logits' dtype: the gradient of loss times grad[0] (fp32); stats as the forward wrote them, the
 * other arguments as it had them. Zero in rows that do not count, whatever they hold; NaN in a row with an index or target
 * out of range. */
int nn_distill_bwd(const float* grad, const void* logits, int64_t T, int64_t sb, int64_t st, const void* values,
                   const int64_t* indices, const int64_t* targets, const double* stats, void* dlogits, int64_t R, int64_t V, int64_t k,
                   double temperature, double weight, int dtype, int value_dtype, void* stream);

const char* nn_distill_last_error(void);

#ifdef __cplusplus
}
#endif

#endif /* NANONEMO_DISTILL_H */
