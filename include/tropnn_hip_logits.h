/*
 * C ABI of the operators on rows of logits in libtropnn_hip.so, beside
 * tropnn_hip.h (status codes, tropnn_stream_t and tropnn_hip_last_error are
 * declared there). They have no counterpart in the reference, whose models
 * end in F.cross_entropy (examples/emnist.py:221).
 *
 * Common rules:
 *  - logits: DEVICE pointer to `rows` rows of `vocab` elements of
 *    TROPNN_LOGITS_*, row r starting at element r * row_stride (row_stride >=
 *    vocab unless rows is 1); element alignment is enough.
 *  - 1 <= vocab <= TROPNN_MAX_VOCAB; rows >= 0 (0: nothing is written except
 *    a loss, which is NaN for the mean over no rows and 0 for the sum).
 *  - The library does not allocate: `workspace` holds at least the bytes the
 *    matching _workspace_size query returns for the same arguments (NULL is
 *    fine where that is 0), 16-byte aligned, contents irrelevant before and
 *    after the call (but for tropnn_hip_distill_grad with `holds`).
 *  - Calls are asynchronous on `stream`, and can be captured in a HIP graph.
 *  - The order of a row's logits is: larger value first, NaN before every
 *    number, -0 equal to +0, equal values by ascending index.
 */
#ifndef TROPNN_HIP_LOGITS_H
#define TROPNN_HIP_LOGITS_H

#include "tropnn_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

#define TROPNN_HIP_LOGITS_ABI_VERSION 1

#define TROPNN_LOGITS_F32 0
#define TROPNN_LOGITS_F16 1
#define TROPNN_LOGITS_BF16 2

#define TROPNN_MAX_VOCAB 1048576
#define TROPNN_MAX_TOP 1024

int tropnn_hip_logits_abi_version(void);

/*
 * The k first logits of every row in the order above (1 <= k <=
 * TROPNN_MAX_TOP, k <= vocab) and the log-mass of the others:
 *   values  [rows][k]  elements of `dtype`
 *   indices [rows][k]  int64
 *   log_rest [rows]    f32, log sum over the other logits x of
 *                      exp(x / temperature); -inf where there are none, or
 *                      all of them are -inf; NaN where one is
 */
size_t tropnn_hip_top_logits_workspace_size(int64_t rows, int64_t vocab, int dtype, int64_t k);
int tropnn_hip_top_logits(int64_t rows, int64_t vocab, int64_t row_stride, const void *logits, int dtype, int64_t k,
                          float temperature, void *values, int64_t *indices, float *log_rest, void *workspace,
                          size_t workspace_bytes, tropnn_stream_t stream);

/*
 * Distillation from a teacher's top logits. Per row, with z = logits / t,
 * q = softmax(z), and the teacher's list (values v_j, indices i_j, j < k;
 * entries of a negative index are no part of it):
 *   Z   = log(sum_j exp(v_j / t) + exp(log_rest))     (log_rest NULL: without it)
 *   p_j = exp(v_j / t - Z),  p_0 = exp(log_rest - Z)  (NULL: 0)
 *   q_0 = sum of q over the classes outside the list
 *   L   = t^2 (sum_j p_j log(p_j / q_{i_j}) + p_0 log(p_0 / q_0)),  0 log 0 = 0
 * Rows of weight 0 and rows without a list entry have L = 0 and a zero
 * gradient. loss[0] = scale * sum_r w_r L_r / D, D = sum_r w_r (mean != 0) or
 * 1; weights NULL: all ones. grad (NULL: not wanted), [rows][vocab]
 * contiguous elements of `dtype`, is d loss / d logits.
 * A row's indices are distinct. An index >= vocab makes the row's loss NaN.
 * values: [rows][k] of values_dtype; indices int64 [rows][k]; log_rest and
 * weights f32 [rows]; 1 <= k <= TROPNN_MAX_TOP.
 */
size_t tropnn_hip_distill_workspace_size(int64_t rows, int64_t vocab, int dtype, int64_t k, int want_grad);
int tropnn_hip_distill(int64_t rows, int64_t vocab, int64_t row_stride, const void *logits, int dtype, int64_t k,
                       const void *values, int values_dtype, const int64_t *indices, const float *log_rest,
                       const float *weights, float temperature, float scale, int mean, float *loss, void *grad,
                       void *workspace, size_t workspace_bytes, tropnn_stream_t stream);

/*
 * The chain rule's product of that gradient with the incoming one, factor[0]:
 * grad = factor[0] * d loss / d logits, rounded once to `dtype`. The arguments
 * are those of tropnn_hip_distill and `grad` is non-NULL; no loss is given.
 * holds != 0: grad is what tropnn_hip_distill wrote for the same arguments and,
 * where the mean is weighted (mean != 0 and weights), workspace is that call's,
 * neither touched since. Where factor[0] is 1, grad is then left alone.
 * holds == 0: the contents of both are irrelevant.
 */
int tropnn_hip_distill_grad(int64_t rows, int64_t vocab, int64_t row_stride, const void *logits, int dtype, int64_t k,
                            const void *values, int values_dtype, const int64_t *indices, const float *log_rest,
                            const float *weights, float temperature, float scale, int mean, const float *factor,
                            int holds, void *grad, void *workspace, size_t workspace_bytes, tropnn_stream_t stream);

/*
 * x[i] *= factor[0] for n contiguous elements of TROPNN_LOGITS_*, nothing
 * where factor[0] is 1: the chain rule's product of a saved gradient with the
 * incoming one, which is usually 1. It rounds a second time, which in f32 is
 * nothing; what 16 bits lost at a small scale (f16 has no number below 2^-24)
 * no factor brings back, so such a gradient takes tropnn_hip_distill_grad.
 */
int tropnn_hip_scale_in_place(int64_t n, void *x, int dtype, const float *factor, tropnn_stream_t stream);

/*
 * One token per row from the row's logits x and a given number u in [0, 1):
 *   weight  e_i = exp2((x_i - max) * (log2(e) / temperature)) in f32, w_i =
 *           floor(2^40 e_i) as an integer (so every sum below is exact)
 *   top_k   keep the first top_k logits of the order (<= 0: all)
 *   top_p   of those, keep each one the sum of whose predecessors is below
 *           max(1, floor(top_p * sum))  (>= 1: all)
 *   min_p   of those, keep e_i >= min(min_p, 1)
 *   token   the first i, by index, at which the running sum of the kept w
 *           passes min(floor(u * sum), sum - 1)
 * tokens int64 [rows]; log_probs f32 [rows], log(w_token / sum of the kept).
 * temperature <= 0 or NaN: the first logit of the order, log-probability 0.
 * A row with a NaN or without a logit above -inf has token -1 and
 * log-probability NaN. Each parameter is either one value for all rows or,
 * where its array is not NULL, the row's own.
 */
size_t tropnn_hip_sample_workspace_size(int64_t rows, int64_t vocab, int dtype);
int tropnn_hip_sample(int64_t rows, int64_t vocab, int64_t row_stride, const void *logits, int dtype,
                      const float *uniforms, const float *temperatures, float temperature, const int32_t *top_ks,
                      int32_t top_k, const float *top_ps, float top_p, const float *min_ps, float min_p,
                      int64_t *tokens, float *log_probs, void *workspace, size_t workspace_bytes,
                      tropnn_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* TROPNN_HIP_LOGITS_H */
