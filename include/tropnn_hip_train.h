/*
 * C ABI of the operators that train a token model on its own answers, in
 * libtropnn_hip.so beside tropnn_hip.h and tropnn_hip_logits.h (status codes,
 * tropnn_stream_t, tropnn_hip_last_error and the TROPNN_LOGITS_* types are
 * declared there): log-probabilities of given tokens, the clipped policy loss,
 * the preference loss, and the Adam step with 8-bit states. They have no
 * counterpart in the reference, whose training is F.cross_entropy and
 * torch.optim.AdamW (examples/emnist.py:221, 310).
 *
 * Common rules:
 *  - logits: DEVICE pointer to `rows` rows of `vocab` elements of
 *    TROPNN_LOGITS_*, row r starting at element r * row_stride (row_stride >=
 *    vocab unless rows is 1); element alignment is enough.
 *    1 <= vocab <= TROPNN_MAX_VOCAB, 0 <= rows < 2^31.
 *  - tokens: int64 [rows]. A negative one is none: the row takes no part,
 *    whatever its logits hold. One >= vocab makes its row's values NaN.
 *  - The library does not allocate: workspaces hold at least the bytes that the
 *    matching _workspace_size query returns, 16-byte aligned, contents
 *    irrelevant before and after the call.
 *  - Calls are asynchronous on `stream`, and can be captured in a HIP graph.
 */
#ifndef TROPNN_HIP_TRAIN_H
#define TROPNN_HIP_TRAIN_H

#include "tropnn_hip_logits.h"

#ifdef __cplusplus
extern "C" {
#endif

#define TROPNN_HIP_TRAIN_ABI_VERSION 2

/* elements of an 8-bit state that share an exponent byte */
#define TROPNN_STATE_BLOCK 32

int tropnn_hip_train_abi_version(void);

/* the number of the capture that records `stream`, which no other has; 0: none does */
unsigned long long tropnn_hip_capture_id(tropnn_stream_t stream);

/*
 * log_probs[r] = z_a - log sum_i exp(z_i), z = logits / temperature, a =
 * tokens[r]; 0 where there is no token; NaN where a logit of the row is NaN or
 * +inf, or all are -inf. In f32, in f64 (of f32 sums, without the last rounding), or
 * both: one of the two may be NULL. stats (f32 [rows][2], or NULL): what
 * tropnn_hip_token_gradient needs of the row.
 */
int tropnn_hip_token_log_probs(int64_t rows, int64_t vocab, int64_t row_stride, const void *logits, int dtype,
                               const int64_t *tokens, double temperature, float *log_probs, double *log_probs_f64,
                               float *stats, tropnn_stream_t stream);

/*
 * grad[r][i] = f_r / temperature * ([i == a] - softmax(z)_i), contiguous
 * elements of `dtype`, rounded once, with
 *   f_r = coefs[r / rows_per_coef] * factor[0] / norm[0]  (NULL: 1 in their place)
 * and stats as tropnn_hip_token_log_probs or tropnn_hip_policy wrote them for
 * the same logits, tokens and temperature. Rows without a token, and those whose
 * coefficient or factor is 0, get zeros, whatever they hold.
 * holds != 0: grad is what this call writes for a factor of 1; where factor[0]
 * is 1, it is then left alone.
 */
int tropnn_hip_token_gradient(int64_t rows, int64_t vocab, int64_t row_stride, const void *logits, int dtype,
                              const int64_t *tokens, double temperature, const float *stats, const float *coefs,
                              int64_t rows_per_coef, const float *norm, const float *factor, int holds, void *grad,
                              tropnn_stream_t stream);

/*
 * Per row with a token and a weight other than 0, with lp its log-probability:
 *   q = exp(lp - old_log_probs[r]), A = advantages[r], d = ref_log_probs[r] - lp
 *   L = -min(q A, clamp(q, 1 - low, 1 + high) A) + kl_weight (exp(d) - d - 1)
 * (the last term only where ref_log_probs is not NULL and kl_weight is not 0).
 * loss[0] = scale * sum_r w_r L_r / D, D = sum of w_r over the rows with a
 * token (mean != 0) or 1; weights NULL: all ones. All arrays f32 [rows].
 * Written: log_probs [rows]; coefs [rows], w_r scale dL/dlp / 2^j; norm [1], D /
 * 2^j, with j such that norm has a size of 1/2 to 1 (j 0 where D is 0 or not finite): a
 * term may be past f32 where its share of the mean is not; stats [rows][2]; so that
 * tropnn_hip_token_gradient(coefs, rows_per_coef 1, norm) gives d loss / d logits.
 * grad (NULL: not wanted) is that gradient, rounded once; it can be had where
 * tropnn_hip_policy_grad_fits says so.
 */
int tropnn_hip_policy_grad_fits(int64_t rows, int64_t vocab, int dtype);
size_t tropnn_hip_policy_workspace_size(int64_t rows, int64_t vocab, int dtype, int want_grad);
int tropnn_hip_policy(int64_t rows, int64_t vocab, int64_t row_stride, const void *logits, int dtype,
                      const int64_t *tokens, double temperature, const float *old_log_probs, const float *advantages,
                      const float *ref_log_probs, const float *weights, double low, double high, double kl_weight,
                      double scale, int mean, float *loss, float *log_probs, float *coefs, float *norm, float *stats,
                      void *grad, void *workspace, size_t workspace_bytes, tropnn_stream_t stream);

/*
 * From the log-probabilities of pairs of sequences, token_log_probs f64 and
 * tokens int64, both [2][pairs][length] (the preferred sequences first):
 *   S = sum of a sequence's log-probabilities over its tokens (average != 0:
 *       their mean; a sequence without tokens: 0)
 *   h = beta ((S_0 - reference_0) - (S_1 - reference_1)) - margin
 *   L = -(1 - smoothing) log sigmoid(h) - smoothing log sigmoid(-h)
 * loss[0] = scale * sum_p w_p L_p / D, D = sum w_p (mean != 0) or 1. Pairs of
 * weight 0 take no part, whatever they hold. reference f32 [2][pairs] (NULL:
 * zeros), weights f32 [pairs] (NULL: ones). Written: log_probs f32 [2][pairs],
 * S; coefs f32 [2][pairs], w scale dL / d(a token's log-probability) / 2^j; norm
 * [1], D / 2^j, with j as above; so that tropnn_hip_token_gradient(coefs,
 * rows_per_coef length, norm) gives d loss / d logits.
 */
size_t tropnn_hip_preference_workspace_size(int64_t pairs, int64_t length);
int tropnn_hip_preference(int64_t pairs, int64_t length, const int64_t *tokens, const double *token_log_probs,
                          const float *reference, const float *weights, double beta, double margin, double smoothing,
                          int average, double scale, int mean, float *loss, float *log_probs, float *coefs, float *norm,
                          void *workspace, size_t workspace_bytes, tropnn_stream_t stream);

/*
 * One Adam (decoupled_weight_decay 0) or AdamW step of n_tensors f32 tensors
 * whose states are held in 8 bits. Element i of tensor k, with t = *steps[k] + 1
 * (then stored to *steps[k]), every operation of m and u rounded to f32, in the
 * order beta1 m + (1 - beta1) g and beta2 (u u) + (1 - beta2) (g g):
 *   AdamW:  p = p (1 - lr wd)        Adam: g = g + wd p           (wd != 0)
 *   m = beta1 m + (1 - beta1) g,  u = sqrt(beta2 u^2 + (1 - beta2) g^2)
 *   p = p - (lr / (1 - beta1^t)) (m / (u (1 / sqrt(1 - beta2^t)) + eps))
 * the last to a few units in the last place of the step; a denominator below 2^-126
 * counts as that.
 * m and u (the root of torch's exp_avg_sq) are e4m3 numbers (OCP, one byte) in
 * units of a power of two that TROPNN_STATE_BLOCK consecutive elements share:
 * 2^(b - 127), b the block's exponent byte, the least at which the block's
 * largest finite value is at most 448. They are rounded up or down at random:
 * of the 32-bit number
 *   x = i * 0x9E3779B9 + t * 0xBB67AE85;  x = (x ^ x >> 16) * 0x6A09E667;
 *   x = (x ^ x >> 15) * 0x3C6EF373;       x = x ^ x >> 16          (mod 2^32)
 * the low 16 bits decide for m, the high ones for u, so the expected value is
 * the f32 one (to 2^-17 of a step). A u above 0 becomes no 0; what is not finite
 * becomes NaN. A u of NaN counts as infinite: an element whose gradient's square is
 * past f32 (from 1.85e19 on) takes no step, then and from then on, while m is
 * finite; an infinite or NaN gradient makes its parameter NaN. The root may be the
 * f32 beside the nearest. Zero bytes are a state of zeros.
 * params, grads, exp_avgs, exp_avg_exponents, roots, root_exponents, steps: HOST
 * arrays of n_tensors DEVICE pointers: numels[k] f32 (4-byte aligned) for the
 * first two, numels[k] bytes for the codes, (numels[k] + 31) / 32 bytes for the
 * exponents, one f32 for a step counter; all distinct.
 */
size_t tropnn_hip_adam8_workspace_size(int n_tensors);
int tropnn_hip_adam8_step(int n_tensors, float *const *params, const float *const *grads, uint8_t *const *exp_avgs,
                          uint8_t *const *exp_avg_exponents, uint8_t *const *roots, uint8_t *const *root_exponents,
                          const int64_t *numels, float *const *steps, double lr, double beta1, double beta2, double eps,
                          double weight_decay, int decoupled_weight_decay, void *workspace, size_t workspace_bytes,
                          tropnn_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* TROPNN_HIP_TRAIN_H */
