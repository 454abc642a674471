/*
 * rwkv_token_scores.h -- C ABI of what a language model's answer is scored by,
 * on gfx950: the log probability of a given token, the entropy and the most
 * likely alternatives of each row of logits, and the gradient of all three.
 * No counterpart in the reference.
 *
 * Forward, for each row r of logits ([rows, vocab] row-major in dtype) and its
 * token t_r (int64):
 *   max_r      = max_j x_rj,   log_sum_r = log sum_j exp(x_rj - max_r)
 *   log p_rj   = x_rj - max_r - log_sum_r
 *   log_prob_r = log p_r,t_r
 *   entropy_r  = -sum_j p_rj log p_rj, where 0 log 0 = 0
 *   top_ids_r  the `top` largest logits' indices, largest first, the lower
 *              index first among equals; top_log_probs_r their log p_rj
 * Logits of minus infinity (tokens that a mask leaves out) have probability 0;
 * they come last among the alternatives, with a log probability of minus
 * infinity. A row without a distribution -- every logit minus infinity, or one
 * of them NaN or plus infinity -- gets NaN throughout, and -1 for its ids. A
 * token outside [0, vocab) gets a NaN log probability; the rest of its row is
 * as ever. No log probability is above 0 and no entropy below it, by rounding
 * either.
 *
 * Backward, with g = log_prob_grad[r], h = entropy_grad[r], t_i =
 * top_grad[r][i] (each of the three arrays may be NULL: zeros):
 *   dx_rj = [j == t_r] g + sum_i [j == top_ids_ri] t_i
 *           - p_rj (g + sum_i t_i + h (log p_rj + entropy_r))
 * summed in fp32 and rounded once to dtype, zero where p_rj is 0 and j is
 * neither the token nor an alternative. A token outside [0, vocab) has no
 * first term. A row without a distribution has a NaN gradient.
 *
 * Conventions are those of wkv7.h: status codes (checked on the host before
 * any launch), WKV7_DTYPE_* codes, work enqueued on `stream` without
 * synchronising, nothing allocated, outputs that overlap no other operand.
 * Every operand is aligned to its element.
 */
#ifndef RWKV_RS_AMD_TOKEN_SCORES_H
#define RWKV_RS_AMD_TOKEN_SCORES_H

#include "wkv7.h"

#ifdef __cplusplus
extern "C" {
#endif

/* The most alternatives of a row. */
#define RWKV_TOKEN_SCORES_MAX_TOP 64

/* log_prob, entropy, row_max, row_log_sum [rows], top_log_probs [rows, top]
 * fp32, top_ids [rows, top] int64. The maxima and log sums are for the backward,
 * and may be NULL; so are the last two when top is 0. Sizes: 0 <= rows, 0 <
 * vocab, both below 2^31, 0 <= top <= min(vocab, the most). */
int rwkv_token_scores_forward(const void *logits, const int64_t *tokens, int64_t rows,
                              int64_t vocab, int64_t top, int dtype, float *log_prob,
                              float *entropy, float *row_max, float *row_log_sum,
                              float *top_log_probs, int64_t *top_ids, void *stream);

/* row_max, row_log_sum, entropy and top_ids are the forward's. */
int rwkv_token_scores_backward(const void *logits, const int64_t *tokens, const float *row_max,
                               const float *row_log_sum, const float *entropy,
                               const int64_t *top_ids, const float *log_prob_grad,
                               const float *entropy_grad, const float *top_grad, int64_t rows,
                               int64_t vocab, int64_t top, int dtype, void *logits_grad, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* RWKV_RS_AMD_TOKEN_SCORES_H */
