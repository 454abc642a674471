/*
 * rwkv_lm_loss_ignore.h -- C ABI of the training loss of rwkv_lm_loss.h on
 * gfx950 where some rows are not learned (prompts, padding): the same, but a row
 * whose target is ignore_index is not read, whatever its logits hold. Its loss and
 * what is kept of it (row_lse, row_max, row_argmax) are 0, and so is its gradient,
 * l2wrap's term included. Any other target outside [0, vocab) gives a NaN loss, as
 * there. Arguments, statuses and rules are those of rwkv_lm_loss.h. No counterpart
 * in the reference.
 */
#ifndef RWKV_RS_AMD_LM_LOSS_IGNORE_H
#define RWKV_RS_AMD_LM_LOSS_IGNORE_H

#include "rwkv_lm_loss.h"

#ifdef __cplusplus
extern "C" {
#endif

int rwkv_cross_entropy_l2wrap_ignore_forward(const void *logits, const int64_t *targets,
                                             int64_t rows, int64_t vocab, int dtype,
                                             int64_t ignore_index, float *row_loss,
                                             float *row_lse, float *row_max,
                                             int32_t *row_argmax, void *stream);

int rwkv_cross_entropy_l2wrap_ignore_backward(const void *logits, const int64_t *targets,
                                              const float *row_lse, const float *row_max,
                                              const int32_t *row_argmax,
                                              const float *row_loss_grad, float l2wrap_scale,
                                              int64_t rows, int64_t vocab, int dtype,
                                              int64_t ignore_index, void *logits_grad,
                                              void *stream);

#ifdef __cplusplus
}
#endif

#endif /* RWKV_RS_AMD_LM_LOSS_IGNORE_H */
