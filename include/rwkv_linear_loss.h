/*
 * rwkv_linear_loss.h -- C ABI of the language model's training loss straight
 * from its last hidden states and its unembedding, on gfx950: the cross entropy
 * with l2wrap's gradient term of rwkv_lm_loss.h, of logits that are formed in
 * tiles and never stored. Statuses, dtype codes and threading rules are wkv7.h's.
 * No counterpart in the reference, which forms the logits (model.rs:150-169).
 *
 * hidden [rows, c], weight [vocab, c] row-major in dtype, targets int64 [rows].
 *
 * Forward:
 *   z_rj   = sum_k hidden_rk weight_jk      (exact products, fp32 sums)
 *   max_r     = max_j z_rj
 *   log_sum_r = log sum_j exp(z_rj - max_r)
 *   loss_r    = (max_r - z_r,t_r) + log_sum_r
 * to row_loss, row_log_sum, row_max (fp32 [rows]) and row_argmax (int32 [rows], the
 * first index of the row's maximum); the last three are kept for the backward. The
 * maximum and the logarithm stay apart: in one number they would be rounded to a
 * step of the logits' size. A
 * row whose target is ignore_index has loss 0, and nothing depends on its hidden
 * state; one whose target is otherwise outside [0, vocab) has a NaN loss. A row with a NaN or
 * plus infinity among its logits has a NaN loss; minus infinity is a probability of
 * 0 (bf16 operands; fp32 ones' products make it NaN).
 *
 * Backward, with g_r = row_loss_grad[r] (fp32 [rows]):
 *   D_rj = g_r (exp(z_rj - max_r - log_sum_r) - [j == t_r]) + [j == argmax_r] l2wrap_scale max_r
 *   hidden_grad = D weight,   weight_grad = D^T hidden
 * in dtype, each rounded once; either pointer may be NULL (not wanted). A row
 * whose target is ignore_index has D = 0; a target otherwise outside [0, vocab)
 * no target term. z is formed again, a piece of the vocabulary at a time, with at
 * most 512 MiB of D in memory (or a tile of 256 words). D is held in fp16, each row
 * over the size of its own factors, |g_r| or |l2wrap_scale max_r|: 11 bits of each
 * element, but never finer than 2^-37 of the row's larger factor; for fp32 operands in
 * two such numbers, 22 bits (or whole, in three bf16 ones). The hidden gradient's
 * products round it to bf16 for bf16 operands, but for the target and the argmax,
 * whose error is put back. The weight gradient's are fp16, of hidden states scaled by
 * a power of two and by their row's factor over the largest row's: each holds 11 bits
 * (22 for fp32 operands), but never finer than 2^-37 of the largest magnitude and
 * factor. With bf16 operands the sums of the hidden gradient hold 2^14 of the weights:
 * these are below 2^112 in magnitude.
 *
 * fp32 operands are multiplied as two fp16 numbers each, after a power of two that
 * brings the operand's largest magnitude to 2^13 .. 2^14: 22 bits of each element, but
 * never finer than 2^-38 of that largest magnitude, three products, fp32 sums. Where
 * there are few rows and many words, as three bf16 numbers each that hold an element
 * whole, of nine products the six of 2^-15 and more.
 *
 * Operands are aligned to their elements, and where c is a multiple of 8, hidden,
 * weight and their gradients to 16 bytes. What a call writes may not overlap
 * anything else that it is given.
 */
#ifndef RWKV_RS_AMD_LINEAR_LOSS_H
#define RWKV_RS_AMD_LINEAR_LOSS_H

#include "wkv7.h"

#ifdef __cplusplus
extern "C" {
#endif

/* The most of each size, and of an operand's elements. */
#define RWKV_LINEAR_LOSS_MAX_ROWS (1 << 22)
#define RWKV_LINEAR_LOSS_MAX_VOCAB (1 << 22)
#define RWKV_LINEAR_LOSS_MAX_C (1 << 16)
#define RWKV_LINEAR_LOSS_MAX_ELEMENTS ((int64_t)1 << 33)

/* Device memory that a call asks for (16-byte aligned, no initialisation; calls
 * that may overlap in time need one each), or -1 for sizes or a dtype that are not
 * supported. */
int64_t rwkv_linear_loss_forward_workspace_bytes(int64_t rows, int64_t vocab, int64_t c, int dtype);
int64_t rwkv_linear_loss_backward_workspace_bytes(int64_t rows, int64_t vocab, int64_t c, int dtype);

int rwkv_linear_loss_forward(const void *hidden, const void *weight, const int64_t *targets,
                             int64_t rows, int64_t vocab, int64_t c, int dtype,
                             int64_t ignore_index, float *row_loss, float *row_log_sum,
                             float *row_max, int32_t *row_argmax, void *workspace,
                             int64_t workspace_bytes, void *stream);

/* row_log_sum, row_max and row_argmax are the forward's of the same operands. */
int rwkv_linear_loss_backward(const void *hidden, const void *weight, const int64_t *targets,
                              const float *row_log_sum, const float *row_max,
                              const int32_t *row_argmax, const float *row_loss_grad,
                              float l2wrap_scale, int64_t rows, int64_t vocab, int64_t c,
                              int dtype, int64_t ignore_index, void *hidden_grad,
                              void *weight_grad, void *workspace, int64_t workspace_bytes,
                              void *stream);

#ifdef __cplusplus
}
#endif

#endif /* RWKV_RS_AMD_LINEAR_LOSS_H */
