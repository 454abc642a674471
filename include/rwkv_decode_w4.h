/*
 * rwkv_decode_w4.h -- the decode step of rwkv_decode.h with 4-bit weights: a
 * cell's six large matrices, and the unembedding, are rwkv_w4.h's packed
 * weights and scales. Everything else is as it is there; a product is formed as
 * in rwkv_w4_linear and rounded to bf16.
 */
#ifndef RWKV_RS_AMD_RWKV_DECODE_W4_H
#define RWKV_RS_AMD_RWKV_DECODE_W4_H

#include "rwkv_decode.h"
#include "rwkv_w4.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct rwkv_w4_matrix {
  const void *packed, *scales;
} rwkv_w4_matrix;

/* In the place of rwkv_decode_cell_params' matrices of these names, with the
 * same shapes; one group size (32, 64 or 128) for all. */
typedef struct rwkv_decode_w4_weights {
  rwkv_w4_matrix receptance, key, value, output, channel_key, channel_value;
  int64_t group;
} rwkv_decode_w4_weights;

/* rwkv_decode_cell with its six matrices taken from `weights`; those of
 * `params` are not looked at. The workspace is rwkv_decode_cell's. */
int rwkv_decode_cell_w4(const rwkv_decode_cell_params *params,
                        const rwkv_decode_w4_weights *weights, float *x,
                        const int32_t *batch_ids, void *state,
                        const float *shift_time_in, float *shift_time_out,
                        const float *shift_channel_in, float *shift_channel_out,
                        const int32_t *elapsed_t, int64_t rows, int64_t num_heads,
                        int64_t full_batch, int state_dtype, int use_dither,
                        void *workspace, int64_t workspace_bytes, void *stream);

/* rwkv_decode_head with a 4-bit unembedding [vocab, C]. */
int rwkv_decode_head_w4(const float *x, const float *norm_weight,
                        const float *norm_bias, float norm_eps,
                        const rwkv_w4_matrix *unembed, int64_t group, int64_t rows,
                        int64_t num_heads, int64_t vocab, void *logits,
                        void *workspace, int64_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* RWKV_RS_AMD_RWKV_DECODE_W4_H */
