/*
 * rwkv_w4.h -- C ABI of products with 4-bit weights on gfx950: quantising a
 * linear layer's weight, restoring it, and multiplying rows of activations
 * with it. Statuses, dtype codes and threading rules are wkv7.h's. No
 * counterpart in the reference.
 *
 * The format. A weight is a 4-bit float (a sign, two exponent bits, one
 * mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6 with either sign) times the bf16
 * scale of its group, `group` consecutive inputs of one output; group is 32,
 * 64 or 128. The matrix [out, in] is stored in blocks of 16 outputs and 128
 * inputs, the last ones filled up with zero weights. With ob = ceil(out / 16)
 * and ib = ceil(in / 128):
 *   packed  uint8 [ob][ib][4][16][16]: byte 4 j + b of [n][k][g][r] holds the
 *           weights of output 16 n + r at inputs 128 k + 32 j + 8 g + 2 b (low
 *           half) and the one after it (high half)
 *   scales  bf16 [ob][ib][16][128 / group]: [n][k][r][q] is that of output
 *           16 n + r and inputs 128 k + group q ..
 * Code c stands for the magnitude number c & 7, negative when c & 8. A lane of
 * a matrix instruction reads its 32 weights as 16 consecutive bytes.
 *
 * packed and scales are aligned to 16 bytes, other operands to their elements.
 * What a call writes may not overlap anything else that it is given.
 */
#ifndef RWKV_RS_AMD_RWKV_W4_H
#define RWKV_RS_AMD_RWKV_W4_H

#include "wkv7.h"

#ifdef __cplusplus
extern "C" {
#endif

/* The most outputs and inputs, and the most rows, that a call takes. A weight
 * has at most 2^31 - 1 blocks. */
#define RWKV_W4_MAX_DIM (1 << 26)
#define RWKV_W4_MAX_ROWS (1 << 20)

/* Bytes of `packed` and of `scales`, or -1 for sizes or a group that are not
 * supported. */
int64_t rwkv_w4_packed_bytes(int64_t out, int64_t in);
int64_t rwkv_w4_scales_bytes(int64_t out, int64_t in, int64_t group);

/* weight [out, in] (fp32 or bf16) to packed and scales. A group's scale is
 * its largest magnitude times 1/6, rounded to bf16 (at most the largest bf16
 * number six times which is an fp32 number); a weight takes the nearest
 * value, ties going to an even mantissa, and beyond 6 scales the largest. A
 * group with an infinity or a NaN gets a NaN scale, so that what is computed
 * with it is NaN. */
int rwkv_w4_quantize(const void *weight, int64_t out, int64_t in, int64_t group,
                     int dtype, void *packed, void *scales, void *stream);

/* The weights that packed and scales stand for, [out, in] in dtype (exact in
 * fp32, rounded once in bf16). */
int rwkv_w4_dequantize(const void *packed, const void *scales, int64_t out,
                       int64_t in, int64_t group, int dtype, void *weight,
                       void *stream);

/* Device memory that rwkv_w4_linear asks for (16-byte aligned, no
 * initialisation), 0 for none (always up to 16 rows), or -1 for sizes or a dtype
 * that are not supported: with few outputs and many inputs, workgroups share
 * the inputs and leave their sums there. */
int64_t rwkv_w4_linear_workspace_bytes(int64_t rows, int64_t out, int64_t in,
                                       int dtype);

/* y [rows, out] = x [rows, in] W^T, x and y in dtype. Products are exact in
 * fp32 (bf16 x) or formed from x's three bf16 parts, which hold it whole (fp32
 * x; what of it is below 2^-133 is lost); sums are fp32, the scale is applied to
 * a group's sum in fp32, and y is rounded once. Sums are kept 1024 times too
 * small, so that none overflows where y does not; a group adds up to 2^-140 to
 * the error of a y near the least numbers. */
int rwkv_w4_linear(const void *x, const void *packed, const void *scales,
                   int64_t rows, int64_t out, int64_t in, int64_t group,
                   int dtype, void *y, void *workspace, int64_t workspace_bytes,
                   void *stream);

#ifdef __cplusplus
}
#endif

#endif /* RWKV_RS_AMD_RWKV_W4_H */
