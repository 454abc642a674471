/*
 * rwkv_dropout.h -- C ABI of dropout on gfx950 whose mask comes from a
 * counter-based generator and is never stored: the backward draws it again.
 * Statuses, dtype codes and threading rules are wkv7.h's. No counterpart in the
 * reference.
 *
 * Element i of n is kept where the 16-bit number u_i is below
 *   T = (1 - p) 65536, rounded to an integer (ties to even)
 * and then multiplied by 65536 / T, so that p is a multiple of 2^-16 and the
 * expectation is exact. u_8q+2k and u_8q+2k+1 are the low and the high half of word
 * k of Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as
 * easy as 1, 2, 3", 2011) at the counter (q mod 2^32, q / 2^32, site, step mod
 * 2^32) and the key (seed mod 2^32, seed / 2^32). seed and step are read from
 * rng[0] and rng[1] on the device when the kernel runs, so that a captured graph
 * draws another mask at each replay if it counts rng[1] up. Calls of one step
 * differ by their site.
 *
 *   out_i = residual_i + (kept ? x_i 65536 / T : 0)
 * in fp32, rounded once to out_dtype; residual (in out_dtype) may be NULL: zeros. A
 * dropped element counts as 0 whatever it is, NaN and infinities too. The backward is the
 * same call on the gradient, without a residual, from out_dtype to dtype; the
 * residual's gradient is the incoming one.
 *
 * Operands are aligned to their elements (rng to 8 bytes); what a call writes may
 * not overlap anything else that it is given.
 */
#ifndef RWKV_RS_AMD_DROPOUT_H
#define RWKV_RS_AMD_DROPOUT_H

#include "wkv7.h"

#ifdef __cplusplus
extern "C" {
#endif

/* The most elements. */
#define RWKV_DROPOUT_MAX_N ((int64_t)1 << 40)

/* x, residual, out [n]; 0 <= p <= 1; 0 <= site < 2^32. */
int rwkv_dropout(const void *x, const void *residual, const int64_t *rng, int64_t site, double p,
                 int64_t n, int dtype, int out_dtype, void *out, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* RWKV_RS_AMD_DROPOUT_H */
