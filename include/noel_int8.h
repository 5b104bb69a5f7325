/*
 * Projections in 8-bit integers: weights in memory take a byte each, with a
 * scale for every output channel; tokens are cast to 8 bits with a scale for
 * every token.  The reference multiplies blocks of quantised weights with
 * fp32 activations on the host (Sain-Kai/noel src/dequant.c:412-470); these
 * entry points have no counterpart there.
 */
#ifndef NOEL_INT8_H
#define NOEL_INT8_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Columns of an 8-bit product at most: its sums are exact in 32 bits. */
enum { NOEL_I8_MAX_COLS = 131071 };

/*
 * Cast rows to 8 bits, each with its own scale:
 *   d_scale[r] = max(max_c |d_x[r][c]| / 127, 2^-126), rounded to fp32,
 *   d_q[r][c]  = d_x[r][c] / d_scale[r] to the nearest integer, ties to even
 * (of the exact quotient, so -127 .. 127).  A row that holds an infinity or a
 * NaN gets the scale NaN and zeros.  Weights are cast the same way, an output
 * channel to a row.
 * d_x [rows][ldx] of type NOEL_HEAD_F32, NOEL_HEAD_F16 or NOEL_HEAD_BF16
 * (noel_lmhead.h), aligned to the element size; d_q [rows][ldq] 16-byte
 * aligned, ldq a multiple of 16, its columns from cols on left as they are;
 * d_scale [rows].  Returns NOEL_OK or a negative status
 * (noel_sampler_cuda_last_error_message() says why).  Asynchronous on stream;
 * allocates nothing and may be captured into a graph.
 */
int noel_i8_cast(const void *d_x, int type, size_t ldx, int rows, int cols, int8_t *d_q, size_t ldq, float *d_scale,
                 void *stream);

/*
 * d_y[t][v] = d_w_scale[v] * d_a_scale[t] * sum_c d_a[t][c] * d_w[v][c] for t
 * < tokens, v < rows: sums exact, the sum's fp32 value times d_w_scale[v],
 * then times d_a_scale[t], each rounded to fp32, and to bf16 where d_y is.  A
 * result does not depend on the other tokens and rows of the call.
 * tokens and rows may be 2^31 - 513 at most.
 * d_a [tokens][lda] and d_w [rows][ldw] (cols used, 1 .. NOEL_I8_MAX_COLS)
 * 16-byte aligned with lda and ldw multiples of 16; d_y [tokens][ldy] of dtype
 * NOEL_DTYPE_F32 or NOEL_DTYPE_BF16 (noel_sampler_cuda.h), aligned to the
 * element size, apart from the inputs; its columns from rows on are left as
 * they are.  Waits inside the kernel are limited
 * (noel_sampler_cuda_set_wait_limit) and reported by
 * noel_sampler_cuda_sync_check of the stream (of any, for a call that a graph
 * captured); once one has run out no further tile is begun, the others end as
 * well, and the call within another limit and a millisecond.  Otherwise as
 * noel_i8_cast.
 */
int noel_i8_product(const int8_t *d_a, size_t lda, const float *d_a_scale, int tokens, const int8_t *d_w, size_t ldw,
                    const float *d_w_scale, int rows, int cols, void *d_y, int dtype, size_t ldy, void *stream);

/* Bytes of the scratch that noel_i8_linear needs. */
size_t noel_i8_linear_workspace_bytes(int tokens, int cols);

/*
 * A projection: noel_i8_cast of the tokens d_x [tokens][ldx] into d_work, then
 * noel_i8_product, whose first weights are on their way while the tokens are
 * cast.  d_work (16-byte aligned, work_bytes >=
 * noel_i8_linear_workspace_bytes(tokens, cols)) is scratch of this call until
 * it has run.
 */
int noel_i8_linear(const void *d_x, int type, size_t ldx, int tokens, const int8_t *d_w, size_t ldw,
                   const float *d_w_scale, int rows, int cols, void *d_y, int dtype, size_t ldy, void *d_work,
                   size_t work_bytes, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* NOEL_INT8_H */
