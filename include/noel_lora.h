/*
 * Low-rank adapters of many requests at once beside a shared projection: the
 * projection (the LM head of noel_lmhead.h, or any other with fp32 outputs)
 * is computed for the whole batch with one weight, and each token's own
 * adapter adds its low-rank part.  The reference has no adapters; this entry
 * point has no counterpart there.
 */
#ifndef NOEL_LORA_H
#define NOEL_LORA_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/*
 * n_adapters adapters of one weight [rows][cols]: adapter i is
 * scale[i] * B_i A_i with A_i [rank][cols] at d_a + i * stride_a (rows lda
 * elements apart) and B_i [rows][rank] at d_b + i * stride_b (rows ldb
 * elements apart), both of one type (NOEL_HEAD_F32, NOEL_HEAD_F16 or
 * NOEL_HEAD_BF16 of noel_lmhead.h) and aligned to the element size.  An
 * adapter of a smaller rank says so in d_ranks; what its arrays hold beyond
 * that rank is not used.
 */
typedef struct {
    const void *d_a;
    size_t lda, stride_a;
    const void *d_b;
    size_t ldb, stride_b;
    const float *d_scale;   /* [n_adapters]; NULL: 1 */
    const int32_t *d_ranks; /* [n_adapters] (clamped to 0 .. rank); NULL: rank */
    int type;
    int n_adapters;
    int rank;               /* 1 .. 256 */
} noel_lora_t;

/* Bytes of the scratch that noel_lora_apply needs for batch tokens. */
size_t noel_lora_workspace_bytes(int batch, int rank);

/*
 * d_y[t] += scale[i] * B_i (A_i d_x[t]), i = d_adapter[t], for t < batch:
 * d_x [batch][ldx] (cols used) and d_y [batch][ldy] (rows used) fp32, 4-byte
 * aligned and apart from each other.  A token whose d_adapter is outside 0 ..
 * n_adapters - 1 has no adapter and its row of d_y is left as it was.
 *
 * Products of fp16 and bf16 weights enter their sums exactly, of fp32 weights to
 * 2^-30 (of numbers above 2^-100).  Of A_i x 32 columns at a time, and of B_i
 * times that 64 ranks at a time (fp32 weights 32), are added by matrix
 * instructions of 16 products, which add in 32 bits and cut where fp32 rounds;
 * those sums are added in fp32, the latter to d_y one after the other.  The order
 * depends on the adapters' sizes and on whether d_x, ldx, d_a, lda and stride_a
 * are all multiples of 16 bytes: a token's result does not depend on which and
 * how many other tokens are in the batch, on its place there, on n_adapters or on
 * the addresses and pitches of B_i and d_y.  Where a sum in fp32 is infinite or
 * NaN the result is one of the two.
 *
 * d_work (16-byte aligned, work_bytes >= noel_lora_workspace_bytes(batch, rank))
 * is scratch of this call until it has run.  Returns NOEL_OK or a negative status
 * (noel_sampler_cuda_last_error_message() says why).  Asynchronous on stream;
 * allocates nothing and may be captured into a graph.
 */
int noel_lora_apply(const noel_lora_t *lora, const int32_t *d_adapter, const float *d_x, size_t ldx, int batch,
                    int cols, int rows, float *d_y, size_t ldy, void *d_work, size_t work_bytes, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* NOEL_LORA_H */
