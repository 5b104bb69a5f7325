/*
 * Sampling where every row has settings of its own: temperature, top-k,
 * top-p and min-p for each request of a batch, with the random numbers given.
 * The reference samples with one configuration and draws its own numbers
 * (Sain-Kai/noel src/sampler.c:80-192; noel_sampler_sample_batch here); this
 * entry point has no counterpart there.
 */
#ifndef NOEL_REQUESTS_H
#define NOEL_REQUESTS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Ids of a row at most. */
enum { NOEL_REQUESTS_MAX_VOCAB = 1048576 };

/* Settings of each row; NULL leaves the setting out for every row. */
typedef struct {
    const float *d_temperature; /* [batch]; NULL: 1 */
    const int32_t *d_top_k;     /* [batch]; NULL or <= 0: all ids */
    const float *d_top_p;       /* [batch]; NULL, >= 1 or NaN: all */
    const float *d_min_p;       /* [batch]; NULL, <= 0 or NaN: all */
} noel_request_params_t;

/*
 * Draw one id from each row.  With x the row's logits, m the largest of them
 * and T its temperature, in this order:
 *
 *   left are the ids with x >= m - 30 T, and with x >= m + T ln(min(min_p, 1));
 *   of those the first top_k by (x descending, id ascending);
 *   of those, in that order, the fewest (one at least) whose weights
 *     exp((x - m) / T) sum to at least top_p times the sum of all of theirs;
 *   the id drawn is the lowest of those at which the running sum of their
 *     weights, in the order of ids, exceeds u times their sum (u >= 1: the
 *     highest id left; u < 0 or NaN: as 0).
 *
 * T <= 0 or NaN takes the largest logit, the lowest id of several.  A NaN or
 * -infinity among the logits is never drawn; several +infinity share the draw
 * alike; a row with nothing to draw gets id -1, probability 0 and count 0.
 * Sums are of weights rounded to multiples of 2^-43 and exact, so results do
 * not depend on the batch or on the order of anything.
 *
 * d_logits [batch][ld] of dtype NOEL_DTYPE_F32 or NOEL_DTYPE_BF16, aligned to
 * the element size, the first vocab columns used and left as they are;
 * d_uniforms [batch] u in [0, 1); d_ids [batch]; d_probs [batch] the drawn id's
 * weight over the sum of those left (NULL: not wanted); d_counts [batch] how
 * many ids were left (NULL: not wanted).  d_work (16-byte aligned, work_bytes
 * >= noel_sample_requests_workspace_bytes(batch, vocab)) is scratch of this
 * call until it has run.  Returns NOEL_OK or a negative status
 * (noel_sampler_cuda_last_error_message() says why).  Asynchronous on stream;
 * allocates nothing and may be captured into a graph.
 */
int noel_sample_requests(const noel_request_params_t *params, const void *d_logits, int dtype, int batch, int vocab,
                         size_t ld, const float *d_uniforms, int32_t *d_ids, float *d_probs, int32_t *d_counts,
                         void *d_work, size_t work_bytes, void *stream);

/* Bytes of the scratch that noel_sample_requests needs. */
size_t noel_sample_requests_workspace_bytes(int batch, int vocab);

#ifdef __cplusplus
}
#endif

#endif /* NOEL_REQUESTS_H */
