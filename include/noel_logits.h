/*
 * Per-request processing of logits on the GPU, in place, between the logits
 * and the sampler: penalties for repeated tokens, biases and masks, each with
 * values of its own for every row of the batch.  The reference has one
 * repetition penalty for every row (Sain-Kai/noel src/sampler.c:87-103) and,
 * in its pipeline, a mask that keeps a single id
 * (src/pipeline_stages.c:81-94); this entry point has no counterpart there.
 */
#ifndef NOEL_LOGITS_H
#define NOEL_LOGITS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/*
 * What is applied to row b, id v.  With history h = d_history[b][0 .. len) and
 * its first prompt_len ids the prompt, n = the number of times v occurs in
 * h[prompt_len .. len), and seen = v occurs anywhere in h:
 *
 *   x = x > 0 ? x / repetition[b] : x * repetition[b]      where seen
 *   x = x - frequency[b] * n - presence[b]                 where n > 0
 *   x = x + the sum of the row's biases on v               where it has any
 *   x = -infinity                                          where masked
 *
 * The repetition penalty is applied once however often v occurs (the
 * sampler's own penalty is applied once per occurrence).  Ids that the
 * columns do not hold are skipped, so rows may be padded with -1.  An id
 * listed several times among a row's biases gets their sum, added in list
 * order.  Every array may be NULL, which leaves its part out.  A mask wins
 * over everything else, NaN included; a row whose mask allows nothing becomes
 * -infinity throughout.
 */
typedef struct {
    const int32_t *d_history;      /* [batch][hld] token ids */
    size_t hld;
    int history_len;               /* ids per row, at most */
    const int32_t *d_history_lens; /* [batch] ids of each row (clamped to 0 .. history_len); NULL: history_len */
    const int32_t *d_prompt_lens;  /* [batch] leading ids that are prompt; NULL: 0 */
    const float *d_repetition;     /* [batch]; NULL: 1 */
    const float *d_frequency;      /* [batch]; NULL: 0 */
    const float *d_presence;       /* [batch]; NULL: 0 */
    const int32_t *d_bias_ids;     /* [batch][bld] token ids */
    const float *d_bias;           /* [batch][bld] */
    size_t bld;
    int bias_len;                  /* biases per row */
    const uint32_t *d_mask;        /* [mask_rows][mld] words; bit v % 32 of word v / 32 set: id v is allowed */
    size_t mld;
    int mask_rows;
    const int32_t *d_mask_rows;    /* [batch] row of d_mask (outside 0 .. mask_rows - 1: no mask); NULL: row b */
    int v_begin;                   /* id of the first column (a vocabulary shard's; 0 for whole rows) */
} noel_logits_params_t;

/*
 * Apply params to d_logits [batch][ld] (dtype NOEL_DTYPE_F32 or
 * NOEL_DTYPE_BF16, aligned to the element size; column c holds id
 * params->v_begin + c for c < vocab <= ld) in place.  Computed in fp32; a
 * bf16 element is rounded once, at the end.  Elements that no rule touches
 * keep their bits, and so do columns from vocab on.  history_len < 2^29,
 * bias_len <= 16384.  Returns NOEL_OK or a negative status
 * (noel_sampler_cuda_last_error_message() says why).  Asynchronous on
 * stream; allocates nothing and may be captured into a graph.
 */
int noel_logits_process(const noel_logits_params_t *params, void *d_logits, int dtype, int batch, int vocab, size_t ld,
                        void *stream);

#ifdef __cplusplus
}
#endif

#endif /* NOEL_LOGITS_H */
