/*
 * The LM head feeding the sampler on the GPU: the reference's final
 * projection and sampling call (Sain-Kai/noel src/engine.c:377-387:
 * noel_gemv_quantized, src/dequant.c:412-470, then noel_sampler_sample) for a
 * batch of tokens whose hidden states and output weights are on the device.
 */
#ifndef NOEL_LMHEAD_H
#define NOEL_LMHEAD_H

#include <stddef.h>
#include <stdint.h>

#include "noel_int8.h"
#include "noel_logits.h"
#include "noel_lora.h"
#include "noel_requests.h"
#include "sampler.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Row formats of the output weight, with the reference's GGML type ids
 * (include/gguf_loader.h:20-48). */
enum { NOEL_HEAD_F32 = 0, NOEL_HEAD_F16 = 1, NOEL_HEAD_BF16 = 30 };

/*
 * d_logits[b][v] = d_weight[v] . d_hidden[b] for v < vocab, b < batch, in
 * noel_gemv_quantized's summation order (the logits equal the reference's bit
 * for bit), then noel_sampler_sample_batch on those logits in the same stream
 * (histories, RNG states, ids and probabilities as there).  d_weight rows are
 * ldw elements apart and 16-byte aligned; hidden_dim must be a multiple of 8;
 * d_hidden rows are ldh floats apart (16-byte aligned).  d_logits [batch][vocab]
 * receives the logits (they stay in L2 for the sampler when batch x vocab x 4
 * bytes fits).  The weights are read once per eight tokens.  Returns NOEL_OK or
 * a negative status (noel_sampler_cuda_last_error_message() says why).
 */
int noel_lmhead_sample(const noel_sampler_config_t *cfg, const void *d_weight, int weight_type, size_t ldw,
                       const float *d_hidden, size_t ldh, int batch, int hidden_dim, int vocab,
                       const int32_t *d_history, int history_len, size_t hld, uint64_t *d_rng, int32_t *d_ids,
                       float *d_probs, float *d_logits, void *stream);

/*
 * noel_lmhead_sample with what differs from request to request: after the
 * projection, token t's adapter adds its part to the logits (lora and
 * d_adapter [batch], noel_lora_apply; the adapters' rows are the vocabulary
 * and their cols hidden_dim), then process is applied to them
 * (noel_logits_process), then the batch is sampled; all in the same stream.
 * lora or process may be NULL, and with both NULL this is
 * noel_lmhead_sample.  d_work (work_bytes) is noel_lora_apply's scratch and
 * may be NULL without lora.  d_logits receives the logits that were sampled.
 */
int noel_lmhead_sample_ex(const noel_sampler_config_t *cfg, const void *d_weight, int weight_type, size_t ldw,
                          const float *d_hidden, size_t ldh, int batch, int hidden_dim, int vocab,
                          const noel_lora_t *lora, const int32_t *d_adapter, const noel_logits_params_t *process,
                          const int32_t *d_history, int history_len, size_t hld, uint64_t *d_rng, int32_t *d_ids,
                          float *d_probs, float *d_logits, void *d_work, size_t work_bytes, void *stream);

/*
 * The path of a batch whose output weights are in 8 bits and whose requests
 * all differ: noel_i8_linear of the hidden states d_hidden [batch][ldh] (type
 * NOEL_HEAD_F32, NOEL_HEAD_F16 or NOEL_HEAD_BF16) with d_weight [vocab][ldw]
 * and d_weight_scale [vocab] into d_logits [batch][vocab] fp32, then each
 * token's adapter (lora and d_adapter; fp32 hidden states only), then process
 * (noel_logits_process), then noel_sample_requests with params and
 * d_uniforms; all in the same stream.  lora or process may be NULL.  d_logits
 * receives the logits that were sampled.  d_work (16-byte aligned, work_bytes
 * >= noel_lmhead_i8_workspace_bytes(batch, hidden_dim, vocab, lora's rank, or 0
 * without)) is scratch of this call until it has run.  What any step would
 * refuse is refused before the first one runs.  Allocates nothing and may be
 * captured into a graph.
 */
int noel_lmhead_i8_sample(const noel_request_params_t *params, const int8_t *d_weight, size_t ldw,
                          const float *d_weight_scale, const void *d_hidden, int hidden_type, size_t ldh, int batch,
                          int hidden_dim, int vocab, const noel_lora_t *lora, const int32_t *d_adapter,
                          const noel_logits_params_t *process, const float *d_uniforms, int32_t *d_ids, float *d_probs,
                          int32_t *d_counts, float *d_logits, void *d_work, size_t work_bytes, void *stream);

/* Bytes of the scratch that noel_lmhead_i8_sample needs. */
size_t noel_lmhead_i8_workspace_bytes(int batch, int hidden_dim, int vocab, int rank);

#ifdef __cplusplus
}
#endif

#endif /* NOEL_LMHEAD_H */
