/*
 * What the library's translation units share on the host: the calling
 * thread's status and message, and the per-device context.
 */
#pragma once

#include <cuda_runtime.h>

#include <stddef.h>

#include "noel_logits.h"
#include "noel_lora.h"
#include "noel_sampler_cuda.h"

namespace noel {

/* Keep code and the formatted message as the thread's last error; returns code. */
__attribute__((visibility("hidden"), format(printf, 2, 3))) int fail(int code, const char *fmt, ...);
/* Clear them; returns NOEL_OK. */
__attribute__((visibility("hidden"))) int ok();
/* The current device's number of SMs (an error where it is not sm_100). */
__attribute__((visibility("hidden"))) int device_sms(int *sms);
/* Let kernel take bytes of dynamic shared memory on the current device. */
__attribute__((visibility("hidden"))) int dynamic_smem(const void *kernel, size_t bytes);
/* Limit of the device-side waits of the calling thread's calls, in ns. */
__attribute__((visibility("hidden"))) unsigned long long wait_limit_ns();
/* Whether the thread asked that its next call load nothing (which ends the request). */
__attribute__((visibility("hidden"))) bool take_stall();
/* What noel_lora_apply and noel_logits_process (of fp32 logits) refuse of these arguments; nothing is launched. */
__attribute__((visibility("hidden"))) int lora_check(const noel_lora_t *lora, const int32_t *adapter, const float *x, size_t ldx,
                                                     int batch, int cols, int rows, float *y, size_t ldy, void *work,
                                                     size_t work_bytes);
__attribute__((visibility("hidden"))) int logits_check(const noel_logits_params_t *params, float *logits, int batch, int vocab,
                                                       size_t ld);
/* Whether a product in 8 bits gave up since the stream's last call of this: one launched on the stream, or one of a graph. */
__attribute__((visibility("hidden"))) int i8_wait_failed(cudaStream_t s, bool *failed);

#define CUDA_TRY(call)                                                                     \
    do {                                                                                   \
        cudaError_t e_ = (call);                                                           \
        if (e_ != cudaSuccess) return fail(NOEL_ERR_CUDA, "%s: %s", #call, cudaGetErrorString(e_)); \
    } while (0)

}  // namespace noel
