/*
 * Host side of sampling with every row's own settings
 * (include/noel_requests.h).
 */
#include "noel_requests.h"

#include "host.h"
#include "requests.cuh"

using namespace noel;

namespace {

bool misaligned(const void *p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to != 0; }

int request_args(const noel_request_params_t *p, const void *logits, int dtype, int batch, int vocab, size_t ld,
                 const float *u, int32_t *ids, float *probs, int32_t *counts, const void *work, size_t work_bytes,
                 RequestArgs *out) {
    if (!p) return fail(NOEL_ERR_INVALID_ARG, "params is NULL");
    if (dtype != NOEL_DTYPE_F32 && dtype != NOEL_DTYPE_BF16) return fail(NOEL_ERR_UNSUPPORTED, "dtype %d (F32 0, BF16 1)", dtype);
    if (batch < 0 || vocab <= 0) return fail(NOEL_ERR_INVALID_ARG, "batch %d / vocab %d", batch, vocab);
    if (vocab > NOEL_REQUESTS_MAX_VOCAB) return fail(NOEL_ERR_TOO_LARGE, "vocab %d (1..%d)", vocab, NOEL_REQUESTS_MAX_VOCAB);
    if (batch > 1 << 24) return fail(NOEL_ERR_TOO_LARGE, "batch %d", batch);
    if (ld < (size_t)vocab) return fail(NOEL_ERR_INVALID_ARG, "ld %zu < vocab %d", ld, vocab);
    if (misaligned(logits, dtype == NOEL_DTYPE_F32 ? 4 : 2)) return fail(NOEL_ERR_INVALID_ARG, "logits not aligned to their elements");
    const void *arrays[] = {p->d_temperature, p->d_top_k, p->d_top_p, p->d_min_p, u, ids, probs, counts};
    for (const void *q : arrays)
        if (misaligned(q, 4)) return fail(NOEL_ERR_INVALID_ARG, "arrays must be 4-byte aligned");
    if (misaligned(work, 16)) return fail(NOEL_ERR_INVALID_ARG, "scratch must be 16-byte aligned");
    if (batch > 0 && (!logits || !u || !ids)) return fail(NOEL_ERR_INVALID_ARG, "logits, uniforms and ids are required");
    const size_t need = noel_sample_requests_workspace_bytes(batch, vocab);
    if (need > 0 && (!work || work_bytes < need))
        return fail(NOEL_ERR_INVALID_ARG, "scratch of %zu bytes, %zu wanted", work ? work_bytes : 0, need);
    RequestArgs a{};
    a.logits = logits, a.ld = (int64_t)ld, a.batch = batch, a.vocab = vocab;
    a.temperature = p->d_temperature, a.top_k = p->d_top_k, a.top_p = p->d_top_p, a.min_p = p->d_min_p;
    a.u = u, a.ids = ids, a.probs = probs, a.counts = counts;
    *out = a;
    return NOEL_OK;
}

template <typename T>
int request_launch(RequestArgs a, cudaStream_t s) {
    constexpr int kCluster = kReqMaxCluster, kMost = 190 * 1024;
    const int unit = kReqThreads;  // every warp's region in whole turns
    a.per = ((a.vocab + kCluster - 1) / kCluster + unit - 1) / unit * unit;
    size_t smem = (size_t)a.per * sizeof(T);
    a.resident = smem <= kMost;
    if (!a.resident) smem = 0;
    const int r = dynamic_smem((const void *)sample_requests_kernel<T>, smem);
    if (r) return r;
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3((unsigned)a.batch * kCluster);
    lc.blockDim = dim3(kReqThreads);
    lc.dynamicSmemBytes = smem;
    lc.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = kCluster;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    lc.attrs = at;
    lc.numAttrs = 1;
    CUDA_TRY(cudaLaunchKernelEx(&lc, sample_requests_kernel<T>, a));
    CUDA_TRY(cudaGetLastError());
    return NOEL_OK;
}

}  // namespace

extern "C" size_t noel_sample_requests_workspace_bytes(int, int) { return 0; }

extern "C" int noel_sample_requests(const noel_request_params_t *params, const void *d_logits, int dtype, int batch,
                                    int vocab, size_t ld, const float *d_uniforms, int32_t *d_ids, float *d_probs,
                                    int32_t *d_counts, void *d_work, size_t work_bytes, void *stream) try {
    RequestArgs a{};
    int r = request_args(params, d_logits, dtype, batch, vocab, ld, d_uniforms, d_ids, d_probs, d_counts, d_work, work_bytes, &a);
    if (r) return r;
    if (batch == 0) return ok();
    int sms = 0;
    r = device_sms(&sms);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (!r) r = dtype == NOEL_DTYPE_F32 ? request_launch<float>(a, s) : request_launch<__nv_bfloat16>(a, s);
    return r ? r : ok();
} catch (...) {
    return fail(NOEL_ERR_CUDA, "host memory");
}
