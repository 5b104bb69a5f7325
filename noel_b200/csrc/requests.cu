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
    a.status = static_cast<int32_t *>(const_cast<void *>(work));
    *out = a;
    return NOEL_OK;
}

/* a kernel over grid CTAs in clusters, after the one before it or (dependent) once that allows it */
template <typename... A>
cudaError_t launch(void (*kernel)(A...), int grid, int threads, size_t smem, int cluster, bool dependent, cudaStream_t s, A... args) {
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3((unsigned)grid);
    lc.blockDim = dim3((unsigned)threads);
    lc.dynamicSmemBytes = smem;
    lc.stream = s;
    cudaLaunchAttribute at[2];
    unsigned n = 0;
    if (cluster > 1) {
        at[n].id = cudaLaunchAttributeClusterDimension;
        at[n].val.clusterDim.x = (unsigned)cluster;
        at[n].val.clusterDim.y = at[n].val.clusterDim.z = 1;
        ++n;
    }
    if (dependent) {
        at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    lc.attrs = at;
    lc.numAttrs = n;
    return cudaLaunchKernelEx(&lc, kernel, args...);
}

template <typename T>
int request_launch(RequestArgs a, int sms, cudaStream_t s) {
    constexpr int kMost = 190 * 1024;
    /* the pass */
    PassArgs p{};
    p.r = a;
    int parts = 8;
    while (parts > 1 && (int64_t)a.batch * parts > 4 * sms) parts /= 2;
    const int per_vec = 16 / (int)sizeof(T), per_turn = parts * kPassThreads * kPassEach / per_vec;
    p.turns = (a.vocab / per_vec + per_turn - 1) / per_turn;
    if (p.turns < 1) p.turns = 1;
    auto divisor = [](int x, int y) {
        while (y) {
            const int z = x % y;
            x = y, y = z;
        }
        return x;
    };
    p.step = (int)(p.turns * 0.618);
    while (p.step > 1 && divisor(p.turns, p.step) != 1) --p.step;
    if (p.step < 1) p.step = 1;
    p.order = parts == 1 && a.batch > 4 * sms && a.batch <= 4096;  // more than one turn of the GPU; each CTA looks at all settings
    const size_t pass_smem = kPassKeep * sizeof(uint64_t);
    int r = dynamic_smem((const void *)sample_pass_kernel<T>, pass_smem);
    if (r) return r;
    /* one division of the SMs' memory for both kernels, or neither starts where the other runs */
    for (const void *kernel : {(const void *)sample_pass_kernel<T>, (const void *)sample_requests_kernel<T>})
        CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
    /* the rows that it does not take, and those that it leaves */
    const int64_t row = (int64_t)a.vocab * sizeof(T);
    const int cluster = row > 262144 ? 16 : row > 131072 ? 8 : row > 65536 ? 4 : 2;
    if (cluster > 8)
        CUDA_TRY(cudaFuncSetAttribute((const void *)sample_requests_kernel<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    const int unit = kReqThreads;  // every warp's region in whole turns
    a.per = ((a.vocab + cluster - 1) / cluster + unit - 1) / unit * unit;
    size_t smem = (size_t)a.per * sizeof(T);
    a.resident = smem <= kMost;
    if (!a.resident) smem = 0;
    r = dynamic_smem((const void *)sample_requests_kernel<T>, smem);
    if (r) return r;
    CUDA_TRY(launch(sample_pass_kernel<T>, a.batch * parts, kPassThreads, pass_smem, parts, false, s, p));
    const int most = a.batch < 256 ? sms / cluster : 2 * sms / cluster;
    CUDA_TRY(launch(sample_requests_kernel<T>, (a.batch < 2 * sms / cluster ? a.batch : most) * cluster, kReqThreads, smem, cluster, true, s, a));
    return NOEL_OK;
}

}  // namespace

extern "C" size_t noel_sample_requests_workspace_bytes(int batch, int vocab) {
    return batch > 0 && vocab > 0 ? (size_t)batch * sizeof(int32_t) : 0;  // whether a row is settled
}

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
    if (!r) r = dtype == NOEL_DTYPE_F32 ? request_launch<float>(a, sms, s) : request_launch<__nv_bfloat16>(a, sms, s);
    return r ? r : ok();
} catch (...) {
    return fail(NOEL_ERR_CUDA, "host memory");
}
