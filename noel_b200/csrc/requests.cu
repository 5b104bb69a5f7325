/*
 * Host side of sampling with every row's own settings
 * (include/noel_requests.h), and of the path from 8-bit output weights to it.
 */
#include "noel_requests.h"

#include "host.h"
#include "noel_lmhead.h"
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
    /* a row to a CTA where the batch fills the GPU (four CTAs to an SM), to a cluster of up to eight elsewhere: 256 mixed
     * rows of 152,064 fp32 in 1, 2 and 4 parts 186, 164 and 161 us, 1024 rows 271, 316 and 395 */
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
    /* the rows that it does not take, and those that it leaves, in clusters by the row's size: 1024 rows of 256,000 bf16
     * with 10 rows left take 295 us in clusters of 16 and 330 in clusters of 8, 37 open rows of 50,001 bf16 53, 42 and 33 us
     * in clusters of 16 (two turns of the GPU), 8 and 4 */
    const int64_t row = (int64_t)a.vocab * sizeof(T);
    int cluster = row > 262144 ? 16 : row > 131072 ? 8 : row > 65536 ? 4 : 2;
    while (cluster < 16 && (int64_t)a.batch * cluster <= sms / 2 && a.vocab / cluster >= 2048) cluster *= 2;  // SMs are free
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
    /*
     * A CTA or two to an SM.  Where the pass settles the rows, one spares the launch of the others: chat settings, 20 rows
     * 23.5 us against 27.2, 128 rows 38.9 and 42.5; min-p 18.6 and 20.7, 26.4 and 30.3.  Where it leaves them two are
     * faster: 128 rows of wide nuclei 784 us against 685, without filters 257 and 237; 255 nucleus rows of 256,000 bf16 176
     * and 158.  With 256 mixed rows some are left in most batches.
     */
    const int most = a.batch < 256 ? sms / cluster : 2 * sms / cluster;
    CUDA_TRY(launch(sample_requests_kernel<T>, (a.batch <= 2 * sms / cluster ? a.batch : most) * cluster, kReqThreads, smem, cluster, true, s, a));
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

/* ------------------------------- 8-bit LM head -> adapters -> processing -> sampler */
namespace {
/* the steps run one after the other, so they share one scratch */
size_t head_work(int batch, int hidden_dim, int vocab, int rank) {
    const size_t sizes[] = {noel_i8_linear_workspace_bytes(batch, hidden_dim), rank > 0 ? noel_lora_workspace_bytes(batch, rank) : 0,
                            noel_sample_requests_workspace_bytes(batch, vocab)};
    size_t most = 0;
    for (const size_t n : sizes) most = n > most ? n : most;
    return most;
}
}  // namespace

extern "C" size_t noel_lmhead_i8_workspace_bytes(int batch, int hidden_dim, int vocab, int rank) {
    return batch > 0 ? head_work(batch, hidden_dim, vocab, rank) : 0;
}

extern "C" int noel_lmhead_i8_sample(const noel_request_params_t *params, const int8_t *d_weight, size_t ldw,
                                     const float *d_weight_scale, const void *d_hidden, int hidden_type, size_t ldh,
                                     int batch, int hidden_dim, int vocab, const noel_lora_t *lora,
                                     const int32_t *d_adapter, const noel_logits_params_t *process, const float *d_uniforms,
                                     int32_t *d_ids, float *d_probs, int32_t *d_counts, float *d_logits, void *d_work,
                                     size_t work_bytes, void *stream) try {
    /* what a later step would refuse of the whole batch is refused before the first one runs; noel_i8_linear, the first
     * one, checks its own arguments before it launches */
    RequestArgs a{};
    int r = request_args(params, d_logits, NOEL_DTYPE_F32, batch, vocab, (size_t)(vocab > 0 ? vocab : 0), d_uniforms, d_ids,
                         d_probs, d_counts, d_work, work_bytes, &a);
    if (r) return r;
    if (lora && hidden_type != NOEL_HEAD_F32) return fail(NOEL_ERR_UNSUPPORTED, "adapters need fp32 hidden states (type %d)", hidden_type);
    if (lora && (r = lora_check(lora, d_adapter, static_cast<const float *>(d_hidden), ldh, batch, hidden_dim, vocab, d_logits,
                                (size_t)vocab, d_work, work_bytes)))
        return r;
    /* what noel_logits_process refuses by its plan for the device are more rows and columns than request_args lets by */
    if (process && (r = logits_check(process, d_logits, batch, vocab, (size_t)vocab))) return r;
    const size_t need = noel_lmhead_i8_workspace_bytes(batch, hidden_dim, vocab, lora ? lora->rank : 0);
    if (need > 0 && (!d_work || work_bytes < need))
        return fail(NOEL_ERR_INVALID_ARG, "scratch of %zu bytes, %zu wanted", d_work ? work_bytes : 0, need);
    r = noel_i8_linear(d_hidden, hidden_type, ldh, batch, d_weight, ldw, d_weight_scale, vocab, hidden_dim, d_logits,
                       NOEL_DTYPE_F32, (size_t)vocab, d_work, work_bytes, stream);
    if (!r && lora)
        r = noel_lora_apply(lora, d_adapter, static_cast<const float *>(d_hidden), ldh, batch, hidden_dim, vocab, d_logits,
                            (size_t)vocab, d_work, work_bytes, stream);
    if (!r && process) r = noel_logits_process(process, d_logits, NOEL_DTYPE_F32, batch, vocab, (size_t)vocab, stream);
    if (!r)
        r = noel_sample_requests(params, d_logits, NOEL_DTYPE_F32, batch, vocab, (size_t)vocab, d_uniforms, d_ids, d_probs,
                                 d_counts, d_work, work_bytes, stream);
    return r;
} catch (...) {
    return fail(NOEL_ERR_CUDA, "host memory");
}
