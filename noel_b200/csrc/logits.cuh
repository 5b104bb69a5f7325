/*
 * Per-request processing of logits (include/noel_logits.h): penalties for
 * repeated tokens, biases and masks on a batch of rows, in place.
 *
 * Per row b and id v, with n the occurrences of v among the row's generated
 * ids and seen = v is anywhere in the history:
 *   x = x > 0 ? x / rep : x * rep (seen);  x -= freq n, x -= pres (n > 0);
 *   x += biases on v;  x = -inf (masked)
 * in fp32 with one rounding to bf16 at the end.
 */
#pragma once

#include "sampler_device.cuh"

#include <cuda_bf16.h>

namespace noel {

struct LogitsArgs {
    void *logits;
    int64_t ld;
    int batch, vocab, v_begin;
    const int32_t *hist;
    int64_t hld;
    int hist_len;
    const int32_t *hist_lens, *prompt_lens;
    const float *rep, *freq, *pres;
    const int32_t *bias_ids;
    const float *bias;
    int64_t bld;
    int bias_len;
    const uint32_t *mask;
    int64_t mld;
    int mask_rows;
    const int32_t *mask_row;
    int slices;
};

constexpr int kLogitsThreads = 256;
constexpr int kLogitsSlice = 8192;       // columns of a CTA: one 32-bit word of shared memory each
constexpr int kLogitsMaxBias = 64 * kLogitsThreads;
constexpr int kLogitsMaxHistory = 1 << 29;

/* a column's word: the occurrences among the generated ids, and three marks */
constexpr uint32_t kSeenPrompt = 1u << 31;
constexpr uint32_t kHasBias = 1u << 30;
constexpr uint32_t kManyBiases = 1u << 29;
constexpr uint32_t kCount = kManyBiases - 1;

__device__ __forceinline__ float logit_load(const float *p) { return *p; }
__device__ __forceinline__ float logit_load(const uint16_t *p) { return __uint_as_float((uint32_t)*p << 16); }
__device__ __forceinline__ void logit_store(float *p, float x) { *p = x; }
__device__ __forceinline__ void logit_store(uint16_t *p, float x) {
    *p = __bfloat16_as_ushort(__float2bfloat16_rn(x));  // the one rounding to 16 bits
}

struct RowRules {
    float rep, freq, pres;
};

__device__ __forceinline__ RowRules row_rules(const LogitsArgs &a, int row) {
    return {a.rep ? a.rep[row] : 1.0f, a.freq ? a.freq[row] : 0.0f, a.pres ? a.pres[row] : 0.0f};
}

__device__ __forceinline__ float penalised(float x, uint32_t w, const RowRules &r) {
    const uint32_t n = w & kCount;
    if (w & (kSeenPrompt | kCount)) x = x > 0.0f ? __fdiv_rn(x, r.rep) : __fmul_rn(x, r.rep);
    if (n) x = __fsub_rn(__fsub_rn(x, __fmul_rn(r.freq, (float)n)), r.pres);
    return x;
}

/* the row's mask, or NULL */
__device__ __forceinline__ const uint32_t *row_mask(const LogitsArgs &a, int row) {
    if (!a.mask) return nullptr;
    const int m = a.mask_row ? a.mask_row[row] : row;
    return m >= 0 && m < a.mask_rows ? a.mask + (size_t)m * (size_t)a.mld : nullptr;
}

__device__ __forceinline__ bool allowed(const uint32_t *mask, int id) {
    return !mask || (mask[id >> 5] >> (id & 31) & 1u);
}

/* One CTA per row and slice of kLogitsSlice columns: the slice's words are
 * counted in shared memory from the whole history, then the slice's columns
 * are gone through. */
template <typename T>
__global__ void __launch_bounds__(kLogitsThreads) logits_process_kernel(const __grid_constant__ LogitsArgs a) {
    __shared__ uint32_t word[kLogitsSlice];
    const int tid = threadIdx.x;
    const int row = blockIdx.x / a.slices;
    const int c0 = (blockIdx.x % a.slices) * kLogitsSlice;
    const int width = min(kLogitsSlice, a.vocab - c0);
    const int id0 = a.v_begin + c0;
    T *x = static_cast<T *>(a.logits) + (size_t)row * (size_t)a.ld + c0;
    const uint32_t *mask = row_mask(a, row);
    const RowRules rules = row_rules(a, row);
    for (int i = tid; i < width; i += kLogitsThreads) word[i] = 0u;
    __syncthreads();
    if (a.hist) {
        const int32_t *h = a.hist + (size_t)row * (size_t)a.hld;
        const int len = a.hist_lens ? min(max(a.hist_lens[row], 0), a.hist_len) : a.hist_len;
        const int prompt = a.prompt_lens ? a.prompt_lens[row] : 0;
        for (int i = tid; i < len; i += kLogitsThreads) {
            const int64_t c = (int64_t)h[i] - id0;
            if (c < 0 || c >= width) continue;
            if (i < prompt) atomicOr(&word[c], kSeenPrompt);
            else atomicAdd(&word[c], 1u);
        }
    }
    __syncthreads();  // counts are whole before the marks above them are set
    unsigned long long mine = 0ull;  // the biases whose column this thread marked first
    const int32_t *bi = a.bias_ids ? a.bias_ids + (size_t)row * (size_t)a.bld : nullptr;
    const float *bv = a.bias_ids ? a.bias + (size_t)row * (size_t)a.bld : nullptr;
    const int nb = a.bias_ids ? a.bias_len : 0;
    for (int i = tid, k = 0; i < nb; i += kLogitsThreads, ++k) {
        const int64_t c = (int64_t)bi[i] - id0;
        if (c < 0 || c >= width) continue;
        if (atomicOr(&word[c], kHasBias) & kHasBias) atomicOr(&word[c], kManyBiases);
        else mine |= 1ull << k;
    }
    __syncthreads();
    for (int i = tid, k = 0; i < nb; i += kLogitsThreads, ++k) {
        if (!(mine >> k & 1ull)) continue;
        const int id = bi[i];
        const uint32_t w = word[id - id0];
        if (!allowed(mask, id)) continue;
        float b = bv[i];
        if (w & kManyBiases) {  // which thread came first is chance; the sum goes by the list's order
            b = 0.0f;
            for (int j = 0; j < nb; ++j)
                if (bi[j] == id) b = __fadd_rn(b, bv[j]);
        }
        T *p = x + (id - id0);
        logit_store(p, __fadd_rn(penalised(logit_load(p), w, rules), b));
    }
    for (int i = tid; i < width; i += kLogitsThreads) {
        const uint32_t w = word[i];
        if (!allowed(mask, id0 + i)) logit_store(x + i, -INFINITY);
        else if (w && !(w & kHasBias)) logit_store(x + i, penalised(logit_load(x + i), w, rules));
    }
}

}  // namespace noel
