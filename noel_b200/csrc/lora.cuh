/*
 * Low-rank adapters beside a shared projection (include/noel_lora.h):
 * y[t] += scale_i B_i (A_i x[t]), i = adapter[t].
 *
 * Two kernels: the first writes scale_i A_i x[t] (rank numbers a token) to
 * the caller's scratch, the second multiplies it by B_i and adds it to y.
 */
#pragma once

#include "lmhead.cuh"

namespace noel {

constexpr int kLoraMaxRank = 256;
constexpr int kLoraThreads = 256;

struct LoraArgs {
    const void *a, *b;
    int64_t lda, stride_a, ldb, stride_b;
    const float *scale;
    const int32_t *ranks;
    int n, rank;
    const int32_t *adapter;
    const float *x;
    int64_t ldx;
    int batch, cols, rows;
    float *y;
    int64_t ldy;
    float *low;  // [batch][rank]
};

template <int WT>
__device__ __forceinline__ float lora_weight(const void *p, size_t i) {
    if (WT == kHeadF32) return static_cast<const float *>(p)[i];
    const uint16_t u = static_cast<const uint16_t *>(p)[i];
    return WT == kHeadBF16 ? __uint_as_float((uint32_t)u << 16) : __half2float(__ushort_as_half(u));
}

__device__ __forceinline__ int lora_rank(const LoraArgs &a, int i) {
    return a.ranks ? min(max(a.ranks[i], 0), a.rank) : a.rank;
}

/* one warp per token and rank */
template <int WT>
__global__ void __launch_bounds__(kLoraThreads) lora_shrink_kernel(const __grid_constant__ LoraArgs a) {
    const int lane = threadIdx.x & 31;
    const int64_t w = ((int64_t)blockIdx.x * kLoraThreads + threadIdx.x) >> 5;
    const int t = (int)(w / a.rank), r = (int)(w % a.rank);
    if (t >= a.batch) return;
    const int i = a.adapter[t];
    if (i < 0 || i >= a.n || r >= lora_rank(a, i)) return;
    const size_t at = (size_t)i * (size_t)a.stride_a + (size_t)r * (size_t)a.lda;
    const float *x = a.x + (size_t)t * (size_t)a.ldx;
    float s = 0.0f;
    for (int d = lane; d < a.cols; d += 32) s = __fmaf_rn(x[d], lora_weight<WT>(a.a, at + d), s);
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(kFull, s, o);
    if (lane == 0) a.low[(size_t)t * a.rank + r] = a.scale ? s * a.scale[i] : s;
}

/* one thread per token (blockIdx.y) and row */
template <int WT>
__global__ void __launch_bounds__(kLoraThreads) lora_expand_kernel(const __grid_constant__ LoraArgs a) {
    const int v = blockIdx.x * kLoraThreads + threadIdx.x;
    for (int t = blockIdx.y; t < a.batch; t += gridDim.y) {
        const int i = a.adapter[t];
        if (i < 0 || i >= a.n || v >= a.rows) continue;
        const int n = lora_rank(a, i);
        const size_t at = (size_t)i * (size_t)a.stride_b + (size_t)v * (size_t)a.ldb;
        float s = 0.0f;
        for (int r = 0; r < n; ++r) s = __fmaf_rn(a.low[(size_t)t * a.rank + r], lora_weight<WT>(a.b, at + r), s);
        float *y = a.y + (size_t)t * (size_t)a.ldy + v;
        *y = __fadd_rn(*y, s);
    }
}

}  // namespace noel
