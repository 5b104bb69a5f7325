/*
 * Low-rank adapters beside a shared projection (include/noel_lora.h):
 * y[t] += scale_i B_i (A_i x[t]), i = adapter[t].
 *
 * The tokens of a batch are taken in items: up to 16 tokens of one adapter,
 * so that an adapter's weights are read once for 16 tokens.  The first kernel
 * multiplies an item's x by A_i (its rank numbers per token go to the caller's
 * scratch), the second multiplies those by B_i and adds them to y.  What has
 * to move is y, read and written, and the weights of the adapters in use; the
 * products are matrix instructions (16 tokens x 8 rows x 16) so that they stay
 * behind the memory at any rank.
 *
 * fp32 numbers go through 16-bit matrix instructions in parts: x is cut into
 * three bf16 numbers of 8 significant bits each, which hold its 24 bits
 * exactly; bf16 weights are one part, fp16 weights two (exactly), fp32 weights
 * three.  All products of parts are added, smallest first, but for the last
 * parts' of two fp32 numbers (2^-30 of the product), so a sum is as exact as
 * in fp32.
 */
#pragma once

#include "lmhead.cuh"

#include <cooperative_groups.h>

#include <utility>

namespace noel {

constexpr int kLoraMaxRank = 256;
constexpr int kLoraBatch = 2048;    // tokens of one pass over the adapters
constexpr int kLoraItem = 16;       // tokens of an item
constexpr int kLoraWarpBatch = 32;  // tokens up to which every warp finds the items by itself
constexpr int kShrinkThreads = 512;
constexpr int kShrinkSplit = 8;     // CTAs of a cluster that share an item's columns, at most
constexpr int kExpandThreads = 256;
constexpr int kExpandWaves = 16;    // CTAs of the second kernel per SM, at most

/* the items of a batch above kLoraWarpBatch, in the scratch */
struct LoraPlan {
    int n;                       // items
    int adapter[kLoraBatch];     // of each item
    int first[kLoraBatch + 1];   // place in order of its first token
    int order[kLoraBatch];       // tokens, item by item
};

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
    uint16_t *low;   // [batch][3][rank_pad] bf16 parts of scale A x
    int rank_pad;    // 16, or the rank rounded up to 32
    LoraPlan *plan;  // NULL: every warp finds the items
    int vec_x, vec_a, vec_b, vec_y;  // rows start on 16 bytes (B with rank_pad 16: on 4 elements)
};

__device__ __forceinline__ int lora_rank(const LoraArgs &a, int i) {
    return a.ranks ? min(max(a.ranks[i], 0), a.rank) : a.rank;
}

/* ------------------------------------------------------------- the items */
/* Item k of a batch of at most 32 tokens: its adapter (-1: there is none) and
 * its tokens as a mask.  Token t belongs to lane t; the items are in the order
 * of their first tokens. */
__device__ __forceinline__ int warp_item(const LoraArgs &a, int k, uint32_t &tokens, int &items) {
    const int lane = threadIdx.x & 31;
    const int i = lane < a.batch ? a.adapter[lane] : -1;
    const bool valid = i >= 0 && i < a.n;
    const uint32_t same = __match_any_sync(kFull, valid ? i : -1);
    const int rank = __popc(same & lanemask_lt());
    const uint32_t heads = __ballot_sync(kFull, valid && rank % kLoraItem == 0);
    items = __popc(heads);
    tokens = 0u;
    if (k >= items) return -1;
    const int head = __fns(heads, 0, k + 1);
    const int adapter = __shfl_sync(kFull, i, head), chunk = __shfl_sync(kFull, rank, head) / kLoraItem;
    tokens = __ballot_sync(kFull, valid && i == adapter && rank / kLoraItem == chunk);
    return adapter;
}

/* One CTA: tokens of one adapter counted and numbered in a table of adapters,
 * adapters numbered in the table's order, every 16 tokens an item.  Which
 * token of an adapter gets which number is chance; no result depends on it. */
template <int kPlanThreads, int PER>  // for up to kPlanThreads x PER tokens
__global__ void __launch_bounds__(kPlanThreads) lora_plan_kernel(const __grid_constant__ LoraArgs a) {
    constexpr int kPlanSlots = 2 * kPlanThreads * PER;  // a power of two
    __shared__ int key[kPlanSlots], count[kPlanSlots];
    __shared__ int wsum[kPlanThreads / 32], wtok[kPlanThreads / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    for (int s = tid; s < kPlanSlots; s += kPlanThreads) {
        key[s] = 0;
        count[s] = 0;
    }
    __syncthreads();
    int slot[PER], number[PER];
#pragma unroll
    for (int u = 0; u < PER; ++u) {
        const int t = u * kPlanThreads + tid;
        const int i = t < a.batch ? a.adapter[t] : -1;
        slot[u] = -1;
        if (i < 0 || i >= a.n) continue;
        uint32_t p = (uint32_t)i * 0x9E3779B1u / (0xFFFFFFFFu / kPlanSlots + 1u);
        for (int probe = 0; probe < kPlanSlots; ++probe) {  // at most half of the slots are taken
            const int prev = atomicCAS(&key[p], 0, i + 1);
            if (prev == 0 || prev == i + 1) break;
            p = (p + 1) % kPlanSlots;
        }
        slot[u] = (int)p;
        number[u] = atomicAdd(&count[p], 1);
    }
    __syncthreads();
    /* prefix sums over the slots: items and tokens */
    constexpr int SPT = kPlanSlots / kPlanThreads;
    int items = 0, toks = 0;
#pragma unroll
    for (int u = 0; u < SPT; ++u) {
        const int c = count[tid * SPT + u];
        items += (c + kLoraItem - 1) / kLoraItem;
        toks += c;
    }
    int pi = items, pt = toks;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int vi = __shfl_up_sync(kFull, pi, o), vt = __shfl_up_sync(kFull, pt, o);
        if (lane >= o) {
            pi += vi;
            pt += vt;
        }
    }
    if (lane == 31) {
        wsum[warp] = pi;
        wtok[warp] = pt;
    }
    __syncthreads();
    int bi = 0, bt = 0;
    for (int w = 0; w < warp; ++w) {
        bi += wsum[w];
        bt += wtok[w];
    }
    if (tid == kPlanThreads - 1) {
        a.plan->n = bi + pi;
        a.plan->first[bi + pi] = bt + pt;
    }
    bi += pi - items;
    bt += pt - toks;
#pragma unroll
    for (int u = 0; u < SPT; ++u) {
        const int s = tid * SPT + u, c = count[s];
        for (int k = 0; k * kLoraItem < c; ++k) {
            a.plan->adapter[bi + k] = key[s] - 1;
            a.plan->first[bi + k] = bt + k * kLoraItem;
        }
        key[s] = bt;  // from here on the place of the slot's first token
        bi += (c + kLoraItem - 1) / kLoraItem;
        bt += c;
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < PER; ++u)
        if (slot[u] >= 0) a.plan->order[key[slot[u]] + number[u]] = u * kPlanThreads + tid;
}

/* -------------------------------------------------------------- the parts */
/* v's next part: its upper 16 bits; what is left stays in v.  An infinity or a
 * NaN is one part (a NaN keeps a bit in the part that is taken). */
__device__ __forceinline__ uint32_t take_part(float &v) {
    uint32_t u = __float_as_uint(v);
    if ((u & 0x7F800000u) == 0x7F800000u) {
        if (u & 0x007FFFFFu) u |= 0x00400000u;
        v = 0.0f;
        return u & 0xFFFF0000u;
    }
    u &= 0xFFFF0000u;
    v = __fsub_rn(v, __uint_as_float(u));  // exact
    return u;
}
/* the next parts of two numbers as a bf16 pair */
__device__ __forceinline__ uint32_t take_parts(float &lo, float &hi) {
    return __byte_perm(take_part(lo), take_part(hi), 0x7632);
}
/* N numbers in P parts, as bf16 pairs */
template <int N, int P>
__device__ __forceinline__ void split(float (&f)[N], uint32_t (&x)[P][N / 2]) {
    float odd = 0.0f;  // stays 0 unless a number is infinite or NaN
#pragma unroll
    for (int e = 0; e < N; ++e) odd = __fmaf_rn(f[e], 0.0f, odd);
    if (odd == 0.0f) {
#pragma unroll
        for (int i = 0; i < P; ++i)
#pragma unroll
            for (int e = 0; e < N; e += 2) {
                const uint32_t u = __float_as_uint(f[e]), v = __float_as_uint(f[e + 1]);
                x[i][e / 2] = __byte_perm(u, v, 0x7632);
                if (i + 1 < P) {
                    f[e] = __fsub_rn(f[e], __uint_as_float(u & 0xFFFF0000u));
                    f[e + 1] = __fsub_rn(f[e + 1], __uint_as_float(v & 0xFFFF0000u));
                }
            }
    } else {
#pragma unroll
        for (int i = 0; i < P; ++i)
#pragma unroll
            for (int e = 0; e < N; e += 2) x[i][e / 2] = take_parts(f[e], f[e + 1]);
    }
}

template <int WT>
constexpr int kWeightParts = WT == kHeadBF16 ? 1 : WT == kHeadF16 ? 2 : 3;

/* N consecutive weights as bf16 pairs, part by part */
template <int WT, int N>
struct Weights {
    uint32_t p[kWeightParts<WT>][N / 2];
};

/* weights at p; valid (<= N) of them exist and used (<= N) of them count, the
 * others are 0; vec: p is aligned to the N weights (16 bytes at most) */
template <int WT, int N>
__device__ __forceinline__ Weights<WT, N> load_weights(const void *p, int valid, int used, bool vec) {
    Weights<WT, N> w;
    if (WT == kHeadBF16) {
        uint32_t *u = w.p[0];
        if (vec && valid >= N) {
            if (N == 8) {
                const uint4 q = __ldg(static_cast<const uint4 *>(p));
                u[0] = q.x, u[1] = q.y, u[N / 2 - 2] = q.z, u[N / 2 - 1] = q.w;
            } else {
                const uint2 q = __ldg(static_cast<const uint2 *>(p));
                u[0] = q.x, u[1] = q.y;
            }
            if (used < N) {
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (e >= used) u[e / 2] &= e & 1 ? 0x0000FFFFu : 0xFFFF0000u;
            }
        } else {
            const uint16_t *h = static_cast<const uint16_t *>(p);
#pragma unroll
            for (int e = 0; e < N; e += 2)
                u[e / 2] = (e < used ? (uint32_t)h[e] : 0u) | (e + 1 < used ? (uint32_t)h[e + 1] << 16 : 0u);
        }
    } else {
        float f[N];
        if (WT == kHeadF16) {
            const __half *h = static_cast<const __half *>(p);
            if (vec && valid >= N) {
                uint32_t u[N / 2];
                if (N == 8) {
                    const uint4 q = __ldg(static_cast<const uint4 *>(p));
                    u[0] = q.x, u[1] = q.y, u[N / 2 - 2] = q.z, u[N / 2 - 1] = q.w;
                } else {
                    const uint2 q = __ldg(static_cast<const uint2 *>(p));
                    u[0] = q.x, u[1] = q.y;
                }
#pragma unroll
                for (int e = 0; e < N; ++e)
                    f[e] = e < used ? __half2float(__ushort_as_half((uint16_t)(u[e / 2] >> (16 * (e & 1))))) : 0.0f;
            } else {
#pragma unroll
                for (int e = 0; e < N; ++e) f[e] = e < used ? __half2float(h[e]) : 0.0f;
            }
        } else {
            const float *s = static_cast<const float *>(p);
            if (vec && valid >= N) {
#pragma unroll
                for (int e = 0; e < N; e += 4) {
                    const float4 q = __ldg(reinterpret_cast<const float4 *>(s + e));
                    f[e] = q.x, f[e + 1] = q.y, f[e + 2] = q.z, f[e + 3] = q.w;
                }
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (e >= used) f[e] = 0.0f;
            } else {
#pragma unroll
                for (int e = 0; e < N; ++e) f[e] = e < used ? s[e] : 0.0f;
            }
        }
        split<N, kWeightParts<WT>>(f, w.p);
    }
    return w;
}

template <int WT, int N>
__device__ __forceinline__ Weights<WT, N> no_weights() {
    Weights<WT, N> w;
#pragma unroll
    for (int j = 0; j < kWeightParts<WT>; ++j)
#pragma unroll
        for (int e = 0; e < N / 2; ++e) w.p[j][e] = 0u;
    return w;
}

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

/* c += x w over 4 N contracted numbers, of which lane 4 g + q holds N
 * consecutive ones of tokens g (x0) and g + 8 (x1) and of weight row g: the
 * order of a contraction is free, so lane q's numbers 4 s .. 4 s + 3 stand in
 * the places that instruction s gives to lane q.  x?[part][pair]. */
template <int WT, int N>
__device__ __forceinline__ void multiply(float (&c)[4], const uint32_t (&x0)[3][N / 2], const uint32_t (&x1)[3][N / 2],
                                         const Weights<WT, N> &w) {
    constexpr int P = kWeightParts<WT>;
    __syncwarp();  // lanes may have loaded by different ways
#pragma unroll
    for (int sum = P + 1; sum >= 0; --sum)  // the smallest products first
#pragma unroll
        for (int j = P - 1; j >= 0; --j) {
            const int i = sum - j;
            if (i < 0 || i > 2 || (P == 3 && i == 2 && j == 2)) continue;
#pragma unroll
            for (int s = 0; s < N / 4; ++s)
                mma_bf16(c, x0[i][2 * s], x1[i][2 * s], x0[i][2 * s + 1], x1[i][2 * s + 1], w.p[j][2 * s],
                         w.p[j][2 * s + 1]);
        }
}

/* 8 numbers of x at p (valid of them exist) in three parts */
__device__ __forceinline__ void load_x(const float *p, int valid, bool vec, uint32_t (&x)[3][4]) {
    float f[8];
    if (vec && valid >= 8) {
        const float4 q0 = __ldg(reinterpret_cast<const float4 *>(p)), q1 = __ldg(reinterpret_cast<const float4 *>(p) + 1);
        f[0] = q0.x, f[1] = q0.y, f[2] = q0.z, f[3] = q0.w, f[4] = q1.x, f[5] = q1.y, f[6] = q1.z, f[7] = q1.w;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = e < valid ? __ldg(p + e) : 0.0f;
    }
    split<8, 3>(f, x);
}

/* ------------------------------------------------------------ the kernels */
/* An item: its adapter (-1: none), its number of tokens, and the tokens of a
 * lane's two rows of the instructions (g and g + 8; -1: none). */
struct LoraItem {
    int adapter, m, t0, t1;
};
__device__ __forceinline__ LoraItem lora_item(const LoraArgs &a, int k) {
    const int g = (threadIdx.x & 31) >> 2;
    LoraItem it{-1, 0, -1, -1};
    if (a.plan) {
        if (k >= a.plan->n) return it;
        const int first = a.plan->first[k];
        it.adapter = a.plan->adapter[k];
        it.m = min(a.plan->first[k + 1] - first, kLoraItem);
        if (g < it.m) it.t0 = a.plan->order[first + g];
        if (g + 8 < it.m) it.t1 = a.plan->order[first + g + 8];
    } else {
        uint32_t tokens;
        int items;
        it.adapter = warp_item(a, k, tokens, items);
        it.m = __popc(tokens);
        if (g < it.m) it.t0 = (int)__fns(tokens, 0, g + 1);
        if (g + 8 < it.m) it.t1 = (int)__fns(tokens, 0, g + 9);
    }
    return it;
}

/* One cluster per item (blockIdx.y) and 16 ranks (blockIdx.z): its CTAs' warps
 * take the columns in turns of 32, each turn's products are added up from 0 by
 * the matrix instructions and then to the warp's sums in fp32 (the
 * instructions cut what they add to), the warps' sums are added in their order
 * and the CTAs' in theirs.  An item's weights are 128 KB at rank 16 and 4096
 * columns; one CTA takes them in no faster than 6 us, so few items are spread
 * over clusters of up to eight. */
template <int WT>
__global__ void __launch_bounds__(kShrinkThreads) lora_shrink_kernel(const __grid_constant__ LoraArgs a) {
    constexpr int WARPS = kShrinkThreads / 32;
    constexpr int ES = WT == kHeadF32 ? 4 : 2;
    __shared__ float part[WARPS][kLoraItem][16];
    __shared__ float2 gather[kShrinkSplit][kLoraItem][8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3;
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the plan is there
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const LoraItem it = lora_item(a, blockIdx.y);
    if (it.adapter < 0) return;  // the whole cluster
    const cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
    auto begun = cluster.barrier_arrive();  // a CTA's shared memory is written by others once it has begun
    const int i = it.adapter, n = lora_rank(a, i), r0 = blockIdx.z * 16;
    float acc[2][4] = {};
    if (r0 < n) {
        const float *x0 = a.x + (size_t)max(it.t0, 0) * (size_t)a.ldx, *x1 = a.x + (size_t)max(it.t1, 0) * (size_t)a.ldx;
        const int ra = r0 + g, rb = ra + 8;
        const char *w = static_cast<const char *>(a.a) + (size_t)i * (size_t)a.stride_a * ES;
        const char *wa = w + (size_t)min(ra, n - 1) * (size_t)a.lda * ES, *wb = w + (size_t)min(rb, n - 1) * (size_t)a.lda * ES;
        const bool vec = a.vec_x && a.vec_a;
#pragma unroll 2
        for (int k0 = (blockIdx.x * WARPS + warp) * 32; k0 < a.cols; k0 += 32 * WARPS * gridDim.x) {
            const int k = k0 + 8 * q, left = a.cols - k;
            uint32_t p0[3][4] = {}, p1[3][4] = {};
            Weights<WT, 8> ba = no_weights<WT, 8>(), bb = no_weights<WT, 8>();
            if (vec && k0 + 32 <= a.cols) {
                if (ra < n) ba = load_weights<WT, 8>(wa + (size_t)k * ES, 8, 8, true);
                if (rb < n) bb = load_weights<WT, 8>(wb + (size_t)k * ES, 8, 8, true);
                if (it.t0 >= 0) load_x(x0 + k, 8, true, p0);
                if (it.t1 >= 0) load_x(x1 + k, 8, true, p1);
            } else if (left > 0) {
                if (ra < n) ba = load_weights<WT, 8>(wa + (size_t)k * ES, left, min(left, 8), false);
                if (rb < n) bb = load_weights<WT, 8>(wb + (size_t)k * ES, left, min(left, 8), false);
                if (it.t0 >= 0) load_x(x0 + k, left, false, p0);
                if (it.t1 >= 0) load_x(x1 + k, left, false, p1);
            }
            float c[2][4] = {};
            multiply<WT, 8>(c[0], p0, p1, ba);
            multiply<WT, 8>(c[1], p0, p1, bb);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                acc[0][e] = __fadd_rn(acc[0][e], c[0][e]);
                acc[1][e] = __fadd_rn(acc[1][e], c[1][e]);
            }
        }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        *reinterpret_cast<float2 *>(&part[warp][g][8 * h + 2 * q]) = make_float2(acc[h][0], acc[h][1]);
        *reinterpret_cast<float2 *>(&part[warp][g + 8][8 * h + 2 * q]) = make_float2(acc[h][2], acc[h][3]);
    }
    __syncthreads();
    /* two ranks of one token per thread; warp w has tokens 4 w .. 4 w + 3 */
    const int row = threadIdx.x >> 3, r = 2 * (threadIdx.x & 7);
    float u = 0.0f, v = 0.0f;
    if (threadIdx.x < kLoraItem * 8) {
#pragma unroll
        for (int k = 0; k < WARPS; ++k) {
            const float2 s = *reinterpret_cast<const float2 *>(&part[k][row][r]);
            u = __fadd_rn(u, s.x);
            v = __fadd_rn(v, s.y);
        }
    }
    cluster.barrier_wait(std::move(begun));
    if (gridDim.x > 1) {
        if (threadIdx.x < kLoraItem * 8)
            *cluster.map_shared_rank(&gather[blockIdx.x][row][r / 2], 0) = make_float2(u, v);
        cluster.sync();
        if (blockIdx.x) return;
        if (threadIdx.x < kLoraItem * 8) {
            u = v = 0.0f;
            for (int k = 0; k < (int)gridDim.x; ++k) {
                const float2 s = gather[k][row][r / 2];
                u = __fadd_rn(u, s.x);
                v = __fadd_rn(v, s.y);
            }
        }
    }
    if (threadIdx.x >= kLoraItem * 8) return;
    /* token `row` of the item is what lanes 4 (row % 8) hold as t0 or t1 */
    const int ta = __shfl_sync(kFull, it.t0, 4 * (row & 7)), tb = __shfl_sync(kFull, it.t1, 4 * (row & 7));
    const int t = row < 8 ? ta : tb;
    if (t < 0) return;
    if (a.scale) {
        const float s = a.scale[i];
        u = __fmul_rn(u, s);
        v = __fmul_rn(v, s);
    }
    if (r0 + r >= n) u = 0.0f;  // not even an infinite scale gives an unused rank a value
    if (r0 + r + 1 >= n) v = 0.0f;
#pragma unroll
    for (int k = 0; k < 3; ++k)
        *reinterpret_cast<uint32_t *>(a.low + ((size_t)t * 3 + k) * a.rank_pad + r0 + r) = take_parts(u, v);
}

/* N parts (8 or 4) of a token's low-rank numbers */
template <int N>
__device__ __forceinline__ void load_low(const LoraArgs &a, int t, int r, uint32_t (&x)[3][N / 2]) {
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        const uint16_t *p = a.low + ((size_t)t * 3 + k) * a.rank_pad + r;
        if (N == 8) {
            const uint4 v = *reinterpret_cast<const uint4 *>(p);
            x[k][0] = v.x, x[k][1] = v.y, x[k][N / 2 - 2] = v.z, x[k][N / 2 - 1] = v.w;
        } else {
            const uint2 v = *reinterpret_cast<const uint2 *>(p);
            x[k][0] = v.x, x[k][1] = v.y;
        }
    }
}

/* One item per blockIdx.y; the warps of its CTAs take 16 PAIRS rows of B_i at
 * a time.  N is the number of ranks a lane holds: 4 for ranks up to 16, else 8
 * (a group of 32 ranks at a time).  Column h of instruction j of a pair stands
 * for row 4 (h / 2) + 2 j + h % 2 of its 16, which gives lane q the four rows
 * 4 q .. 4 q + 3 of the result: 16 bytes of y. */
template <int WT, int N, int PAIRS>
__global__ void __launch_bounds__(kExpandThreads, 2) lora_expand_kernel(const __grid_constant__ LoraArgs a) {
    constexpr int ES = WT == kHeadF32 ? 4 : 2, ROWS = 16 * PAIRS;
    const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    const LoraItem it = lora_item(a, blockIdx.y);  // the kernel before let this one begin when the plan was there
    if (it.adapter < 0) {
        asm volatile("griddepcontrol.wait;" ::: "memory");  // no CTA ends before the kernel before
        return;
    }
    const int n = lora_rank(a, it.adapter);
    const bool full = a.vec_b && a.vec_y && n % N == 0;
    /* this lane's first row of B_i and ranks, and its tokens' rows of y */
    const char *w = static_cast<const char *>(a.b) +
                    ((size_t)it.adapter * (size_t)a.stride_b + (size_t)(4 * (g >> 1) + (g & 1)) * (size_t)a.ldb + N * q) * ES;
    float *y0 = a.y + (size_t)max(it.t0, 0) * (size_t)a.ldy + 4 * q, *y1 = a.y + (size_t)max(it.t1, 0) * (size_t)a.ldy + 4 * q;
    uint32_t x0[3][N / 2] = {}, x1[3][N / 2] = {};
    bool have = false;  // the low-rank numbers are there, and the first group of them in x0 and x1
    const int64_t step = (int64_t)gridDim.x * (kExpandThreads / 32) * ROWS;
    for (int64_t v0 = ((int64_t)blockIdx.x * (kExpandThreads / 32) + (threadIdx.x >> 5)) * ROWS; v0 < a.rows; v0 += step) {
        const bool inside = full && v0 + ROWS <= a.rows;
        const char *wv = w + (size_t)v0 * (size_t)a.ldb * ES;
        float4 o0[PAIRS], o1[PAIRS];
        if (inside) {
#pragma unroll
            for (int p = 0; p < PAIRS; ++p) {
                if (it.t0 >= 0) o0[p] = *reinterpret_cast<const float4 *>(y0 + v0 + 16 * p);
                if (it.t1 >= 0) o1[p] = *reinterpret_cast<const float4 *>(y1 + v0 + 16 * p);
            }
        }
        float c[PAIRS][2][4] = {};
        for (int r0 = 0; r0 < n; r0 += 4 * N) {
            const int r = r0 + N * q;
            Weights<WT, N> b[PAIRS][2];
#pragma unroll
            for (int p = 0; p < PAIRS; ++p)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const char *at = wv + ((size_t)(16 * p + 2 * j) * (size_t)a.ldb + r0) * ES;
                    b[p][j] = no_weights<WT, N>();
                    if (inside) {
                        if (r < n) b[p][j] = load_weights<WT, N>(at, N, N, true);
                    } else if (v0 + 16 * p + 4 * (g >> 1) + 2 * j + (g & 1) < a.rows && r < n) {
                        b[p][j] = load_weights<WT, N>(at, N, min(n - r, N), false);
                    }
                }
            if (!have) asm volatile("griddepcontrol.wait;" ::: "memory");
            if (!have || n > 4 * N) {
                if (it.t0 >= 0) load_low<N>(a, it.t0, r, x0);
                if (it.t1 >= 0) load_low<N>(a, it.t1, r, x1);
                have = true;
            }
#pragma unroll
            for (int p = 0; p < PAIRS; ++p)
#pragma unroll
                for (int j = 0; j < 2; ++j) multiply<WT, N>(c[p][j], x0, x1, b[p][j]);
        }
#pragma unroll
        for (int p = 0; p < PAIRS; ++p) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if ((h ? it.t1 : it.t0) < 0) continue;
                float *y = (h ? y1 : y0) + v0 + 16 * p;
                const float d[4] = {c[p][0][2 * h], c[p][0][2 * h + 1], c[p][1][2 * h], c[p][1][2 * h + 1]};
                if (inside) {
                    float4 o = h ? o1[p] : o0[p];
                    o.x = __fadd_rn(o.x, d[0]);
                    o.y = __fadd_rn(o.y, d[1]);
                    o.z = __fadd_rn(o.z, d[2]);
                    o.w = __fadd_rn(o.w, d[3]);
                    *reinterpret_cast<float4 *>(y) = o;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (v0 + 16 * p + 4 * q + e < a.rows) y[e] = __fadd_rn(y[e], d[e]);
                }
            }
        }
    }
    if (!have) asm volatile("griddepcontrol.wait;" ::: "memory");
}

}  // namespace noel
