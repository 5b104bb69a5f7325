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

namespace noel {

constexpr int kLoraMaxRank = 256;
constexpr int kLoraBatch = 2048;    // tokens of one pass over the adapters
constexpr int kLoraItem = 16;       // tokens of an item
constexpr int kLoraWarpBatch = 32;  // tokens up to which every warp finds the items by itself
constexpr int kShrinkThreads = 512;
constexpr int kExpandThreads = 256;
constexpr int kExpandRows = 64;     // rows of B_i of a warp's turn
constexpr int kPlanThreads = 1024;
constexpr int kPlanSlots = 4096;

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
__global__ void __launch_bounds__(kPlanThreads) lora_plan_kernel(const __grid_constant__ LoraArgs a) {
    __shared__ int key[kPlanSlots], count[kPlanSlots];
    __shared__ int wsum[kPlanThreads / 32], wtok[kPlanThreads / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    for (int s = tid; s < kPlanSlots; s += kPlanThreads) {
        key[s] = 0;
        count[s] = 0;
    }
    __syncthreads();
    constexpr int PER = kLoraBatch / kPlanThreads;
    int slot[PER], number[PER];
#pragma unroll
    for (int u = 0; u < PER; ++u) {
        const int t = u * kPlanThreads + tid;
        const int i = t < a.batch ? a.adapter[t] : -1;
        slot[u] = -1;
        if (i < 0 || i >= a.n) continue;
        uint32_t p = ((uint32_t)i * 0x9E3779B1u) >> 20;  // the top 12 bits: kPlanSlots
        for (int probe = 0; probe < kPlanSlots; ++probe) {  // at most half of the slots are taken
            const int prev = atomicCAS(&key[p], 0, i + 1);
            if (prev == 0 || prev == i + 1) break;
            p = (p + 1) % kPlanSlots;
        }
        slot[u] = (int)p;
        number[u] = atomicAdd(&count[p], 1);
    }
    __syncthreads();
    /* prefix sums over the slots, four to a thread: items and tokens */
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
#pragma unroll
        for (int j = 0; j < kWeightParts<WT>; ++j)
#pragma unroll
            for (int e = 0; e < N; e += 2) w.p[j][e / 2] = take_parts(f[e], f[e + 1]);
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
#pragma unroll
    for (int i = 0; i < 3; ++i)
#pragma unroll
        for (int e = 0; e < 8; e += 2) x[i][e / 2] = take_parts(f[e], f[e + 1]);
}

/* ------------------------------------------------------------ the kernels */
/* One CTA per item (blockIdx.x) and 16 ranks (blockIdx.y): the warps take the
 * columns in turns of 32, each turn's products are added up from 0 by the
 * matrix instructions and then to the warp's sums in fp32 (the instructions cut
 * what they add to), and the warps' sums are added in their order. */
template <int WT>
__global__ void __launch_bounds__(kShrinkThreads) lora_shrink_kernel(const __grid_constant__ LoraArgs a) {
    constexpr int WARPS = kShrinkThreads / 32;
    constexpr int ES = WT == kHeadF32 ? 4 : 2;
    __shared__ float part[WARPS][kLoraItem][16];
    __shared__ int tok[kLoraItem];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3;
    asm volatile("griddepcontrol.wait;" ::: "memory");               // the plan is there
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    int i, m;
    if (a.plan) {
        if ((int)blockIdx.x >= a.plan->n) return;
        i = a.plan->adapter[blockIdx.x];
        const int first = a.plan->first[blockIdx.x];
        m = min(a.plan->first[blockIdx.x + 1] - first, kLoraItem);
        if (threadIdx.x < kLoraItem) tok[threadIdx.x] = (int)threadIdx.x < m ? a.plan->order[first + threadIdx.x] : -1;
    } else {
        uint32_t tokens;
        int items;
        i = warp_item(a, blockIdx.x, tokens, items);
        if (i < 0) return;
        m = __popc(tokens);
        if (threadIdx.x < kLoraItem) tok[threadIdx.x] = (int)threadIdx.x < m ? (int)__fns(tokens, 0, threadIdx.x + 1) : -1;
    }
    __syncthreads();
    const int n = lora_rank(a, i), r0 = blockIdx.y * 16;
    float acc[2][4] = {};
    if (r0 < n) {
        const int t0 = tok[g], t1 = tok[g + 8];
        const float *x0 = a.x + (size_t)max(t0, 0) * (size_t)a.ldx, *x1 = a.x + (size_t)max(t1, 0) * (size_t)a.ldx;
        const char *w = static_cast<const char *>(a.a) + (size_t)i * (size_t)a.stride_a * ES;
        const int ra = r0 + g, rb = ra + 8;
#pragma unroll 2
        for (int k0 = warp * 32; k0 < a.cols; k0 += 32 * WARPS) {
            const int k = k0 + 8 * q, left = a.cols - k;
            uint32_t p0[3][4] = {}, p1[3][4] = {};
            if (t0 >= 0 && left > 0) load_x(x0 + k, left, a.vec_x, p0);
            if (t1 >= 0 && left > 0) load_x(x1 + k, left, a.vec_x, p1);
            const Weights<WT, 8> wa = ra < n && left > 0
                ? load_weights<WT, 8>(w + ((size_t)ra * (size_t)a.lda + k) * ES, left, min(left, 8), a.vec_a)
                : no_weights<WT, 8>();
            const Weights<WT, 8> wb = rb < n && left > 0
                ? load_weights<WT, 8>(w + ((size_t)rb * (size_t)a.lda + k) * ES, left, min(left, 8), a.vec_a)
                : no_weights<WT, 8>();
            float c[2][4] = {};
            multiply<WT, 8>(c[0], p0, p1, wa);
            multiply<WT, 8>(c[1], p0, p1, wb);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                acc[0][e] = __fadd_rn(acc[0][e], c[0][e]);
                acc[1][e] = __fadd_rn(acc[1][e], c[1][e]);
            }
        }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        part[warp][g][8 * h + 2 * q] = acc[h][0];
        part[warp][g][8 * h + 2 * q + 1] = acc[h][1];
        part[warp][g + 8][8 * h + 2 * q] = acc[h][2];
        part[warp][g + 8][8 * h + 2 * q + 1] = acc[h][3];
    }
    __syncthreads();
    /* two ranks of one token per thread */
    if (threadIdx.x < kLoraItem * 8) {
        const int row = threadIdx.x >> 3, r = 2 * (threadIdx.x & 7), t = tok[row];
        if (t >= 0) {
            float u = 0.0f, v = 0.0f;
#pragma unroll
            for (int k = 0; k < WARPS; ++k) {
                u = __fadd_rn(u, part[k][row][r]);
                v = __fadd_rn(v, part[k][row][r + 1]);
            }
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
    }
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

/* A warp's turn: 64 rows of B_i for one item.  N is the number of ranks a lane
 * holds: 4 for ranks up to 16, else 8 (a group of 32 ranks at a time). */
template <int WT, int N>
__global__ void __launch_bounds__(kExpandThreads, 2) lora_expand_kernel(const __grid_constant__ LoraArgs a) {
    constexpr int ES = WT == kHeadF32 ? 4 : 2, PAIRS = 2;  // 16 rows to a pair of instructions' columns
    const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the low-rank numbers are there
    int items;
    uint32_t tokens = 0u;
    if (a.plan) items = a.plan->n;
    else warp_item(a, 32, tokens, items);
    const int tiles = (a.rows + kExpandRows - 1) / kExpandRows;
    const int64_t turns = (int64_t)items * tiles, step = (int64_t)gridDim.x * (kExpandThreads / 32);
    for (int64_t u = ((int64_t)blockIdx.x * kExpandThreads + threadIdx.x) >> 5; u < turns; u += step) {
        const int item = (int)(u % items), v0 = (int)(u / items) * kExpandRows;
        int i, t0, t1;
        if (a.plan) {
            i = a.plan->adapter[item];
            const int first = a.plan->first[item], m = min(a.plan->first[item + 1] - first, kLoraItem);
            t0 = g < m ? a.plan->order[first + g] : -1;
            t1 = g + 8 < m ? a.plan->order[first + g + 8] : -1;
        } else {
            int all;
            i = warp_item(a, item, tokens, all);
            const int m = __popc(tokens);
            t0 = g < m ? (int)__fns(tokens, 0, g + 1) : -1;
            t1 = g + 8 < m ? (int)__fns(tokens, 0, g + 9) : -1;
        }
        const int n = lora_rank(a, i);
        const char *w = static_cast<const char *>(a.b) + (size_t)i * (size_t)a.stride_b * ES;
        float *y0 = a.y + (size_t)max(t0, 0) * (size_t)a.ldy, *y1 = a.y + (size_t)max(t1, 0) * (size_t)a.ldy;
#pragma unroll 1
        for (int b0 = v0; b0 < v0 + kExpandRows && b0 < a.rows; b0 += 16 * PAIRS) {
            float c[PAIRS][2][4] = {};
            for (int r0 = 0; r0 < n; r0 += 4 * N) {
                const int r = r0 + N * q;
                uint32_t x0[3][N / 2] = {}, x1[3][N / 2] = {};
                if (t0 >= 0) load_low<N>(a, t0, r, x0);
                if (t1 >= 0) load_low<N>(a, t1, r, x1);
#pragma unroll
                for (int p = 0; p < PAIRS; ++p)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        /* column h of instruction j stands for row 4 (h / 2) + 2 j + h % 2 of the 16, which
                         * gives lane q the four rows 4 q .. 4 q + 3 */
                        const int v = b0 + 16 * p + 4 * (g >> 1) + 2 * j + (g & 1);
                        const Weights<WT, N> b = v < a.rows && r < n
                            ? load_weights<WT, N>(w + ((size_t)v * (size_t)a.ldb + r) * ES, a.rank - r, min(n - r, N), a.vec_b)
                            : no_weights<WT, N>();
                        multiply<WT, N>(c[p][j], x0, x1, b);
                    }
            }
#pragma unroll
            for (int p = 0; p < PAIRS; ++p) {
                const int v = b0 + 16 * p + 4 * q;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if ((h ? t1 : t0) < 0) continue;
                    float *y = (h ? y1 : y0) + v;
                    const float d[4] = {c[p][0][2 * h], c[p][0][2 * h + 1], c[p][1][2 * h], c[p][1][2 * h + 1]};
                    if (a.vec_y && v + 4 <= a.rows) {
                        float4 o = *reinterpret_cast<const float4 *>(y);
                        o.x = __fadd_rn(o.x, d[0]);
                        o.y = __fadd_rn(o.y, d[1]);
                        o.z = __fadd_rn(o.z, d[2]);
                        o.w = __fadd_rn(o.w, d[3]);
                        *reinterpret_cast<float4 *>(y) = o;
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (v + e < a.rows) y[e] = __fadd_rn(y[e], d[e]);
                    }
                }
            }
        }
    }
}

}  // namespace noel
