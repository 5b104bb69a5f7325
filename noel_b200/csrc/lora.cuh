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
 *
 * Measured on the device, in a CUDA graph, at 152,064 rows x 4096 columns (and
 * as back-to-back calls from Python): one token at rank 16 in 7.4 us (14.5); 64
 * tokens with 64 bf16 adapters of rank 16 in 77 us (84; 399 MB, 5.2 TB/s); 256
 * tokens over eight fp16 adapters of ranks up to 32 in 73 us (78; 287 MB); 2048
 * tokens over four bf16 adapters of rank 64 in 510 us (556; 2.6 GB, 5.1 TB/s).
 * What bounds the second kernel: at rank 16 nothing alone, half of the issue
 * slots, 41 % of the matrix pipe and 5.2 TB/s of memory are busy; at rank 64
 * memory at 5.6 TB/s, with 36 % of the issue slots and 52 % of the matrix pipe.
 */
#pragma once

#include "lmhead.cuh"
#include "sector.cuh"

#include <cooperative_groups.h>

#include <utility>

namespace noel {

constexpr int kLoraMaxRank = 256;
constexpr int kLoraBatch = 2048;    // tokens of one pass over the adapters
constexpr int kLoraItem = 16;       // tokens of an item
constexpr int kLoraWarpBatch = 32;  // tokens up to which every warp finds the items by itself (one token: 9.0 -> 7.5 us)
constexpr int kShrinkThreads = 256;
constexpr int kExpandThreads = 256;
/* turns between asking the L2 for a line of y and copying it from there (2048 tokens at rank 64: 551 us without, 496,
 * 521 and 535 us at 1, 2 and 4) */
constexpr int kExpandFetch = 1;
/* turns of the GPU's CTA slots that the second kernel's work is cut into (64 adapters, 256 and 2048 tokens: 73, 75, 582
 * us at 2; 77, 75, 513 at 4; 81, 78, 560 at 6) */
constexpr int kExpandWaves = 4;

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
    int r_begin, r_count;  // ranks that the second kernel takes: some of many, or all
    LoraPlan *plan;  // NULL: every warp finds the items
    int staged;                      // bytes at a time that fill the second kernel's stages: 16, 4, or 0: not staged
    int vec_x, vec_a, vec_b, vec_y;  // rows start on 16 bytes (B with rank_pad 16: on 4 elements; y: 2 for 32 bytes)
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
/* N numbers in P parts, as bf16 pairs; of an infinity or NaN the second part is
 * a NaN */
template <int N, int P>
__device__ __forceinline__ void split_finite(float (&f)[N], uint32_t (&x)[P][N / 2]) {
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
}
/* the same, an infinity or NaN whole in its first part */
template <int N, int P>
__device__ __forceinline__ void split(float (&f)[N], uint32_t (&x)[P][N / 2]) {
    float odd = 0.0f;  // stays 0 unless a number is infinite or NaN
#pragma unroll
    for (int e = 0; e < N; ++e) odd = __fmaf_rn(f[e], 0.0f, odd);
    if (odd == 0.0f) {
        split_finite<N, P>(f, x);
    } else {
#pragma unroll
        for (int i = 0; i < P; ++i)
#pragma unroll
            for (int e = 0; e < N; e += 2) x[i][e / 2] = take_parts(f[e], f[e + 1]);
    }
}

template <int WT>
constexpr int kWeightParts = WT == kHeadBF16 ? 1 : WT == kHeadF16 ? 2 : 3;
template <int WT>
constexpr int kWeightBytes = WT == kHeadF32 ? 4 : 2;

/* N consecutive weights: as they lie in memory, and as bf16 pairs part by part */
template <int WT, int N>
struct Raw {
    uint32_t u[N * kWeightBytes<WT> / 4];
};
template <int WT, int N>
struct Weights {
    uint32_t p[kWeightParts<WT>][N / 2];
};

template <int WT, int N>
__device__ __forceinline__ Raw<WT, N> raw_zero() {
    Raw<WT, N> r;
#pragma unroll
    for (int e = 0; e < N * kWeightBytes<WT> / 4; ++e) r.u[e] = 0u;
    return r;
}
/* from 16-byte aligned memory (8 where there are 8 bytes) */
template <int WT, int N>
__device__ __forceinline__ Raw<WT, N> raw_load(const void *p) {
    Raw<WT, N> r;
    constexpr int WORDS = N * kWeightBytes<WT> / 4;
    if (WORDS == 2) {
        const uint2 q = __ldg(static_cast<const uint2 *>(p));
        r.u[0] = q.x, r.u[1] = q.y;
    } else {
#pragma unroll
        for (int e = 0; e < WORDS; e += 4) {
            const uint4 q = __ldg(static_cast<const uint4 *>(p) + e / 4);
            r.u[e] = q.x, r.u[e + 1] = q.y, r.u[(e + 2) % WORDS] = q.z, r.u[(e + 3) % WORDS] = q.w;
        }
    }
    return r;
}
/* every STRIDE-th from p on, one by one; those from the used-th on (counting all) are 0 */
template <int WT, int N, int STRIDE = 1>
__device__ __forceinline__ Raw<WT, N> raw_elements(const void *p, int used) {
    Raw<WT, N> r;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        if (WT == kHeadF32) {
            r.u[e % (N * kWeightBytes<WT> / 4)] = e * STRIDE < used ? __ldg(static_cast<const uint32_t *>(p) + e * STRIDE) : 0u;
        } else {
            const uint32_t h = e * STRIDE < used ? (uint32_t)__ldg(static_cast<const uint16_t *>(p) + e * STRIDE) : 0u;
            r.u[e / 2] = e & 1 ? r.u[e / 2] | h << 16 : h;
        }
    }
    return r;
}
template <int WT, int N>
__device__ __forceinline__ Weights<WT, N> weights(const Raw<WT, N> &r) {
    Weights<WT, N> w;
    if (WT == kHeadBF16) {
#pragma unroll
        for (int e = 0; e < N / 2; ++e) w.p[0][e] = r.u[e];
    } else {
        float f[N];
#pragma unroll
        for (int e = 0; e < N; ++e)
            f[e] = WT == kHeadF32 ? __uint_as_float(r.u[e % (N * kWeightBytes<WT> / 4)])
                                  : __half2float(__ushort_as_half((uint16_t)(r.u[e / 2] >> (16 * (e & 1)))));
        split_finite<N, kWeightParts<WT>>(f, w.p);  // an infinity comes out as a NaN
    }
    return w;
}

/* c = a b + c, or a b alone */
__device__ __forceinline__ void mma_bf16(float (&c)[4], bool from_zero, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
    if (from_zero)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%10, %10, %10, %10};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

/* c (+)= x w over 4 N contracted numbers, of which lane 4 g + q holds N
 * consecutive ones of tokens g (x0) and g + 8 (x1) and of weight row g: the
 * order of a contraction is free, so lane q's numbers 4 s .. 4 s + 3 stand in
 * the places that instruction s gives to lane q.  x?[part][pair]. */
template <int WT, int N>
__device__ __forceinline__ void multiply(float (&c)[4], bool from_zero, const uint32_t (&x0)[3][N / 2],
                                         const uint32_t (&x1)[3][N / 2], const Weights<WT, N> &w) {
    constexpr int P = kWeightParts<WT>;
#pragma unroll
    for (int sum = P + 1; sum >= 0; --sum)  // the smallest products first
#pragma unroll
        for (int j = P - 1; j >= 0; --j) {
            const int i = sum - j;
            if (i < 0 || i > 2 || (P == 3 && i == 2 && j == 2)) continue;
#pragma unroll
            for (int s = 0; s < N / 4; ++s) {
                const bool first = s == 0 && (P == 3 ? sum == 3 && j == 2 : sum == P + 1);
                mma_bf16(c, from_zero && first, x0[i][2 * s], x1[i][2 * s], x0[i][2 * s + 1], x1[i][2 * s + 1],
                         w.p[j][2 * s], w.p[j][2 * s + 1]);
            }
        }
}

/* 8 numbers of x */
struct RawX {
    float f[8];
};
__device__ __forceinline__ RawX x_load(const float *p) {
    const float4 a = __ldg(reinterpret_cast<const float4 *>(p)), b = __ldg(reinterpret_cast<const float4 *>(p) + 1);
    return {{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
}
template <int STRIDE>
__device__ __forceinline__ RawX x_elements(const float *p, int used) {
    RawX r;
#pragma unroll
    for (int e = 0; e < 8; ++e) r.f[e] = e * STRIDE < used ? __ldg(p + e * STRIDE) : 0.0f;
    return r;
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

/* One cluster per item (blockIdx.y) and 8 TILES ranks (blockIdx.z).  The
 * columns are taken 32 at a time (a block), a block's products are added up
 * from 0 by the matrix instructions and then to a sum in fp32 (the instructions
 * cut what they add to).  Few items are spread over clusters of up to eight
 * CTAs: one CTA alone takes an item's weights (128 KB at rank 16 and 4096
 * columns) in at its own pace (the two kernels on the device: one token 12.3 us
 * with one CTA, 7.6 with eight; 64 adapters 86 with one, 77 with four).
 *
 * The order of the additions does not depend on that split.  Block k belongs to
 * sum k % 64, a number of the bits 5 .. 0.  The sums that differ in bits 5 and 4
 * only are added in their order, the results that differ in bit 3 as a pair,
 * those in bit 2, in bit 1 and in bit 0.  The CTA's number stands for the lowest
 * bits, the warp's for the three above, and a warp makes the sums of all values
 * of the rest in turn.  (Eight CTAs whatever the number of items: 2048 tokens at
 * rank 64 534 against 509 us.  One CTA where two are taken: 75 adapters x 32,000
 * rows 42.5 against 37.1.) */
template <int WT, int TILES, int CTAS>
__global__ void __launch_bounds__(kShrinkThreads, TILES == 2 || WT == kHeadBF16 ? 2 : 1) lora_shrink_kernel(const __grid_constant__ LoraArgs a) {
    constexpr int WARPS = kShrinkThreads / 32, RANKS = 8 * TILES;
    constexpr int ES = kWeightBytes<WT>;
    constexpr int SUMS = 8 / CTAS, SETS = CTAS == 1 || CTAS == 4 ? 2 : 1;  // sums of a warp, and results it keeps apart
    static_assert(WARPS == 8 && SUMS * CTAS == 8, "64 sums");
    __shared__ float part[SETS][WARPS][kLoraItem][RANKS];
    __shared__ float2 gather[CTAS][kLoraItem][RANKS / 2];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3;
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the plan is there
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const LoraItem it = lora_item(a, blockIdx.y);
    if (it.adapter < 0) return;  // the whole cluster
    const cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
    auto begun = cluster.barrier_arrive();  // a CTA's shared memory is written by others once it has begun
    const int i = it.adapter, n = lora_rank(a, i), r0 = blockIdx.z * RANKS;
    /* the warp's result in its place in part, or added to what is there */
    auto keep = [&](int set, bool add, const float (&v)[TILES][4]) {
#pragma unroll
        for (int h = 0; h < TILES; ++h)
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                float2 *to = reinterpret_cast<float2 *>(&part[set][warp][g + 4 * e][8 * h + 2 * q]);
                const float2 o = add ? *to : make_float2(0.0f, 0.0f);
                *to = make_float2(__fadd_rn(o.x, v[h][e]), __fadd_rn(o.y, v[h][e + 1]));
            }
    };
    if (r0 < n) {
        const float *x0 = a.x + (size_t)max(it.t0, 0) * (size_t)a.ldx, *x1 = a.x + (size_t)max(it.t1, 0) * (size_t)a.ldx;
        const char *w = static_cast<const char *>(a.a) + (size_t)i * (size_t)a.stride_a * ES;
        const char *wr[TILES];
#pragma unroll
        for (int h = 0; h < TILES; ++h) wr[h] = w + (size_t)min(r0 + 8 * h + g, n - 1) * (size_t)a.lda * ES;
        const bool both = it.m > 8;
        const int whole = a.vec_x && a.vec_a ? a.cols / 32 : 0;
        uint32_t p0[3][4] = {}, p1[3][4] = {};
        Raw<WT, 8> b[TILES];
        RawX f0, f1;
        /* a lane's eight of the 32 columns: consecutive ones where rows start on 16 bytes, else every fourth, so
         * that the lanes of a row read side by side */
        auto load = [&](int k0) {
            if (k0 < whole) {
                const int k = 32 * k0 + 8 * q;
#pragma unroll
                for (int h = 0; h < TILES; ++h)
                    if (r0 + 8 * h + g < n) b[h] = raw_load<WT, 8>(wr[h] + (size_t)k * ES);
                if (it.t0 >= 0) f0 = x_load(x0 + k);
                if (both && it.t1 >= 0) f1 = x_load(x1 + k);
            } else {
                const int k = 32 * k0 + q, left = a.cols - k;
#pragma unroll
                for (int h = 0; h < TILES; ++h)
                    if (r0 + 8 * h + g < n) b[h] = raw_elements<WT, 8, 4>(wr[h] + (size_t)k * ES, left);
                if (it.t0 >= 0) f0 = x_elements<4>(x0 + k, left);
                if (both && it.t1 >= 0) f1 = x_elements<4>(x1 + k, left);
            }
        };
#pragma unroll
        for (int h = 0; h < TILES; ++h) b[h] = raw_zero<WT, 8>();
        const int blocks = (a.cols + 31) / 32;
        /* the block to load next, and which of this warp's sums it belongs to: alone, a CTA's warp makes the four
         * sums of bit 3 clear before the others */
        int at = 0, k0 = warp * CTAS + blockIdx.x;
        const int first = k0;
        auto skip = [&] {
            while (k0 >= blocks && ++at < SUMS)
                k0 = first + (CTAS == 1 ? 2 * (at & 3) + (at >> 2) : at) * (WARPS * CTAS);
        };
        skip();
        if (at < SUMS) load(k0);
#pragma unroll 1
        for (int sum = 0; sum < SUMS; ++sum) {
            float acc[TILES][4] = {};
            while (at == sum) {  // the next block's numbers are on their way while this one's are multiplied
                Weights<WT, 8> w8[TILES];
#pragma unroll
                for (int h = 0; h < TILES; ++h) w8[h] = weights<WT, 8>(b[h]);
                if (it.t0 >= 0) split<8, 3>(f0.f, p0);
                if (it.t1 >= 0) split<8, 3>(f1.f, p1);
                k0 += 8 * WARPS;
                skip();
                if (at < SUMS) load(k0);
                __syncwarp();
#pragma unroll
                for (int h = 0; h < TILES; ++h) {
                    float c[4];
                    multiply<WT, 8>(c, true, p0, p1, w8[h]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[h][e] = __fadd_rn(acc[h][e], c[e]);
                }
            }
            if (CTAS == 1) keep(sum >> 2, sum & 3, acc);
            else if (CTAS == 4) keep(sum, false, acc);
            else keep(0, sum > 0, acc);
        }
    } else {
        const float none[TILES][4] = {};
#pragma unroll
        for (int k = 0; k < SETS; ++k) keep(k, false, none);
    }
    __syncthreads();
    /* two ranks of one token per thread: token `row` of the item */
    constexpr int PER_ROW = RANKS / 2, USED = kLoraItem * PER_ROW;
    static_assert(USED <= kShrinkThreads, "a thread for every two ranks");
    const int row = threadIdx.x / PER_ROW, r = 2 * (threadIdx.x % PER_ROW);
    auto number = [&](int set, int k) { return *reinterpret_cast<const float2 *>(&part[set][k][row][r]); };
    auto plus = [](float2 a, float2 b) { return make_float2(__fadd_rn(a.x, b.x), __fadd_rn(a.y, b.y)); };
    /* four in their order, from 0 as where a warp has added them */
    auto row_of = [&](float2 a0, float2 a1, float2 a2, float2 a3) {
        return plus(plus(plus(plus(make_float2(0.0f, 0.0f), a0), a1), a2), a3);
    };
    float2 s = make_float2(0.0f, 0.0f);
    if (threadIdx.x < USED) {
        if (CTAS == 8) {  // the warp's number is bits 5 .. 3
            s = plus(row_of(number(0, 0), number(0, 2), number(0, 4), number(0, 6)),
                     row_of(number(0, 1), number(0, 3), number(0, 5), number(0, 7)));
        } else if (CTAS == 4) {  // the set bit 5, the warp's number bits 4 .. 2
            auto bit3 = [&](int w) {
                return row_of(number(0, w), number(0, w + 4), number(1 % SETS, w), number(1 % SETS, w + 4));
            };
            s = plus(plus(bit3(0), bit3(2)), plus(bit3(1), bit3(3)));
        } else {  // bits 3 .. 1; alone, the set bit 3 and the warp's number bits 2 .. 0
            auto one = [&](int w) { return CTAS == 1 ? plus(number(0, w), number(1 % SETS, w)) : number(0, w); };
            auto pair = [&](int w) { return plus(one(w), one(w + 4)); };
            s = plus(plus(pair(0), pair(2)), plus(pair(1), pair(3)));
        }
    }
    cluster.barrier_wait(std::move(begun));
    if (CTAS > 1) {
        if (threadIdx.x < USED) *cluster.map_shared_rank(&gather[blockIdx.x][row][r / 2], 0) = s;
        cluster.sync();
        if (blockIdx.x) return;
        if (threadIdx.x < USED) {
            auto from = [&](int c) { return gather[c % CTAS][row][r / 2]; };
            auto four = [&](int c) { return CTAS == 8 ? plus(from(c), from(c + 4)) : from(c); };
            auto two = [&](int c) { return CTAS >= 4 ? plus(four(c), four(c + 2)) : from(c); };
            s = plus(two(0), two(1));
        }
    }
    float u = s.x, v = s.y;
    if (threadIdx.x >= USED) return;  // whole warps
    /* the token is what lanes 4 (row % 8) hold as t0 or t1 */
    const int ta = __shfl_sync(kFull, it.t0, 4 * (row & 7)), tb = __shfl_sync(kFull, it.t1, 4 * (row & 7));
    const int t = row < 8 ? ta : tb;
    if (t < 0) return;
    if (a.scale) {
        u = __fmul_rn(u, a.scale[i]);
        v = __fmul_rn(v, a.scale[i]);
    }
    if (r0 + r >= n) u = 0.0f;  // not even an infinite scale gives an unused rank a value
    if (r0 + r + 1 >= n) v = 0.0f;
#pragma unroll
    for (int k = 0; k < 3; ++k)
        *reinterpret_cast<uint32_t *>(a.low + ((size_t)t * 3 + k) * a.rank_pad + r0 + r) = take_parts(u, v);
}

/* N parts (8 or 4) of a token's low-rank numbers, of the ranks from r_begin on */
template <int N>
__device__ __forceinline__ void load_low(const LoraArgs &a, int t, int r, uint32_t (&x)[3][N / 2]) {
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        const uint16_t *p = a.low + ((size_t)t * 3 + k) * a.rank_pad + a.r_begin + r;
        if (N == 8) {
            const uint4 v = *reinterpret_cast<const uint4 *>(p);
            x[k][0] = v.x, x[k][1] = v.y, x[k][N / 2 - 2] = v.z, x[k][N / 2 - 1] = v.w;
        } else {
            const uint2 v = *reinterpret_cast<const uint2 *>(p);
            x[k][0] = v.x, x[k][1] = v.y;
        }
    }
}

/* What a warp of the second kernel knows: its item, and for this lane the first
 * weights of the row that it holds in instruction 0, the bytes from there to
 * its row in instruction 1, and its tokens' rows of y.
 *
 * A warp takes 32 rows of B_i at a time, four instructions wide.  Column h of
 * instruction j stands for row 8 (h / 2) + 2 j + h % 2 of the 32, which gives
 * lane q the eight rows 8 q .. 8 q + 7 of the result: 32 bytes of y, a line for
 * the four lanes of a token.  Where rows of y do not start on 16 bytes it
 * stands for row 8 j + h instead, and y goes by element. */
template <int WT>
struct ExpandLane {
    LoraItem it;
    int n;  // the adapter's ranks among those that are taken
    bool wide;
    const char *b, *w;
    size_t pitch, next;
    float *y0, *y1;
    __device__ __forceinline__ ExpandLane(const LoraArgs &a, const LoraItem &item, int N) : it(item) {
        const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
        constexpr int ES = kWeightBytes<WT>;
        n = min(max(lora_rank(a, it.adapter) - a.r_begin, 0), a.r_count);
        wide = a.vec_y != 0;
        b = static_cast<const char *>(a.b) + ((size_t)it.adapter * (size_t)a.stride_b + a.r_begin) * ES;
        pitch = (size_t)a.ldb * ES;
        w = b + (size_t)(wide ? 8 * (g >> 1) + (g & 1) : g) * pitch + (size_t)(N * q) * ES;
        next = (wide ? 2 : 8) * pitch;
        y0 = a.y + (size_t)max(it.t0, 0) * (size_t)a.ldy;
        y1 = a.y + (size_t)max(it.t1, 0) * (size_t)a.ldy;
    }
};

/* 32 rows from v0 on, any alignment, sizes and end; the sums are those of the
 * kernel below, bit for bit: up to 4 N G ranks by matrix instructions from 0 on,
 * and each such sum added to y in fp32 */
template <int WT, int N, int G>
__device__ __forceinline__ void expand_any(const LoraArgs &a, const ExpandLane<WT> &l, int64_t v0) {
    const int lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
    if (l.n == 0) return;
    float y[4][4] = {}, c[4][4] = {};
    auto each = [&](auto what) {  // number k of instruction j's result and its place in y
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            const int j = k >> 2, h = k >> 1 & 1, b = k & 1;
            const int64_t v = v0 + (l.wide ? 8 * q + 2 * j + b : 8 * j + 2 * q + b);
            if ((h ? l.it.t1 : l.it.t0) >= 0 && v < a.rows) what(y[j][2 * h + b], (h ? l.y1 : l.y0) + v);
        }
    };
    each([](float &f, float *p) { f = *p; });
    uint32_t x0[3][N / 2] = {}, x1[3][N / 2] = {};
    for (int r0 = 0; r0 < l.n; r0 += 4 * N) {
        const int r = r0 + N * q;
        const bool last = r0 / (4 * N) % G == G - 1 || r0 + 4 * N >= l.n;  // of a sum
        if (l.it.t0 >= 0) load_low<N>(a, l.it.t0, r, x0);
        if (l.it.t1 >= 0) load_low<N>(a, l.it.t1, r, x1);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t v = v0 + (l.wide ? 8 * (g >> 1) + 2 * j + (g & 1) : 8 * j + g);
            Raw<WT, N> b = raw_zero<WT, N>();
            if (v < a.rows && r < l.n) {
                const char *p = l.w + (size_t)v0 * l.pitch + j * l.next + (size_t)r0 * kWeightBytes<WT>;
                if (a.vec_b && r + N <= l.n) b = raw_load<WT, N>(p);
                else b = raw_elements<WT, N>(p, l.n - r);
            }
            const Weights<WT, N> wb = weights<WT, N>(b);
            __syncwarp();
            multiply<WT, N>(c[j], false, x0, x1, wb);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (!last) continue;
                y[j][e] = __fadd_rn(y[j][e], c[j][e]);
                c[j][e] = 0.0f;
            }
        }
    }
    each([](float &f, float *p) { *p = f; });
}

/* The second kernel for arrays that the one below cannot take (rows of B_i that
 * start on 2 bytes): one item per blockIdx.y, a warp its 32
 * rows at a time, y on its way while the products are formed (100 tokens x 50,001
 * rows at rank 33: 126 -> 55 us).  Where both could, without that, it took 11.3
 * us for one token and 207 for 64 adapters against 7.5 and 77. */
template <int WT, int N, int G>
__global__ void __launch_bounds__(kExpandThreads) lora_expand_any_kernel(const __grid_constant__ LoraArgs a) {
    const LoraItem it = lora_item(a, blockIdx.y);  // the kernel before let this one begin when the plan was there
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (it.adapter < 0) return;
    const ExpandLane<WT> l(a, it, N);
    const int64_t step = (int64_t)gridDim.x * (kExpandThreads / 32) * 32;
    for (int64_t v0 = ((int64_t)blockIdx.x * (kExpandThreads / 32) + (threadIdx.x >> 5)) * 32; v0 < a.rows; v0 += step)
        expand_any<WT, N, G>(a, l, v0);
}

__device__ __forceinline__ void prefetch_l2(const void *p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }
/* bytes of src and zeros up to 4 or 16 */
__device__ __forceinline__ void cp_async4_at(uint32_t dst, const void *src, uint32_t bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async16_at(uint32_t dst, const void *src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

/* Bytes of one of a warp's stages: 32 rows of B_i (64 bytes more after every eight where a row is 32 bytes), then a line
 * of y for each of 16 tokens. */
__host__ __device__ constexpr int expand_stage_bytes(int ranks, int es) {
    return 32 * ranks * es + (ranks * es == 32 ? 256 : 0) + kLoraItem * 128;
}

/* The second kernel: one item per blockIdx.y.  Every warp has D stages of
 * shared memory, which cp.async fills with the 32 rows of B_i and the lines of
 * y of its turns to come: D - 1 turns are on their way while one is
 * multiplied, and none needs a barrier of the CTA.  The kernel begins while
 * the one before still runs, and its first stages are on their way until that
 * is done.  Rows lie in shared memory with their 16-byte pieces exchanged so
 * that the eight lanes of a quarter warp read eight different ones.
 *
 * N is the number of ranks a lane holds: 4 for ranks up to 16, else 8 (a group
 * of 32 ranks at a time).  A launch takes up to 4 N G ranks, whose low-rank
 * numbers stay in registers; adapters of more ranks take several launches.  The
 * ranks of a launch are one chain of matrix instructions, which cut where fp32
 * rounds: 12 steps (fp16 weights 24), less than the 63 roundings of a
 * sum in fp32 may be off by.  (Each 32 ranks from 0 and added in fp32: 2048
 * tokens at rank 64 531 -> 600 us.)
 * (All ranks in one launch, with two stages and their numbers read again every
 * turn: 512 tokens at rank 128 522 us against 281, 16 adapters 180 against 124.)  WIDE: rows of y and of B_i start on
 * 16 bytes.  Without it rows of y start anywhere: their 32 numbers are copied
 * 4 bytes at a time, and go back through the stage so that a store writes a
 * token's 32 numbers side by side; and so are rows of B_i that do not start on
 * 16 bytes but on 4 (aligned rows taken that way: 97 instead of 77 us for 64
 * adapters; unaligned ones by plain loads: 324 instead of 191 us for 651 tokens
 * x 138,974).  Ranks up to 16 held as if they were 32: 104 instead of 77 us. */
template <int WT, int N, int G, int D, bool WIDE>
__global__ void __launch_bounds__(kExpandThreads, 2) lora_expand_kernel(const __grid_constant__ LoraArgs a) {
    extern __shared__ __align__(128) unsigned char lora_smem[];
    constexpr int ES = kWeightBytes<WT>, ROWS = 32, WARPS = kExpandThreads / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3;
    const LoraItem it = lora_item(a, blockIdx.y);  // the kernel before let this one begin when the plan was there
    const int64_t first = ((int64_t)blockIdx.x * WARPS + warp) * ROWS, step = (int64_t)gridDim.x * WARPS * ROWS;
    if (it.adapter < 0 || first >= a.rows) {
        asm volatile("griddepcontrol.wait;" ::: "memory");  // no warp ends before the kernel before
        return;
    }
    const ExpandLane<WT> l(a, it, N);
    if (l.n == 0) {
        asm volatile("griddepcontrol.wait;" ::: "memory");
        return;
    }
    constexpr int row_bytes = 4 * N * G * ES, stage_bytes = expand_stage_bytes(4 * N * G, ES);
    constexpr int pad8 = row_bytes == 32 ? 64 : 0, y_at = 32 * row_bytes + 4 * pad8;
    constexpr int swap = ES == 2 ? (row_bytes % 128 == 0 ? 4 : 0) : (N == 8 ? 1 : 0);  // of odd rows' pieces
    unsigned char *mem = lora_smem + warp * D * stage_bytes;
    /* how the lanes share a copy of 32 rows: `share` of them a row, in as many rounds; what lies past the adapter's
     * rank is filled with zeros */
    constexpr int share = row_bytes / 16, c_rows = 32 / share;
    const int c_row = lane / share, c_piece = lane % share;
    /* rows side by side: a turn's addresses differ by constants (2048 tokens at rank 64 without a pause: 586 -> 576 us;
     * no gain at rank 16, where a turn has two copies) */
    const bool tight = N == 8 && l.pitch == (size_t)row_bytes;
    const uint32_t c_bytes = (uint32_t)min(max(l.n * ES - c_piece * 16, 0), 16);
    const char *b_from = l.b + (size_t)(first + c_row) * l.pitch + (c_bytes ? c_piece << 4 : 0);
    constexpr int W4 = row_bytes / 4;
    const char *b_from4 = l.b + (size_t)(first + lane / W4) * l.pitch + (4 * (lane % W4) < l.n * ES ? 4 * (lane % W4) : 0);
    const size_t b_round = (size_t)c_rows * l.pitch, b_step = (size_t)step * l.pitch;
    const uint32_t mem_s = (uint32_t)__cvta_generic_to_shared(mem);
    const uint32_t b_to = c_row * row_bytes + (c_row >> 3) * pad8 + ((c_piece ^ (c_row & 1 ? swap : 0)) << 4);
    const uint32_t b_to_round = c_rows * row_bytes + (c_rows >> 3) * pad8;  // c_rows is even: rows keep their oddness
    const float *y_from[kLoraItem / 4];  // this lane's piece of a token's line, four tokens at a time
#pragma unroll
    for (int p = 0; p < kLoraItem / 4; ++p) {
        const int tk = 4 * p + (lane >> 3);
        const int ta = __shfl_sync(kFull, it.t0, 4 * (tk & 7)), tb = __shfl_sync(kFull, it.t1, 4 * (tk & 7));
        const int t = tk < 8 ? ta : tb;
        y_from[p] = a.y + (size_t)max(t, 0) * (size_t)a.ldy + first + 4 * (lane & 7);
    }
    /* without WIDE: the lane's number of the tokens' lines, their rows' places in y, and where number `lane` of
     * token k lies in a stage */
    const float *y_lane = a.y + first + lane;
    __shared__ int64_t y_off[WIDE ? 1 : WARPS][kLoraItem];
    auto line_of = [&](int k) { return y_at + k * 128 + (((lane >> 2) ^ (k & 1)) << 4) + ((lane & 3) << 2); };
    if (!WIDE) {
        const int ta = __shfl_sync(kFull, it.t0, 4 * (lane & 7)), tb = __shfl_sync(kFull, it.t1, 4 * (lane & 7));
        if (lane < kLoraItem) y_off[warp][lane] = (int64_t)max(lane < 8 ? ta : tb, 0) * a.ldy;
        __syncwarp();
    }
    const uint32_t y_to = y_at + (lane >> 3) * 128 + (((lane & 7) ^ (lane >> 3 & 1)) << 4);
    const int turns = (int)((a.rows - ROWS - first + step) / step);  // whole ones
    int ahead = 0;  // the next turn to bring
    /* one lane per token asks the L2 for that token's line kExpandFetch turns before it is copied from there */
    const float *y_fetch;
    {
        const int ta = __shfl_sync(kFull, it.t0, 4 * (lane & 7)), tb = __shfl_sync(kFull, it.t1, 4 * (lane & 7));
        const int t = lane < 8 ? ta : tb;
        y_fetch = a.y + (size_t)max(t, 0) * (size_t)a.ldy + first + kExpandFetch * step;
    }
    auto issue = [&](int stage) {
        if (ahead < turns) {
            const uint32_t to = mem_s + stage * stage_bytes;
            if (!WIDE && a.staged == 4) {  // rows of B_i that start on 4 bytes only
                constexpr int PER = W4 < 32 ? 32 / W4 : 1;  // rows a round
                const int word = lane % W4;
                const char *src = b_from4;
                const uint32_t bytes = (uint32_t)min(max(l.n * ES - 4 * word, 0), 4);
                for (int r = lane / W4; r < ROWS; r += PER, src += PER * l.pitch)
                    cp_async4_at(to + r * row_bytes + (r >> 3) * pad8 + ((word >> 2 ^ (r & 1 ? swap : 0)) << 4) + (word & 3) * 4,
                                 src, bytes);
                b_from4 += b_step;
            } else if (tight) {
#pragma unroll
                for (int r = 0; r < share; ++r)
                    cp_async16_at(to + b_to + r * b_to_round, b_from + r * (c_rows * row_bytes), c_bytes);
            } else {
                const char *src = b_from;
#pragma unroll
                for (int r = 0; r < share; ++r, src += b_round) cp_async16_at(to + b_to + r * b_to_round, src, c_bytes);
            }
            if (!WIDE) {
                for (int k = 0; k < it.m; ++k)
                    cp_async4_at(to + line_of(k), y_lane + y_off[warp][k], 4u);
                y_lane += step;
            }
#pragma unroll
            for (int p = 0; p < kLoraItem / 4; ++p) {
                if (!WIDE || 4 * p >= it.m) break;
                if (4 * p + (lane >> 3) < it.m) cp_async16_at(to + y_to + 512 * p, y_from[p], 16u);
                y_from[p] += step;
            }
            if (lane < it.m && ahead + kExpandFetch < turns) prefetch_l2(y_fetch);
            y_fetch += step;
            b_from += b_step;
            ++ahead;
        }
        cp_async_commit();
    };
#pragma unroll
    for (int s = 0; s < D - 1; ++s) issue(s);
    uint32_t x0[G][3][N / 2] = {}, x1[G][3][N / 2] = {};
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the low-rank numbers are there
#pragma unroll
    for (int k = 0; k < G; ++k) {
        if (k * 4 * N >= l.n) break;
        if (it.t0 >= 0) load_low<N>(a, it.t0, k * 4 * N + N * q, x0[k]);
        if (it.t1 >= 0) load_low<N>(a, it.t1, k * 4 * N + N * q, x1[k]);
    }
    /* where this lane's row of instruction 0 lies in a stage and what instruction j adds, its piece there, and its
     * lines of y */
    const int w_at = (8 * (g >> 1) + (g & 1)) * row_bytes + (g >> 1) * pad8, w_next = 2 * row_bytes;
    const int w_swap = g & 1 ? swap : 0;
    const int line0 = y_at + g * 128 + ((2 * q ^ (g & 1)) << 4), line1 = y_at + g * 128 + ((2 * q + 1 ^ (g & 1)) << 4);
    float *y0 = l.y0 + first + 8 * q, *y1 = l.y1 + first + 8 * q, *y_back = a.y + first + lane;
    const bool both = it.m > 8, line = a.vec_y == 2;
    int st = 0;
    for (int turn = 0; turn < turns; ++turn, y0 += step, y1 += step, y_back += step, st = st + 1 == D ? 0 : st + 1) {
        cp_async_wait<D - 2>();
        __syncwarp();  // stage st has landed for every lane, and no lane still reads the one before it
        issue(st == 0 ? D - 1 : st - 1);
        unsigned char *from = mem + st * stage_bytes;
        float c[4][4];
        auto group = [&](int k, bool from_zero, const uint32_t (&u0)[3][N / 2], const uint32_t (&u1)[3][N / 2]) {
            const int r = k * 4 * N + N * q;
            const unsigned char *row = from + w_at;
#pragma unroll
            for (int j = 0; j < 4; ++j, row += w_next) {
                Raw<WT, N> b;
                if (N * ES == 8) {
                    const uint2 v = *reinterpret_cast<const uint2 *>(row + r * ES);
                    b.u[0] = v.x, b.u[1] = v.y;
                } else {
#pragma unroll
                    for (int e = 0; e < N * ES / 16; ++e) {
                        const uint4 v = *reinterpret_cast<const uint4 *>(row + ((((r * ES >> 4) + e) ^ w_swap) << 4));
                        constexpr int WORDS = N * ES / 4;
                        b.u[4 * e] = v.x, b.u[4 * e + 1] = v.y, b.u[(4 * e + 2) % WORDS] = v.z, b.u[(4 * e + 3) % WORDS] = v.w;
                    }
                }
                multiply<WT, N>(c[j], from_zero, u0, u1, weights<WT, N>(b));
            }
        };
        group(0, true, x0[0], x1[0]);
        if (G > 1 && 4 * N < l.n) group(1, false, x0[G - 1], x1[G - 1]);
        auto add = [&](int h, float *y) {
            float4 *at0 = reinterpret_cast<float4 *>(from + line0 + 1024 * h);
            float4 *at1 = reinterpret_cast<float4 *>(from + line1 + 1024 * h);
            const float4 o = *at0, p = *at1;
            const float f[8] = {o.x, o.y, o.z, o.w, p.x, p.y, p.z, p.w};
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = __fadd_rn(f[e], c[e / 2][2 * h + (e & 1)]);
            if (!WIDE) {
                *at0 = make_float4(v[0], v[1], v[2], v[3]);
                *at1 = make_float4(v[4], v[5], v[6], v[7]);
                return;
            }
            Sector s;
#pragma unroll
            for (int e = 0; e < 8; ++e) s.u[e] = __float_as_uint(v[e]);
            if (line) sector_store(y, s);
            else sector_store16(y, s);
        };
        if (it.t0 >= 0) add(0, y0);
        if (both && it.t1 >= 0) add(1, y1);
        if (!WIDE) {
            __syncwarp();
            for (int k = 0; k < it.m; ++k) y_back[y_off[warp][k]] = *reinterpret_cast<const float *>(from + line_of(k));
        }
    }
    if (first + turns * step < a.rows) expand_any<WT, N, G>(a, l, first + turns * step);  // the last rows
}

}  // namespace noel
