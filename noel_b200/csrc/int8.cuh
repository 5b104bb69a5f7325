/*
 * Projections in 8-bit integers: the cast of tokens with a scale for each,
 * and the product with weights that have a scale for each output channel,
 *   y[t][v] = a_scale[t] * w_scale[v] * sum_d a[t][d] * w[v][d].
 * Sums are exact 32-bit integers (tcgen05.mma kind::i8), so a result does
 * not depend on tiles, on their order or on the rest of the batch.
 */
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <stdint.h>

namespace noel {

/* ------------------------------------------------------------------ cast */

enum I8Type { kI8F32 = 0, kI8F16 = 1, kI8BF16 = 30 };  // NOEL_HEAD_* of noel_lmhead.h

struct I8CastArgs {
    const void *x;  // [rows][ldx]
    int64_t ldx;
    int rows, cols;
    bool vec;       // every row of x starts on 16 bytes
    int8_t *q;      // [rows][ldq], 16-byte aligned rows
    int64_t ldq;
    float *scale;
};

constexpr int kI8CastThreads = 256;
constexpr int kI8CastEach = 16;  // columns of a thread's turn

template <int WT>
struct I8In;
template <>
struct I8In<kI8F32> {
    using T = float;
    static __device__ __forceinline__ float get(float v) { return v; }
};
template <>
struct I8In<kI8F16> {
    using T = __half;
    static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
};
template <>
struct I8In<kI8BF16> {
    using T = __nv_bfloat16;
    static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
};

template <int WT>
__device__ __forceinline__ void i8_load(const I8CastArgs &a, const typename I8In<WT>::T *row, int c, float (&v)[kI8CastEach]) {
    using T = typename I8In<WT>::T;
    if (a.vec && c + kI8CastEach <= a.cols) {
        constexpr int kPer = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < kI8CastEach; i += kPer) {
            const uint4 u = *reinterpret_cast<const uint4 *>(row + c + i);
            const T *e = reinterpret_cast<const T *>(&u);
#pragma unroll
            for (int j = 0; j < kPer; ++j) v[i + j] = I8In<WT>::get(e[j]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < kI8CastEach; ++i) v[i] = c + i < a.cols ? I8In<WT>::get(row[c + i]) : 0.0f;
    }
}

/* x / s to the nearest integer, ties to even, of the exact quotient: the
 * candidate from the rounded reciprocal is off by one at most, and the
 * remainder x - n s is a number of 24 bits, so fmaf gives it exactly. */
__device__ __forceinline__ int i8_quotient(float x, float s, float inv) {
    float n = rintf(x * inv);
    const float twice = 2.0f * fmaf(-n, s, x);
    const bool odd = (__float2int_rn(n) & 1) != 0;
    if (twice > s || (twice == s && odd)) n += 1.0f;
    else if (twice < -s || (twice == -s && odd)) n -= 1.0f;
    return __float2int_rn(n);
}

/* One CTA a row: its largest magnitude, then the cast.  The row is read
 * again for the cast, from the caches. */
template <int WT>
__global__ void __launch_bounds__(kI8CastThreads) i8_cast_kernel(const __grid_constant__ I8CastArgs a) {
    __shared__ uint32_t s_top[kI8CastThreads / 32];
    using T = typename I8In<WT>::T;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int tid = threadIdx.x;
    const T *row = static_cast<const T *>(a.x) + (int64_t)blockIdx.x * a.ldx;
    uint32_t top = 0;  // magnitudes as bits: NaN is above infinity
    for (int c = tid * kI8CastEach; c < a.cols; c += kI8CastThreads * kI8CastEach) {
        float v[kI8CastEach];
        i8_load<WT>(a, row, c, v);
#pragma unroll
        for (int i = 0; i < kI8CastEach; ++i) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    }
    top = __reduce_max_sync(0xFFFFFFFFu, top);
    if ((tid & 31) == 0) s_top[tid >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kI8CastThreads / 32; ++w) top = max(top, s_top[w]);
    const bool finite = top < 0x7F800000u;
    const float s = finite ? fmaxf(__fdiv_rn(__uint_as_float(top), 127.0f), 1.17549435e-38f) : 1.0f;
    const float inv = __frcp_rn(s);
    int8_t *q = a.q + (int64_t)blockIdx.x * a.ldq;
    for (int c = tid * kI8CastEach; c < a.cols; c += kI8CastThreads * kI8CastEach) {
        float v[kI8CastEach];
        i8_load<WT>(a, row, c, v);
        uint32_t word[kI8CastEach / 4];
#pragma unroll
        for (int i = 0; i < kI8CastEach; ++i) {
            const uint32_t b = finite ? (uint32_t)i8_quotient(v[i], s, inv) & 0xFFu : 0u;
            word[i / 4] = i % 4 ? word[i / 4] | b << (8 * (i % 4)) : b;
        }
        if (c + kI8CastEach <= a.cols) {
            *reinterpret_cast<uint4 *>(q + c) = make_uint4(word[0], word[1], word[2], word[3]);
        } else {
#pragma unroll
            for (int i = 0; i < kI8CastEach; ++i)
                if (c + i < a.cols) q[c + i] = (int8_t)(word[i / 4] >> (8 * (i % 4)));
        }
    }
    /* a row with an infinity or a NaN has no cast: its scale makes every result of it NaN */
    if (tid == 0) a.scale[blockIdx.x] = finite ? s : __uint_as_float(0x7FC00000u);
}

/* --------------------------------------------------------------- product */

struct I8Args {
    const float *a_scale;  // [tokens]
    const float *w_scale;  // [rows]
    void *y;               // [tokens][ldy]
    int64_t ldy;
    int tokens, rows, cols;
    bool ranges;           // every group one range of rows and all tokens (one tile of them)
    unsigned long long wait_ns;
    int stall;             // load nothing, so that waits run out
    unsigned *failed;      // counts the products that gave up
};

constexpr int kI8Threads = 352;  // two warps of loads, one of products, eight of results
constexpr int kI8RowsCta = 128;  // rows of w in a CTA's tile (lanes of the tensor memory)
constexpr int kI8Line = 128;     // columns (bytes) of a copy: one swizzled line of each row
constexpr int kI8Box = 32;       // rows of w in one copy where a tile has fewer than 128
constexpr int kI8MaxStages = 12;
constexpr int kI8Ring = 225280;  // bytes of the ring at most
constexpr unsigned long long kI8LandNs = 1000000;  // copies and products that were issued have ended after this, by far

/* lines of a row in a stage: two where tiles are narrow and the weights' stream is what counts (a stage is then 32 KB of
 * them, and the memory is asked for 256 bytes of a row at once) */
__host__ __device__ constexpr int i8_lines(int nt) { return nt <= 64 ? 2 : 1; }
__host__ __device__ constexpr int i8_stage_bytes(int nt, bool pair) {
    return (kI8RowsCta + (pair ? nt / 2 : nt)) * kI8Line * i8_lines(nt);
}
__host__ __device__ constexpr int i8_stages(int nt, bool pair) {
    return kI8Ring / i8_stage_bytes(nt, pair) < kI8MaxStages ? kI8Ring / i8_stage_bytes(nt, pair) : kI8MaxStages;
}
__host__ __device__ constexpr int i8_smem(int nt, bool pair) {
    return i8_stages(nt, pair) * i8_stage_bytes(nt, pair) + 1024;  // stages start on 1024 bytes
}

__device__ __forceinline__ uint32_t i8_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void i8_bar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void i8_bar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
/* arrive at a barrier of either CTA of the cluster */
__device__ __forceinline__ void i8_bar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
/* the address in shared::cluster of CTA rank's variable at this CTA's address */
__device__ __forceinline__ uint32_t i8_peer(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ unsigned long long i8_now() {
    unsigned long long t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}
/* Wait for the phase of that parity; false where the limit ran out, or where stop (if any) says that another wait's has. */
__device__ __forceinline__ bool i8_wait(uint32_t bar, uint32_t parity, unsigned long long limit, const volatile uint32_t *stop) {
    unsigned long long begin = 0;
    for (int i = 0;; ++i) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done)
            : "r"(bar), "r"(parity)
            : "memory");
        if (done) return true;
        if (stop && *stop) return false;
        if (i == 0) begin = i8_now();
        else if ((i & 15) == 0 && i8_now() - begin > limit) return false;
    }
}
/* A wait ran out: the host is to learn of it, and the other waits of the CTA (of both CTAs of a pair) end too. */
template <bool PAIR>
__device__ __forceinline__ void i8_give_up(uint32_t *stop, uint32_t rank, unsigned *failed) {
    atomicAdd(failed, 1u);
    *(volatile uint32_t *)stop = 1;
    if (PAIR) asm volatile("st.relaxed.cluster.shared::cluster.u32 [%0], %1;" ::"r"(i8_peer(i8_addr(stop), rank ^ 1)), "r"(1u) : "memory");
}
/* whether it is so for any of the 256 threads of results, which meet here */
__device__ __forceinline__ bool i8_any(bool mine) {
    uint32_t any;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbar.red.or.pred q, 1, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(any)
        : "r"((uint32_t)mine)
        : "memory");
    return any != 0;
}
template <bool PAIR>
__device__ __forceinline__ void i8_copy(const CUtensorMap *map, uint32_t dst, uint32_t bar, int x, int y) {
    if (PAIR)
        asm volatile(
            "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
            ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
            ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
}
/* Operand rows of 128 bytes in groups of eight, swizzled by 128 bytes: start / 16, stride between groups 1024 / 16,
 * version 1, swizzle mode 2. */
__device__ __forceinline__ uint64_t i8_desc(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | 1ull << 16 | (uint64_t)(1024 >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
template <bool PAIR>
__device__ __forceinline__ void i8_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    if (PAIR)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
            "r"((uint32_t)add) : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
            "r"((uint32_t)add) : "memory");
}
/* arrive at bar (of both CTAs of a pair) when the products issued so far are done */
template <bool PAIR>
__device__ __forceinline__ void i8_commit(uint32_t bar) {
    if (PAIR)
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
            "h"((uint16_t)3) : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void i8_store(float *p, float v) { *p = v; }
__device__ __forceinline__ void i8_store(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }

/* What a group (a CTA, or a pair of CTAs that share tiles of 256 rows) works through. */
template <int NT, bool PAIR>
struct I8Tiles {
    static constexpr int kRows = PAIR ? 2 * kI8RowsCta : kI8RowsCta;
    int row, row_end, t0;
    int group, groups, last, token_tiles, rows;
    bool ranges;
    int64_t index;

    __device__ __forceinline__ I8Tiles(const I8Args &a) {
        group = blockIdx.x / (PAIR ? 2 : 1);
        groups = gridDim.x / (PAIR ? 2 : 1);
        rows = a.rows;
        token_tiles = (a.tokens + NT - 1) / NT;
        ranges = a.ranges;
        last = (int)((int64_t)rows * (group + 1) / groups);
        index = group;
        row = (int)((int64_t)rows * group / groups);
        t0 = 0;
        if (!ranges) place();
        else row_end = min(row + kRows, last);
    }
    __device__ __forceinline__ void place() {
        const int64_t m = index / token_tiles;
        t0 = (int)(index - m * token_tiles) * NT;
        row = (int)min((int64_t)rows, m * kRows);
        row_end = min(rows, row + kRows);
    }
    __device__ __forceinline__ bool more() const { return row < (ranges ? last : rows); }
    __device__ __forceinline__ void next() {
        if (ranges) {
            row += kRows;
            row_end = min(row + kRows, last);
        } else {
            index += groups;
            place();
        }
    }
};

/*
 * A tile is 128 rows of w (256 of a pair of CTAs) by NT tokens: rows are
 * lanes of the tensor memory and tokens its columns, so that a warp's
 * results for a token lie side by side in y, and the few tokens of a decode
 * batch are columns of a narrow tile.  Two lanes copy stages by TMA, the
 * weights' one and the tokens' one, one lane issues their products, eight warps scale and store a
 * finished tile while the next one's products go into the other half of the
 * accumulators.
 *
 * 152,064 rows of 4096 columns: one token 112 us with its cast, 64 tokens 120
 * (HBM: 84 % of the measured copy; copies of 128 rows x 256 bytes, since a copy
 * costs its lane about 100 ns whatever its size: 32 rows at a time 124 us
 * for the copies alone, 128 rows 105).  2048 tokens 870 to 915 us in a dozen
 * single calls (2.8 to 2.9 POPS; products alone on real data 696 us, loads and
 * stores with a quarter of the products 637) and 1050 to 1070 in a loop, where
 * power holds the clocks down.
 * Pairs halve what a CTA needs of the tokens: 913 against 989 us; with tiles
 * of 128 tokens pairs took 1866 against 1354.
 */
template <int NT, bool PAIR, typename OUT>
__global__ void __launch_bounds__(kI8Threads, 1)
    i8_product_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_part,
                      const __grid_constant__ CUtensorMap map_a, const __grid_constant__ I8Args a) {
    constexpr int kStages = i8_stages(NT, PAIR), kStage = i8_stage_bytes(NT, PAIR), kHalf = PAIR ? NT / 2 : NT;
    constexpr int kLines = i8_lines(NT), kLineW = kI8RowsCta * kI8Line, kLineA = kHalf * kI8Line;  // a stage: w's lines, then a's
    constexpr uint32_t kCols = 2 * NT < 32 ? 32 : 2 * NT;
    extern __shared__ unsigned char i8_raw[];
    __shared__ __align__(8) uint64_t s_full[kI8MaxStages], s_empty[kI8MaxStages], s_done[2], s_free[2], s_end;
    __shared__ float s_scale[2][NT];  // of the tile's tokens
    __shared__ uint32_t s_tmem, s_stop;  // s_stop: a wait ran out
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t rank = 0;
    if (PAIR) asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    const uint32_t ring = (i8_addr(i8_raw) + 1023u) & ~1023u;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i) i8_bar_init(i8_addr(&s_full[i]), 1), i8_bar_init(i8_addr(&s_empty[i]), 1);
        for (int i = 0; i < 2; ++i) i8_bar_init(i8_addr(&s_done[i]), 1), i8_bar_init(i8_addr(&s_free[i]), PAIR ? 16 : 8);
        i8_bar_init(i8_addr(&s_end), 1);
        s_stop = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        if (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(i8_addr(&s_tmem)), "r"(kCols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(i8_addr(&s_tmem)), "r"(kCols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    }
    if (PAIR) {
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = s_tmem;
    const int chunks = (a.cols + kLines * kI8Line - 1) / (kLines * kI8Line);
    const volatile uint32_t *stop = &s_stop;
    int stage = 0;  // of the ring, where this warp works with it
    uint32_t phase = 0;

    if (warp == 0 && lane == 0 && !a.stall) {
        /* --------------------------------------------- copies of weights */
        auto copies = [](const I8Tiles<NT, PAIR> &t, int r) {  // rows copied for CTA r of the group
            const int n = min(t.row_end - t.row - r * kI8RowsCta, kI8RowsCta);
            return n <= 0 ? 0 : (n + kI8Box - 1) / kI8Box * kI8Box;
        };
        I8Tiles<NT, PAIR> t(a);
        bool good = true;
        for (; good && !*stop && t.more(); t.next()) {
            const int n = copies(t, rank), row = t.row + (int)rank * kI8RowsCta;
            int all = n + kHalf;
            if (PAIR) all += copies(t, rank ^ 1) + kHalf;
            for (int k = 0; k < chunks; ++k) {
                good = i8_wait(i8_addr(&s_empty[stage]), phase ^ 1, a.wait_ns, stop);
                if (!good) break;
                const uint32_t bar = i8_addr(&s_full[stage]), to = PAIR ? i8_peer(bar, 0) : bar, at = ring + stage * kStage;
                if (rank == 0) i8_bar_expect(bar, (uint32_t)all * kI8Line * kLines);
#pragma unroll
                for (int l = 0; l < kLines; ++l) {
                    const int x = (k * kLines + l) * kI8Line;
                    if (n == kI8RowsCta) {
                        i8_copy<PAIR>(&map_w, at + l * kLineW, to, x, row);
                    } else {
                        for (int i = 0; i < n; i += kI8Box) i8_copy<PAIR>(&map_part, at + l * kLineW + i * kI8Line, to, x, row + i);
                    }
                }
                if (++stage == kStages) stage = 0, phase ^= 1;
            }
        }
        if (!good) i8_give_up<PAIR>(&s_stop, rank, a.failed);
    } else if (warp == 10 && lane == 0 && !a.stall) {
        /* ---------------------------------------------- copies of tokens */
        asm volatile("griddepcontrol.wait;" ::: "memory");  // their cast; the first weights do not wait for it
        bool good = true;
        for (I8Tiles<NT, PAIR> t(a); good && !*stop && t.more(); t.next())
            for (int k = 0; k < chunks; ++k) {
                good = i8_wait(i8_addr(&s_empty[stage]), phase ^ 1, a.wait_ns, stop);
                if (!good) break;
                const uint32_t bar = i8_addr(&s_full[stage]), to = PAIR ? i8_peer(bar, 0) : bar;
#pragma unroll
                for (int l = 0; l < kLines; ++l)
                    i8_copy<PAIR>(&map_a, ring + stage * kStage + kLines * kLineW + l * kLineA, to, (k * kLines + l) * kI8Line,
                                  t.t0 + (int)rank * kHalf);
                if (++stage == kStages) stage = 0, phase ^= 1;
            }
        if (!good) i8_give_up<PAIR>(&s_stop, rank, a.failed);
    } else if (warp == 1 && lane == 0 && rank == 0) {
        /* ----------------------------------------------------- products */
        /* 32-bit sums of signed bytes, N and M of the tile */
        constexpr uint32_t kIdesc = 2u << 4 | 1u << 7 | 1u << 10 | (uint32_t)(NT / 8) << 17 |
                                    (uint32_t)((PAIR ? 256 : 128) / 16) << 24;
        int tile = 0;
        bool good = true;
        for (I8Tiles<NT, PAIR> t(a); good && !*stop && t.more(); t.next(), ++tile) {
            const int half = tile & 1;
            good = i8_wait(i8_addr(&s_free[half]), ((tile >> 1) & 1) ^ 1, a.wait_ns, stop);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            for (int k = 0; good && k < chunks; ++k) {
                good = i8_wait(i8_addr(&s_full[stage]), phase, a.wait_ns, stop);
                if (!good) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint64_t dw = i8_desc(ring + stage * kStage), da = i8_desc(ring + stage * kStage + kLines * kLineW);
#pragma unroll
                for (int l = 0; l < kLines; ++l)
#pragma unroll
                    for (int j = 0; j < kI8Line / 32; ++j)
                        i8_mma<PAIR>(tmem + half * NT, dw + l * (kLineW >> 4) + 2 * j, da + l * (kLineA >> 4) + 2 * j, kIdesc,
                                     k > 0 || l > 0 || j > 0);
                i8_commit<PAIR>(i8_addr(&s_empty[stage]));
                if (++stage == kStages) stage = 0, phase ^= 1;
            }
            if (good) i8_commit<PAIR>(i8_addr(&s_done[half]));
        }
        if (!good) i8_give_up<PAIR>(&s_stop, rank, a.failed);
    } else if (warp >= 2 && warp < 10) {
        /* ------------------------------------------------------ results */
        asm volatile("griddepcontrol.wait;" ::: "memory");
        /* a quarter of the tensor memory's lanes, which is all that a warp may read, and every other 16 tokens */
        const int quarter = warp & 3, side = (warp - 2) >> 2;
        int tile = 0;
        bool failed = false;
        for (I8Tiles<NT, PAIR> t(a); t.more(); t.next(), ++tile) {
            const int half = tile & 1;
            const int r = t.row + (int)rank * kI8RowsCta + quarter * 32 + lane;
            const bool mine = r < t.row_end;
            const float ws = mine ? a.w_scale[r] : 0.0f;
            const int nt = min(NT, a.tokens - t.t0);
            for (int i = threadIdx.x - 64; i < nt; i += 256) s_scale[half][i] = a.a_scale[t.t0 + i];
            if (i8_any(failed)) break;  // all of them or none; the scales of two tiles ago have been used
            if (!__all_sync(0xFFFFFFFFu, i8_wait(i8_addr(&s_done[half]), (tile >> 1) & 1, a.wait_ns, stop))) {
                if (lane == 0) i8_give_up<PAIR>(&s_stop, rank, a.failed);
                failed = true;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            OUT *y = static_cast<OUT *>(a.y) + (int64_t)(t.t0 + side * 16) * a.ldy + r;
#pragma unroll 1
            for (int c = side * 16; c < nt && !failed; c += 32, y += 32 * a.ldy) {
                uint32_t v[16];
                asm volatile(
                    "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                    : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
                      "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                    : "r"(tmem + ((uint32_t)(quarter * 32) << 16) + half * NT + c));
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                if (mine) {
                    const float *as = &s_scale[half][c];
                    OUT *to = y;
                    if (c + 16 <= nt) {
#pragma unroll
                        for (int j = 0; j < 16; ++j, to += a.ldy) i8_store(to, __int2float_rn((int)v[j]) * ws * as[j]);
                    } else {
#pragma unroll
                        for (int j = 0; j < 15; ++j, to += a.ldy)
                            if (c + j < nt) i8_store(to, __int2float_rn((int)v[j]) * ws * as[j]);
                    }
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0 && !failed) i8_bar_arrive(i8_peer(i8_addr(&s_free[half]), 0));
        }
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    if (PAIR) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    __syncthreads();
    if (s_stop) {
        /*
         * A wait ran out, in this CTA or in its pair's other one, so copies into this memory and products of it may be
         * on their way: they end before the CTA does.  A stage of which not all copies were issued never fills, so the
         * time has to do as well.
         */
        if (warp == 1 && lane == 0 && rank == 0) {
            i8_commit<PAIR>(i8_addr(&s_end));
            i8_wait(i8_addr(&s_end), 0, a.wait_ns + kI8LandNs, nullptr);
        } else if (warp == 0 && lane == 0 && !a.stall) {
            const unsigned long long begin = i8_now();
            for (int s = 0; rank == 0 && s < kStages; ++s) {
                const unsigned long long spent = i8_now() - begin;
                if (spent < a.wait_ns) i8_wait(i8_addr(&s_full[s]), s < stage ? phase : phase ^ 1, a.wait_ns - spent, nullptr);
            }
            while (i8_now() - begin < kI8LandNs) __nanosleep(1000);
        }
        __syncwarp();
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        if (PAIR) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        __syncthreads();
    }
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols));
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols));
    }
}

}  // namespace noel
