/*
 * Per-request processing of logits (include/noel_logits.h): penalties for
 * repeated tokens, biases and masks on a batch of rows, in place.
 *
 * Per row b and id v, with n the occurrences of v among the row's generated
 * ids and seen = v is anywhere in the history:
 *   x = x > 0 ? x / rep : x * rep (seen);  x -= freq n, x -= pres (n > 0);
 *   x += biases on v;  x = -inf (masked)
 * in fp32 with one rounding to bf16 at the end.
 *
 * Nothing here reads the row as a whole.  A row's history and bias list name
 * the few logits that the penalties and biases change, and a mask only writes;
 * what has to move is the history, the mask's bits, the touched logits and the
 * masked ones.  What bounds it: strict masks, memory (1024 x 152,064 fp32 that
 * allow 0.5 % of the ids move 621 MB, 582 of which are needed, in 121 us, 5.1
 * TB/s; a bare fill of the rows takes 88 us).  Masks that take little away,
 * neither issue slots nor memory (1024 x 256,000 bf16 that allow 98 %: 112 us at
 * 2.8 TB/s); each masked logit is a store of its own there, a partly written
 * sector that the L2 completes.  Tables, latency: 256 rows with 1024
 * ids and 300 biases take 16 us with a fifth of the warps active and a quarter
 * of the issue slots busy.  Long histories, issue slots (60 % busy): 64 rows of
 * 65,536 ids 44 us.  One row takes 4.7 us.
 *
 * These are times on the device, in a CUDA graph; back-to-back calls from Python
 * take 123, 113, 18, 53 and 7.6 us.
 */
#pragma once

#include "sampler_kernels.cuh"
#include "sampler_warp.cuh"
#include "sector.cuh"

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
    int ranges, range;  // CTAs per row of the rows kernel and their columns
    int cap;            // entries of a CTA's table; 0: none
    int slices, slice;  // CTAs per row of the slice kernel and the words each counts in
};

constexpr int kLogitsThreads = 256;
constexpr int kRowsCtas = 6;         // CTAs per SM the rows kernel is compiled for
constexpr int kMaskPiece = 1024;     // columns of a warp's turn: 32 words of the mask
constexpr int kMaskRange = 131072;   // bytes of a row that a CTA masks, at most
constexpr int kMaskWhole = 22;       // touched sectors of 32 from which on they are written whole
constexpr int kMaskFew = 48;         // masked logits of a warp's turn up to which they are written one by one
constexpr int kTableMax = 8192;      // history plus biases a row's table may take
constexpr int kTableMaskMax = 2048;  // and where the same CTA masks
constexpr int kTableBatch = 8;       // loads in flight per thread of the table
constexpr int kSliceThreads = 512;
constexpr int kSliceMax = 24576;     // columns of a slice: one 32-bit word of shared memory each
constexpr int kLogitsMaxBias = 16384;
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
    float inv;  // 1 / rep, or 0 where quotients by rep are left to the division
};

__device__ __forceinline__ RowRules row_rules(const LogitsArgs &a, int row) {
    const float rep = a.rep ? a.rep[row] : 1.0f;
    return {rep, a.freq ? a.freq[row] : 0.0f, a.pres ? a.pres[row] : 0.0f,
            rep > 0.0009765625f && rep < 1024.0f ? __fdiv_rn(1.0f, rep) : 0.0f};
}

/* x / rep for x > 0: a quotient from the reciprocal, corrected by its
 * remainder (Markstein 1990), which is the rounded quotient where nothing on
 * the way over- or underflows.  x below 2^-101 is taken times 2^100; of a
 * quotient that is subnormal then, the last bit is made odd where a remainder
 * is left (Boldo and Melquiond 2008), so that scaling it back rounds as if
 * from the exact quotient (it has to lose two bits for that; one binade is
 * left to the division, as are huge x and unlikely rep). */
__device__ __forceinline__ float quotient(float x, const RowRules &r) {
    const uint32_t e = __float_as_uint(x) & 0x7F800000u;
    if (r.inv == 0.0f || e > 0x70000000u) return __fdiv_rn(x, r.rep);
    if (e >= 0x0D000000u) {
        const float q = __fmul_rn(x, r.inv);
        return __fmaf_rn(__fmaf_rn(-q, r.rep, x), r.inv, q);
    }
    const float up = __uint_as_float((127u + 100u) << 23), down = __uint_as_float((127u - 100u) << 23);
    const float X = __fmul_rn(x, up);
    float q = __fmul_rn(X, r.inv);
    q = __fmaf_rn(__fmaf_rn(-q, r.rep, X), r.inv, q);
    const float rest = __fmaf_rn(-q, r.rep, X);
    uint32_t b = __float_as_uint(q);
    if (b < (127u - 26u) << 23) {           // subnormal
        if (b >= (127u - 27u) << 23) return __fdiv_rn(x, r.rep);
        if (rest != 0.0f) b = (rest > 0.0f ? b : b - 1u) | 1u;
    }
    return __fmul_rn(__uint_as_float(b), down);
}

__device__ __forceinline__ float penalised(float x, uint32_t w, const RowRules &r) {
    const uint32_t n = w & kCount;
    if (w & (kSeenPrompt | kCount)) x = x > 0.0f ? quotient(x, r) : __fmul_rn(x, r.rep);
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

/* the ids of a row's history that count, and how many of them are prompt */
struct RowHistory {
    const int32_t *ids;
    int len, prompt;
};

__device__ __forceinline__ RowHistory row_history(const LogitsArgs &a, int row) {
    if (!a.hist) return {nullptr, 0, 0};
    return {a.hist + (size_t)row * (size_t)a.hld,
            a.hist_lens ? min(max(a.hist_lens[row], 0), a.hist_len) : a.hist_len,
            a.prompt_lens ? a.prompt_lens[row] : 0};
}

/* the sum of a row's biases on one id, in list order, by a whole warp */
__device__ __forceinline__ float bias_sum(const int32_t *bi, const float *bv, int nb, int id) {
    const int lane = threadIdx.x & 31;
    float s = 0.0f;
    for (int j0 = 0; j0 < nb; j0 += 32) {
        const int j = j0 + lane;
        const bool hit = j < nb && bi[j] == id;
        const float v = hit ? bv[j] : 0.0f;
        for (uint32_t m = __ballot_sync(kFull, hit); m; m &= m - 1)
            s = __fadd_rn(s, __shfl_sync(kFull, v, __ffs(m) - 1));
    }
    return s;
}

/* The table of a CTA's columns [lo, hi) of a row: open addressing in shared
 * memory, entry = (column + 1, word, bias). */
struct Table {
    uint32_t *key, *word;
    float *sum;
    int cap;  // a power of two, a multiple of the CTA's threads, at least 3/2 of what can come in
};

__device__ __forceinline__ uint32_t table_slot(const Table &t, uint32_t k) {
    uint32_t p = hs_hash(k) >> (33 - __ffs(t.cap));
    for (int probe = 0; probe < t.cap; ++probe) {
        uint32_t prev = *(volatile uint32_t *)&t.key[p];  // a repeated id needs no compare-and-swap
        if (prev == 0u) prev = atomicCAS(&t.key[p], 0u, k);
        if (prev == 0u || prev == k) break;
        p = (p + 1) & (uint32_t)(t.cap - 1);
    }
    return p;
}

/* The row's history and bias ids of columns [lo, hi) into the table.  Loads go
 * out kTableBatch at a time: with few CTAs per SM the time of this is the
 * number of load latencies in a row. */
__device__ __forceinline__ void table_fill(const LogitsArgs &a, int row, const Table &t, int lo, int hi) {
    const int tid = threadIdx.x;
    const RowHistory h = row_history(a, row);
    for (int i = tid; i < t.cap / 2; i += kLogitsThreads)  // keys and words
        reinterpret_cast<uint4 *>(t.key)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    for (int i0 = tid; i0 < h.len; i0 += kTableBatch * kLogitsThreads) {
        int id[kTableBatch];
#pragma unroll
        for (int u = 0; u < kTableBatch; ++u) {
            const int i = i0 + u * kLogitsThreads;
            id[u] = i < h.len ? h.ids[i] : -1;
        }
#pragma unroll
        for (int u = 0; u < kTableBatch; ++u) {
            const int64_t c = (int64_t)id[u] - a.v_begin;
            if (id[u] < 0 || c < lo || c >= hi) continue;
            const uint32_t p = table_slot(t, (uint32_t)c + 1u);
            if (i0 + u * kLogitsThreads < h.prompt) atomicOr(&t.word[p], kSeenPrompt);
            else atomicAdd(&t.word[p], 1u);
        }
    }
    const int nb = a.bias_len;
    const int32_t *bi = nb ? a.bias_ids + (size_t)row * (size_t)a.bld : nullptr;
    const float *bv = nb ? a.bias + (size_t)row * (size_t)a.bld : nullptr;
    for (int i0 = tid; i0 < nb; i0 += 2 * kLogitsThreads) {
        int id[2];
        float v[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int i = i0 + u * kLogitsThreads;
            id[u] = i < nb ? bi[i] : -1;
            v[u] = i < nb ? bv[i] : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int64_t c = (int64_t)id[u] - a.v_begin;
            if (id[u] < 0 || c < lo || c >= hi) continue;
            const uint32_t p = table_slot(t, (uint32_t)c + 1u);
            if (atomicOr(&t.word[p], kHasBias) & kHasBias) atomicOr(&t.word[p], kManyBiases);
            else t.sum[p] = v[u];  // the entry's only writer
        }
    }
}

/* Each entry's logit read, changed and written once, masked ones left alone. */
template <typename T>
__device__ __forceinline__ void table_apply(const LogitsArgs &a, int row, const Table &t, const uint32_t *mask) {
    const int tid = threadIdx.x, nb = a.bias_len;
    const RowRules rules = row_rules(a, row);
    const int32_t *bi = nb ? a.bias_ids + (size_t)row * (size_t)a.bld : nullptr;
    const float *bv = nb ? a.bias + (size_t)row * (size_t)a.bld : nullptr;
    T *x = static_cast<T *>(a.logits) + (size_t)row * (size_t)a.ld;
    for (int s0 = tid; s0 < t.cap; s0 += kTableBatch * kLogitsThreads) {  // whole warps
        uint32_t k[kTableBatch], m[kTableBatch];
        float v[kTableBatch];
#pragma unroll
        for (int u = 0; u < kTableBatch; ++u) {
            const int s = s0 + u * kLogitsThreads;
            k[u] = s < t.cap ? t.key[s] : 0u;
            v[u] = k[u] ? logit_load(x + (k[u] - 1u)) : 0.0f;
            const uint32_t id = (uint32_t)a.v_begin + k[u] - 1u;
            m[u] = k[u] && mask ? mask[id >> 5] >> (id & 31u) : 1u;
        }
#pragma unroll
        for (int u = 0; u < kTableBatch; ++u) {
            const int s = s0 + u * kLogitsThreads;
            const bool on = k[u] && (m[u] & 1u);
            const uint32_t w = on ? t.word[s] : 0u;
            float b = on && (w & kHasBias) ? t.sum[s] : 0.0f;
            if (nb) {
                for (uint32_t q = __ballot_sync(kFull, (w & kManyBiases) != 0u); q; q &= q - 1) {
                    const int l = __ffs(q) - 1;
                    const float all = bias_sum(bi, bv, nb, a.v_begin + (int)(__shfl_sync(kFull, k[u], l) - 1u));
                    if ((tid & 31) == l) b = all;
                }
            }
            if (!on) continue;
            float y = penalised(v[u], w, rules);
            if (w & kHasBias) y = __fadd_rn(y, b);
            logit_store(x + (k[u] - 1u), y);
        }
    }
}

/* -infinity for the elements whose bit in gone is set */
__device__ __forceinline__ void sector_mask(Sector &s, uint32_t gone, float) {
#pragma unroll
    for (int e = 0; e < 8; ++e) s.u[e] = gone >> e & 1u ? 0xFF800000u : s.u[e];
}
__device__ __forceinline__ void sector_mask(Sector &s, uint32_t gone, uint16_t) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint32_t keep = (gone >> (2 * e) & 1u ? 0u : 0xFFFFu) | (gone >> (2 * e + 1) & 1u ? 0u : 0xFFFF0000u);
        s.u[e] = (s.u[e] & keep) | (0xFF80FF80u & ~keep);
    }
}

/* The 32 mask bits of columns c .. c + 31, those outside the row as allowed. */
__device__ __forceinline__ uint32_t mask_bits(const LogitsArgs &a, const uint32_t *mask, int64_t c) {
    if (c >= a.vocab) return 0xFFFFFFFFu;
    const int64_t bit = a.v_begin + c, wi = bit >> 5, nw = ((int64_t)a.v_begin + a.vocab + 31) >> 5;
    const uint32_t lo = wi >= 0 ? __ldg(mask + wi) : 0xFFFFFFFFu;
    const uint32_t hi = (bit & 31) && wi + 1 < nw ? __ldg(mask + wi + 1) : 0xFFFFFFFFu;
    uint32_t ok = __funnelshift_r(lo, hi, (uint32_t)bit & 31u);
    if (c < 0) ok |= (1u << -c) - 1u;
    if (c + 32 > a.vocab) ok |= 0xFFFFFFFFu << (a.vocab - c);
    return ok;
}

/* One warp masks the 1024 columns from c0 on, whose mask bits lane l holds 32
 * at a time; c0 lies on 32 bytes of memory and may lie before the row.
 *
 * A line of which some bytes are written and others left costs its read as
 * well, when the L2 gets to it.  So where kMaskWhole of the warp's 32 sectors
 * have something masked, the others and the partly masked ones are read and
 * all 1024 bytes are written in one store; where fewer have, the masked logits
 * are written one by one.  Measured on 512 x 152,064 under masks that allow
 * 50, 90, 95 and 98 % of the ids (fp32: 100, 57, 34, 15 % of the sectors
 * touched; bf16: 100, 81, 56, 28 %): always whole 99, 99, 99, 99 us (bf16 55,
 * 55, 55, 55), always one by one 232, 79, 57, 43 (bf16 235, 74, 45, 31).  With
 * few masked logits in all 1024 columns the lanes do without sectors (99.9 %
 * allowed: 28.9 -> 24.5 us). */
template <typename T>
__device__ __forceinline__ void mask_piece(const LogitsArgs &a, T *x, int64_t c0, uint32_t ok) {
    constexpr int VE = 32 / sizeof(T);  // elements a lane takes at a time
    constexpr int STEPS = kMaskPiece / (32 * VE), BATCH = 2;
    constexpr uint32_t ALL = VE == 32 ? 0xFFFFFFFFu : (1u << VE) - 1u;
    const int lane = threadIdx.x & 31;
    const int masked = (int)__reduce_add_sync(kFull, (uint32_t)__popc(~ok));
    if (masked <= kMaskFew) {  // every lane writes the logits of its own word
        T *own = x + c0 + 32 * lane;
        for (uint32_t g = ~ok; g; g &= g - 1) logit_store(own + (__ffs(g) - 1), -INFINITY);
        return;
    }
    T *at = x + c0 + VE * lane;  // may lie outside the row; nothing there is touched
    /* the steps whose columns all lie inside the row */
    const int first = c0 < 0 ? 1 : 0;
    const int last = (int)min((a.vocab - c0) / (32 * VE), (int64_t)STEPS);
#pragma unroll
    for (int q0 = 0; q0 < STEPS; q0 += BATCH) {
        Sector s[BATCH];
        uint32_t gone[BATCH];
        bool whole[BATCH];
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {  // VE words of the mask cover 32 lanes x VE columns
            const int q = q0 + j;
            const uint32_t w = __shfl_sync(kFull, ok, q * VE + lane * VE / 32);
            gone[j] = ~(w >> (lane * VE % 32)) & ALL;
            whole[j] = __popc(__ballot_sync(kFull, gone[j] != 0u)) >= kMaskWhole && q >= first && q < last;
            if (whole[j] && gone[j] != ALL) s[j] = sector_load(at + q * 32 * VE);
        }
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
            T *to = at + (q0 + j) * 32 * VE;
            if (whole[j]) {
                sector_mask(s[j], gone[j], T{});
                sector_store(to, s[j]);
            } else {
                for (uint32_t g = gone[j]; g; g &= g - 1) logit_store(to + (__ffs(g) - 1), -INFINITY);
            }
        }
    }
}

/* One CTA per row and range of its columns: the table of the range is filled,
 * the range is masked (WRITE; without it the kernel has 64 registers a thread
 * instead of 40: 16.3 against 17.9 us for 256 rows with 1024 ids), and then the table's logits are changed.  The mask
 * never changes an allowed logit's value but may write it back as it read it,
 * so the table's own writes come after the mask's, a CTA's barrier between
 * them.  (One warp filling the table while the others mask was slower in small
 * batches, 27 against 18 us at 64 rows, and no faster in large ones.) */
template <typename T, bool WRITE>
__global__ void __launch_bounds__(kLogitsThreads, WRITE ? kRowsCtas : 4) logits_rows_kernel(const __grid_constant__ LogitsArgs a) {
    extern __shared__ __align__(16) uint32_t logits_smem[];
    __shared__ int turn;
    constexpr int VE = 32 / sizeof(T);
    const int row = blockIdx.x / a.ranges, range = blockIdx.x % a.ranges;
    const uint32_t *mask = row_mask(a, row);
    T *x = static_cast<T *>(a.logits) + (size_t)row * (size_t)a.ld;
    /* ranges begin on 32 bytes of memory, the first one up to VE - 1 columns before the row */
    const int64_t begin = (int64_t)range * a.range - (int)((reinterpret_cast<uintptr_t>(x) / sizeof(T)) % VE);
    const int64_t end = min(begin + a.range, (int64_t)a.vocab);
    const Table t{logits_smem, logits_smem + a.cap, reinterpret_cast<float *>(logits_smem + 2 * a.cap), a.cap};
    const int lo = (int)max(begin, (int64_t)0), hi = (int)max(end, (int64_t)lo);
    if (threadIdx.x == 0) turn = kLogitsThreads / 32;  // every warp's first turn is its own number
    if (a.cap) table_fill(a, row, t, lo, hi);
    if (WRITE && mask) {
        const int lane = threadIdx.x & 31;
        if (!a.cap) __syncthreads();
        int k = threadIdx.x >> 5;
        uint32_t next = mask_bits(a, mask, begin + (int64_t)k * kMaskPiece + 32 * lane);
        while (begin + (int64_t)k * kMaskPiece < end) {
            const uint32_t ok = next;
            const int64_t c = begin + (int64_t)k * kMaskPiece;
            if (lane == 0) k = atomicAdd(&turn, 1);
            k = __shfl_sync(kFull, k, 0);
            next = mask_bits(a, mask, begin + (int64_t)k * kMaskPiece + 32 * lane);  // on its way meanwhile
            mask_piece(a, x, c, ok);
        }
    }
    if (a.cap) {
        __syncthreads();
        table_apply<T>(a, row, t, mask);
    }
}

/* The penalties of a sector's words on its logits: on those whose bit of
 * `change` is set.  All of them are computed, and the odd quotients (see
 * quotient()) again by division. */
template <typename T>
__device__ __forceinline__ void sector_penalise(Sector &s, const uint32_t (&w)[32 / sizeof(T)], uint32_t change,
                                                const RowRules &r) {
    constexpr int VE = 32 / sizeof(T);
    float v[VE];
    uint32_t odd = 0u;
#pragma unroll
    for (int e = 0; e < VE; ++e) {
        const float x = sizeof(T) == 4 ? __uint_as_float(s.u[e % 8])
                                       : __uint_as_float(e & 1 ? s.u[e / 2 % 8] & 0xFFFF0000u : s.u[e / 2 % 8] << 16);
        const uint32_t exponent = __float_as_uint(x) & 0x7F800000u, n = w[e] & kCount;
        if (x > 0.0f && (r.inv == 0.0f || exponent < 0x0D000000u || exponent > 0x70000000u)) odd |= 1u << e;
        const float q = __fmul_rn(x, r.inv);
        float y = x > 0.0f ? __fmaf_rn(__fmaf_rn(-q, r.rep, x), r.inv, q) : __fmul_rn(x, r.rep);
        if (n) y = __fsub_rn(__fsub_rn(y, __fmul_rn(r.freq, (float)n)), r.pres);
        v[e] = y;
    }
    if (odd & change) {
#pragma unroll
        for (int e = 0; e < VE; ++e)
            if (odd & change & 1u << e)
                v[e] = penalised(sizeof(T) == 4 ? __uint_as_float(s.u[e % 8])
                                                : __uint_as_float(e & 1 ? s.u[e / 2 % 8] & 0xFFFF0000u : s.u[e / 2 % 8] << 16),
                                 w[e], r);
    }
#pragma unroll
    for (int e = 0; e < VE; ++e) {
        if (sizeof(T) == 4) {
            if (change >> e & 1u) s.u[e % 8] = __float_as_uint(v[e]);
        } else if (change >> e & 1u) {
            const uint32_t b = __bfloat16_as_ushort(__float2bfloat16_rn(v[e]));
            s.u[e / 2 % 8] = e & 1 ? (s.u[e / 2 % 8] & 0x0000FFFFu) | b << 16 : (s.u[e / 2 % 8] & 0xFFFF0000u) | b;
        }
    }
}

/* Histories too long for a table: one CTA per row and slice of columns counts
 * the whole history's ids of its slice, one word of shared memory per column,
 * and then goes through the slice.  Slice s of S (a power of two) has every
 * S-th line of 128 bytes: frequent tokens have low ids, and slices of
 * consecutive columns leave the first one nearly all the counting; a line
 * belongs to one CTA, which reads and writes it whole if the history touches
 * any of it (a long history touches most of the low ids' lines, and single
 * logits cost memory what whole lines cost). */
template <typename T>
__global__ void __launch_bounds__(kSliceThreads, 2) logits_slice_kernel(const __grid_constant__ LogitsArgs a) {
    extern __shared__ __align__(16) uint32_t logits_smem[];
    uint32_t *word = logits_smem;
    const int tid = threadIdx.x;
    const int row = blockIdx.x / a.slices;
    const uint32_t mine_c = blockIdx.x % a.slices;
    const int sh = __ffs(a.slices) - 1;
    constexpr int VE = 32 / sizeof(T), BLK = 4 * VE;  // columns of a sector and of a line
    const int width = a.slice;  // words of this slice (those past the vocabulary stay 0)
    const RowHistory h = row_history(a, row);
    const RowRules rules = row_rules(a, row);
    const uint32_t *mask = row_mask(a, row);
    for (int i = tid; i < width / 4; i += kSliceThreads) reinterpret_cast<uint4 *>(word)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    /* An id's column is id - v_begin (an id below wraps round to more than vocab), a column's line its bits from
     * LINE on, and its slice the lowest bits of the line; the slice's words hold its lines one after the other. */
    constexpr int LINE = sizeof(T) == 4 ? 5 : 6;
    static_assert(1 << LINE == BLK, "columns of a line");
    const uint32_t of_slice = (uint32_t)(a.slices - 1) << LINE, want = mine_c << LINE;
    auto index_of = [&](int id, uint32_t &c) {
        c = (uint32_t)id - (uint32_t)a.v_begin;
        const bool in = c < (uint32_t)a.vocab && (c & of_slice) == want;
        c = (c >> (LINE + sh) << LINE) | (c & (BLK - 1));  // its word
        return in;
    };
    /* the same and the change of the word without a branch: seven ids of eight are another slice's */
    const uint32_t word_s = (uint32_t)__cvta_generic_to_shared(word);
    auto mark = [&](int id) {
        const uint32_t c = (uint32_t)id - (uint32_t)a.v_begin;
        const uint32_t at = word_s + ((c >> (LINE + sh) << (LINE + 2)) | (c & (BLK - 1)) << 2);
        asm volatile("{\n\t.reg .pred p;\n\t.reg .u32 s;\n\tand.b32 s, %0, %1;\n\tsetp.eq.u32 p, s, %2;\n\t"
                     "setp.lt.and.u32 p, %0, %3, p;\n\t@p st.shared.u32 [%4], %5;\n\t}" ::"r"(c), "r"(of_slice), "r"(want),
                     "r"(a.vocab), "r"(at), "r"(kSeenPrompt) : "memory");
    };
    auto count = [&](int id) {
        const uint32_t c = (uint32_t)id - (uint32_t)a.v_begin;
        const uint32_t at = word_s + ((c >> (LINE + sh) << (LINE + 2)) | (c & (BLK - 1)) << 2);
        asm volatile("{\n\t.reg .pred p;\n\t.reg .u32 s;\n\tand.b32 s, %0, %1;\n\tsetp.eq.u32 p, s, %2;\n\t"
                     "setp.lt.and.u32 p, %0, %3, p;\n\t@p red.shared.add.u32 [%4], %5;\n\t}" ::"r"(c), "r"(of_slice),
                     "r"(want), "r"(a.vocab), "r"(at), "r"(1) : "memory");
    };
    /* the history 16 bytes at a time from its first aligned id on: the prompt
     * only marks, the rest counts */
    auto through = [&](const int32_t *ids, int n, auto take) {
        const int head = min(n, (int)((16 - (reinterpret_cast<uintptr_t>(ids) & 15)) / 4 % 4));
        const int vecs = (n - head) / 4;
        if (tid < head) take(ids[tid]);
        const int4 *v = reinterpret_cast<const int4 *>(ids + head);
#pragma unroll 4
        for (int i = tid; i < vecs; i += kSliceThreads) {
            const int4 q = __ldg(v + i);
            take(q.x);
            take(q.y);
            take(q.z);
            take(q.w);
        }
        const int tail = head + 4 * vecs + tid;
        if (tail < n) take(ids[tail]);
    };
    const int prompt = min(max(h.prompt, 0), h.len);
    through(h.ids, prompt, mark);  // every writer of a word writes the same
    __syncthreads();
    through(h.ids + prompt, h.len - prompt, count);
    const int nb = a.bias_len;
    const int32_t *bi = nb ? a.bias_ids + (size_t)row * (size_t)a.bld : nullptr;
    const float *bv = nb ? a.bias + (size_t)row * (size_t)a.bld : nullptr;
    uint32_t mine = 0u;  // the biases whose column this thread marked first
    static_assert(kLogitsMaxBias <= 32 * kSliceThreads, "one bit of `mine` per bias of a thread");
    for (int i = tid, k = 0; i < nb; i += kSliceThreads, ++k) {
        const int id = bi[i];
        uint32_t c;
        if (!index_of(id, c)) continue;
        if (atomicOr(&word[c], kHasBias) & kHasBias) atomicOr(&word[c], kManyBiases);
        else mine |= 1u << k;
    }
    __syncthreads();
    T *x = static_cast<T *>(a.logits) + (size_t)row * (size_t)a.ld;
    /* a lane takes a sector, four lanes a line, and a line with anything in it
     * is read and written whole; rows that do not start on 32 bytes, and the
     * row's last line, go by element */
    const bool lines = (reinterpret_cast<uintptr_t>(x) & 31) == 0;
    for (int s0 = tid; s0 * VE < width; s0 += kSliceThreads) {  // width / VE is a multiple of 32: whole warps
        const int at = s0 * VE;
        uint32_t w[VE], change = 0u;
#pragma unroll
        for (int e = 0; e < VE; e += 4) {
            const uint4 q = *reinterpret_cast<const uint4 *>(word + at + e);
            w[e] = q.x, w[e + 1] = q.y, w[e + 2] = q.z, w[e + 3] = q.w;
        }
#pragma unroll
        for (int e = 0; e < VE; ++e)
            if (w[e] && !(w[e] & kHasBias)) change |= 1u << e;
        const int c = ((at / BLK << sh) + (int)mine_c) * BLK + at % BLK;
        if (mask && change) change &= mask_bits(a, mask, c);
        const uint32_t touched = __ballot_sync(kFull, change != 0u);
        T *p = x + c;
        if ((touched >> (tid & 28) & 15u) && lines && (int64_t)(c - c % BLK) + BLK <= a.vocab) {
            Sector s = sector_load(p);
            if (change) sector_penalise<T>(s, w, change, rules);
            sector_store(p, s);
        } else if (change) {
#pragma unroll
            for (int e = 0; e < VE; ++e)
                if (change >> e & 1u) logit_store(p + e, penalised(logit_load(p + e), w[e], rules));
        }
    }
    if (nb) __syncthreads();  // the lines are written; biased logits were written as they were read
    for (int i0 = 0, k = 0; i0 < nb; i0 += kSliceThreads, ++k) {  // whole warps
        const int i = i0 + tid;
        const int id = i < nb ? bi[i] : 0;
        const bool on = (mine >> k & 1u) && allowed(mask, id);
        uint32_t c = 0u;
        const uint32_t w = on && index_of(id, c) ? word[c] : 0u;
        float b = on ? bv[i] : 0.0f;
        for (uint32_t m = __ballot_sync(kFull, on && (w & kManyBiases)); m; m &= m - 1) {
            const int l = __ffs(m) - 1;
            const float all = bias_sum(bi, bv, nb, __shfl_sync(kFull, id, l));
            if ((tid & 31) == l) b = all;
        }
        if (on) {
            T *p = x + (id - a.v_begin);
            logit_store(p, __fadd_rn(penalised(logit_load(p), w, rules), b));
        }
    }
}

}  // namespace noel
