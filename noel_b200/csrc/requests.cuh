/*
 * Sampling with every row's own temperature, top-k, top-p and min-p
 * (include/noel_requests.h has the definition).
 *
 * Whatever a row's settings leave is a beginning of its ids in the order (x
 * descending, id ascending): all ids whose key (a number that orders as x
 * does) is above some key K, and the first few of those with key K.  So a row
 * is settled by finding K, first by counting (top-k), then by weights
 * (top-p), and then one walk in the order of ids.
 */
#pragma once

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <stdint.h>

namespace noel {

namespace cg = cooperative_groups;

struct RequestArgs {
    const void *logits;  // [batch][ld]
    int64_t ld;
    int batch, vocab;
    const float *temperature, *top_p, *min_p;
    const int32_t *top_k;
    const float *u;
    int32_t *ids, *counts;
    float *probs;
    int per;             // elements of a row to a CTA of its cluster
    bool resident;       // they fit the shared memory
};

constexpr int kReqThreads = 512;
constexpr int kReqWarps = kReqThreads / 32;
constexpr int kReqBins = 1024;
constexpr int kReqMaxCluster = 8;
constexpr int kReqFraction = 43;  // bits behind the point of a weight: 2^20 of them fit 64 bits, and e^-30 is not 0

/* An element as fp32 that compares as it is drawn: NaN below everything, one zero. */
__device__ __forceinline__ float req_value(float x) { return x != x ? -INFINITY : x + 0.0f; }
__device__ __forceinline__ float req_value(__nv_bfloat16 x) { return req_value(__bfloat162float(x)); }
/* a number that orders as x does */
__device__ __forceinline__ uint32_t req_key(float x) {
    const uint32_t b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float req_unkey(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

/* One row's settings. */
struct ReqRow {
    float m;          // its largest logit
    double inv_t;
    bool greedy;
    uint32_t floor;   // key of the smallest value left by the temperature and by min-p
    int k;            // 0: off
    double p;         // 1: off
    float u;
};

__device__ __forceinline__ double req_exp(const ReqRow &r, float x) {
    return x == r.m ? 1.0 : exp(((double)x - (double)r.m) * r.inv_t);
}
__device__ __forceinline__ uint64_t req_weight(const ReqRow &r, float x) {
    return __double2ull_rn(req_exp(r, x) * (double)(1ull << kReqFraction));
}

__device__ __forceinline__ ReqRow req_row(const RequestArgs &a, int b, float m) {
    ReqRow r;
    const float t = a.temperature ? a.temperature[b] : 1.0f;
    const float least = a.min_p ? a.min_p[b] : 0.0f, p = a.top_p ? a.top_p[b] : 1.0f;
    r.m = m;
    r.greedy = !(t > 0.0f);
    r.inv_t = 1.0 / (double)t;
    r.k = a.top_k ? a.top_k[b] : 0;
    if (r.k <= 0 || r.k >= a.vocab) r.k = 0;
    r.p = p < 1.0f ? fmax((double)p, 0.0) : 1.0;
    const float u = a.u[b];
    r.u = u > 0.0f ? fminf(u, 1.0f) : 0.0f;
    /* in 64 bits, then the smallest fp32 number that is not below */
    double floor = (double)m - 30.0 * (double)t;
    if (least >= 1.0f) floor = (double)m;  // whatever the temperature: an infinite one times ln 1 is NaN
    else if (least > 0.0f) floor = fmax(floor, (double)m + (double)t * log((double)least));
    float f = __double2float_ru(floor);
    if (!(f > -INFINITY)) f = -3.402823466e38f;  // -infinity is never left (an infinite temperature gives NaN here)
    if (isinf(m)) f = m;
    r.floor = req_key(f + 0.0f);
    return r;
}

/* Sum of counts and weights, and its running sums over the CTA's threads. */
struct ReqSum {
    uint32_t n;
    uint64_t w;
};
__device__ __forceinline__ ReqSum operator+(ReqSum a, ReqSum b) { return {a.n + b.n, a.w + b.w}; }
__device__ __forceinline__ ReqSum req_shfl_up(ReqSum v, int by) {
    return {__shfl_up_sync(0xFFFFFFFFu, v.n, by), __shfl_up_sync(0xFFFFFFFFu, v.w, by)};
}

struct ReqShared {
    uint32_t n[kReqBins], lo[kReqBins], hi[kReqBins];  // this CTA's histogram: counts and weights in two words
    uint32_t all_n[kReqBins];                          // the row's
    uint64_t all_w[kReqBins];
    uint64_t mail[2][kReqMaxCluster][2];               // two words from each CTA of the cluster
    ReqSum warp[kReqWarps];
    ReqSum total;
    uint32_t found_bin;
    ReqSum found_above;
    uint32_t warp_n[kReqWarps];
    uint32_t red[kReqWarps];
    int32_t cut_id;
};

template <typename T>
struct ReqSlice {
    const T *global, *shared;
    int n, first;  // elements and the id of the first one
    bool resident;
    __device__ __forceinline__ float at(int i) const { return req_value(resident ? shared[i] : global[i]); }
};

/* every CTA's two words, in the order of ranks (the returned array stays until the second next call) */
__device__ __forceinline__ const uint64_t (*req_exchange(ReqShared &s, int &turn, uint64_t x, uint64_t y))[2] {
    cg::cluster_group cluster = cg::this_cluster();
    const int me = cluster.block_rank(), n = cluster.num_blocks();
    turn ^= 1;
    if ((int)threadIdx.x < n) {
        ReqShared *to = cluster.map_shared_rank(&s, threadIdx.x);
        to->mail[turn][me][0] = x;
        to->mail[turn][me][1] = y;
    }
    cluster.sync();
    return s.mail[turn];
}

/* Inclusive running sums over the CTA's threads; the CTA's sum in s.total. */
__device__ __forceinline__ ReqSum req_scan(ReqShared &s, ReqSum v) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const ReqSum o = req_shfl_up(v, d);
        if (lane >= d) v = v + o;
    }
    if (lane == 31) s.warp[warp] = v;
    __syncthreads();
    ReqSum before = {0, 0};
    for (int w = 0; w < kReqWarps; ++w) {
        if (w < warp) before = before + s.warp[w];
    }
    if (threadIdx.x == kReqThreads - 1) s.total = before + v;
    __syncthreads();
    return before + v;
}

struct ReqCut {
    uint32_t key;   // ids above it are left, and
    uint32_t ties;  // the first so many at it
    ReqSum above;   // of the ids above it
    bool some;      // false: nothing is cut
};

/*
 * The cut at which the row's ids with keys in (lo, hi], largest first, reach
 * a count or (by_weight) a weight: a histogram of 1024 ranges of keys over the
 * range, then of the one that holds the cut, until ranges are single keys.
 * want_share: the weight is that share of all in the range.
 */
template <typename T>
__device__ ReqCut req_cut(const ReqSlice<T> &sl, ReqShared &s, const ReqRow &r, uint32_t lo, uint32_t hi, bool by_weight,
                          uint32_t want_n, double want_share, const uint64_t *all_weight) {
    cg::cluster_group cluster = cg::this_cluster();
    const int me = cluster.block_rank(), nc = cluster.num_blocks(), tid = threadIdx.x;
    ReqSum above = {0, 0};
    uint64_t want_w = 0;
    auto share = [&](uint64_t of) {  // the smallest whole weight that is at least that share
        const uint64_t f = (uint64_t)(want_share * 18446744073709551616.0);
        const uint64_t up = __umul64hi(f, of);
        return up + (f * of != 0);
    };
    if (by_weight && all_weight) want_w = share(*all_weight);
    bool first = true;
    for (;;) {
        const uint32_t span = hi - lo;
        const int shift = span <= kReqBins ? 0 : 32 - __clz((span - 1) / kReqBins);
        for (int i = tid; i < kReqBins; i += kReqThreads) s.n[i] = s.lo[i] = s.hi[i] = 0;
        __syncthreads();
        for (int i = tid; i < sl.n; i += kReqThreads) {
            const float x = sl.at(i);
            const uint32_t key = req_key(x);
            if (key > lo && key <= hi) {
                const uint32_t bin = (hi - key) >> shift;
                const uint64_t w = req_weight(r, x);
                atomicAdd(&s.n[bin], 1u);
                const uint32_t wl = (uint32_t)w, old = atomicAdd(&s.lo[bin], wl);
                const uint32_t carry = old + wl < old;
                if ((uint32_t)(w >> 32) + carry) atomicAdd(&s.hi[bin], (uint32_t)(w >> 32) + carry);
            }
        }
        cluster.sync();
        /* each CTA adds up its share of the ranges over the cluster and tells everyone */
        const int each = kReqBins / nc;
        for (int i = tid; i < each; i += kReqThreads) {
            const int bin = me * each + i;
            uint32_t n = 0;
            uint64_t w = 0;
            for (int c = 0; c < nc; ++c) {
                const ReqShared *o = cluster.map_shared_rank(&s, c);
                n += o->n[bin];
                w += (uint64_t)o->hi[bin] << 32 | o->lo[bin];
            }
            for (int c = 0; c < nc; ++c) {
                ReqShared *o = cluster.map_shared_rank(&s, c);
                o->all_n[bin] = n;
                o->all_w[bin] = w;
            }
        }
        if (tid == 0) s.found_bin = kReqBins;
        cluster.sync();
        constexpr int kEach = kReqBins / kReqThreads;
        ReqSum mine = {0, 0};
        for (int i = 0; i < kEach; ++i) mine = mine + ReqSum{s.all_n[tid * kEach + i], s.all_w[tid * kEach + i]};
        const ReqSum run = req_scan(s, mine);
        if (by_weight && first && !all_weight) want_w = share(s.total.w);
        if (by_weight && want_w == 0) want_w = 1;
        first = false;
        ReqSum before = {above.n + run.n - mine.n, above.w + run.w - mine.w};
        for (int i = 0; i < kEach; ++i) {
            const ReqSum in = {s.all_n[tid * kEach + i], s.all_w[tid * kEach + i]}, after = before + in;
            const bool reached = by_weight ? after.w >= want_w : after.n >= want_n;
            const bool earlier = by_weight ? before.w >= want_w : before.n >= want_n;
            if (reached && !earlier) s.found_bin = tid * kEach + i, s.found_above = before;
            before = after;
        }
        __syncthreads();
        const uint32_t bin = s.found_bin;
        if (bin == kReqBins) return {lo, 0, above + s.total, false};
        above = s.found_above;
        if (shift == 0) {
            const uint32_t key = hi - bin, n = s.all_n[bin];
            __syncthreads();
            uint32_t ties = n;
            if (by_weight) {
                const uint64_t w = req_weight(r, req_unkey(key)), need = want_w - above.w;
                ties = (uint32_t)min((uint64_t)n, (need + w - 1) / w);
            } else {
                ties = want_n - above.n;
            }
            return {key, ties, above, true};
        }
        hi -= bin << shift;
        lo = hi - lo > 1u << shift ? hi - (1u << shift) : lo;
        __syncthreads();
    }
}

/*
 * A cluster of CTAs to a row, each with a part of it in shared memory (read
 * from global memory each time where it does not fit).
 */
template <typename T>
__global__ void __launch_bounds__(kReqThreads) sample_requests_kernel(const __grid_constant__ RequestArgs a) {
    extern __shared__ __align__(16) unsigned char req_raw[];
    __shared__ ReqShared s;
    cg::cluster_group cluster = cg::this_cluster();
    const int me = cluster.block_rank(), nc = cluster.num_blocks();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int b = blockIdx.x / nc;
    int turn = 0;
    /* every CTA of the cluster is there before one writes into another's memory: see the wait below */
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");

    ReqSlice<T> sl;
    sl.first = me * a.per;
    sl.n = max(0, min(a.per, a.vocab - sl.first));
    sl.global = static_cast<const T *>(a.logits) + (int64_t)b * a.ld + sl.first;
    sl.shared = reinterpret_cast<T *>(req_raw);
    sl.resident = a.resident;

    /* the row's largest logit */
    float top = -INFINITY;
    T *keep = reinterpret_cast<T *>(req_raw);
#pragma unroll 8
    for (int i = tid; i < sl.n; i += kReqThreads) {
        const T raw = sl.global[i];
        if (a.resident) keep[i] = raw;
        top = fmaxf(top, req_value(raw));
    }
    const uint32_t most = __reduce_max_sync(0xFFFFFFFFu, req_key(top));
    if (lane == 0) s.red[warp] = most;
    __syncthreads();
    uint32_t key = 0;
    for (int w = 0; w < kReqWarps; ++w) key = max(key, s.red[w]);
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    const uint64_t(*all)[2] = req_exchange(s, turn, key, 0);
    for (int c = 0; c < nc; ++c) key = max(key, (uint32_t)all[c][0]);
    const float m = req_unkey(key);
    if (m == -INFINITY) {
        if (me == 0 && tid == 0) {
            a.ids[b] = -1;
            if (a.probs) a.probs[b] = 0.0f;
            if (a.counts) a.counts[b] = 0;
        }
        return;
    }
    const ReqRow r = req_row(a, b, m);
    if (r.greedy) {
        int32_t id = 0x7FFFFFFF;
        for (int i = tid; i < sl.n; i += kReqThreads)
            if (sl.at(i) == m) {
                id = sl.first + i;
                break;
            }
        id = __reduce_min_sync(0xFFFFFFFFu, id);
        __syncthreads();
        if (lane == 0) s.red[warp] = (uint32_t)id;
        __syncthreads();
        for (int w = 0; w < kReqWarps; ++w) id = min(id, (int32_t)s.red[w]);
        all = req_exchange(s, turn, (uint64_t)id, 0);
        for (int c = 0; c < nc; ++c) id = min(id, (int32_t)all[c][0]);
        if (me == 0 && tid == 0) {
            a.ids[b] = id;
            if (a.probs) a.probs[b] = 1.0f;
            if (a.counts) a.counts[b] = 1;
        }
        return;
    }

    ReqCut cut = {r.floor - 1, 0, {0, 0}, false};
    if (r.k) cut = req_cut(sl, s, r, r.floor - 1, key, false, (uint32_t)r.k, 0.0, nullptr);
    if (r.p < 1.0) {
        uint64_t all_weight = cut.above.w;
        if (cut.some) all_weight += cut.ties * req_weight(r, req_unkey(cut.key));
        const ReqCut by_p = req_cut(sl, s, r, cut.some ? cut.key - 1 : cut.key, key, true, 0, r.p, r.k ? &all_weight : nullptr);
        if (by_p.some) cut = by_p;
    }

    /* of several ids at the cut, the lowest */
    int32_t cut_id = 0x7FFFFFFF;
    const int region = a.per / kReqWarps, begin = warp * region, end = min(sl.n, begin + region);
    if (cut.some) {
        uint32_t n = 0;
        for (int i = begin + lane; i < end; i += 32) n += req_key(sl.at(i)) == cut.key;
        n = __reduce_add_sync(0xFFFFFFFFu, n);
        if (lane == 0) s.warp_n[warp] = n;
        __syncthreads();
        uint32_t mine = 0;
        for (int w = 0; w < kReqWarps; ++w) mine += s.warp_n[w];
        all = req_exchange(s, turn, mine, 0);
        uint32_t before = 0;
        for (int c = 0; c < me; ++c) before += (uint32_t)all[c][0];
        for (int w = 0; w < warp; ++w) before += s.warp_n[w];
        if (tid == 0) s.cut_id = -1;
        __syncthreads();
        if (before < cut.ties && before + n >= cut.ties) {  // the last id left is in this warp's region
            for (int i = begin; i < end; i += 32) {
                const bool tie = i + lane < end && req_key(sl.at(i + lane)) == cut.key;
                const uint32_t bits = __ballot_sync(0xFFFFFFFFu, tie);
                const uint32_t rank = before + __popc(bits & ((1u << lane) - 1)) + 1;
                if (tie && rank == cut.ties) s.cut_id = sl.first + i + lane;
                before += __popc(bits);
            }
        }
        __syncthreads();
        all = req_exchange(s, turn, (uint64_t)(uint32_t)s.cut_id, 0);
        for (int c = 0; c < nc; ++c)
            if ((int32_t)all[c][0] >= 0) cut_id = (int32_t)all[c][0];
    }
    auto weight = [&](int i) -> uint64_t {  // of element i, 0 where it is not left
        const float x = sl.at(i);
        const uint32_t k = req_key(x);
        return k > cut.key || (cut.some && k == cut.key && sl.first + i <= cut_id) ? req_weight(r, x) : 0;
    };

    /* the walk: sums of regions, then the one that the draw ends in */
    ReqSum sum = {0, 0};
    for (int i = begin + lane; i < end; i += 32) {
        const uint64_t w = weight(i);
        sum = sum + ReqSum{w != 0, w};
    }
#pragma unroll
    for (int d = 16; d; d >>= 1)
        sum = sum + ReqSum{__shfl_xor_sync(0xFFFFFFFFu, sum.n, d), __shfl_xor_sync(0xFFFFFFFFu, sum.w, d)};
    __syncthreads();
    if (lane == 0) s.warp[warp] = sum;
    __syncthreads();
    ReqSum cta = {0, 0};
    for (int w = 0; w < kReqWarps; ++w) cta = cta + s.warp[w];
    all = req_exchange(s, turn, cta.w, cta.n);
    uint64_t total = 0, before = 0;
    uint32_t count = 0;
    for (int c = 0; c < nc; ++c) {
        if (c < me) before += all[c][0];
        total += all[c][0];
        count += (uint32_t)all[c][1];
    }
    for (int w = 0; w < warp; ++w) before += s.warp[w].w;
    uint64_t target = r.u >= 1.0f ? total : __umul64hi((uint64_t)((double)r.u * 18446744073709551616.0), total);
    if (target >= total) target = total - 1;
    if (before <= target && target < before + sum.w) {
        bool found = false;
        for (int i = begin; i < end && !found; i += 32) {
            const uint64_t w = i + lane < end ? weight(i + lane) : 0;
            uint64_t run = w;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const uint64_t o = __shfl_up_sync(0xFFFFFFFFu, run, d);
                if (lane >= d) run += o;
            }
            const uint32_t over = __ballot_sync(0xFFFFFFFFu, before + run > target);
            if (over) {
                found = true;
                if (lane == __ffs(over) - 1) {
                    a.ids[b] = sl.first + i + lane;
                    if (a.probs)
                        a.probs[b] = (float)(req_exp(r, sl.at(i + lane)) * (double)(1ull << kReqFraction) / (double)total);
                    if (a.counts) a.counts[b] = (int32_t)count;
                }
            }
            before += __shfl_sync(0xFFFFFFFFu, run, 31);
        }
    }
}

}  // namespace noel
