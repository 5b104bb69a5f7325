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
    int32_t *status;     // [batch] PassStatus
    int per;             // elements of a row to a CTA of its cluster
    bool resident;       // they fit the shared memory
};

constexpr int kReqThreads = 512;
constexpr int kReqWarps = kReqThreads / 32;
constexpr int kReqBins = 1024;
constexpr int kReqList = 1024;
constexpr int kReqMaxCluster = 16;
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
    double c64;       // 64 log2(e) / T
    bool greedy;
    uint32_t floor;   // key of the smallest value left by the temperature and by min-p
    int k;            // 0: off
    double p;         // 1: off
    float u;
};

constexpr int kReqTable = 64;  // 2^(j / 64), in shared memory

__device__ __forceinline__ void req_table(double *table) {
    if (threadIdx.x < kReqTable) table[threadIdx.x] = exp2((double)threadIdx.x / kReqTable);
}

/*
 * exp((x - m) / T) for x from the row's floor on: 2^(t / 64) with t from -2771
 * to 0, its whole part by the table and the exponent, the rest (half of one
 * at most, z = its natural exponent, below 0.0055) by the exponential
 * series, whose next term z^6 / 720 is below 2^-54.
 */
__device__ __forceinline__ double req_exp(const ReqRow &r, float x, const double *table) {
    if (x == r.m) return 1.0;  // infinite ones too
    const double t = ((double)x - (double)r.m) * r.c64;
    const double up = t + 6755399441055744.0;  // 1.5 * 2^52: its low bits are t to the nearest whole number
    const int k = __double2loint(up);
    const double z = (t - (up - 6755399441055744.0)) * (0.69314718055994531 / kReqTable);
    double v = fma(1.0 / 120, z, 1.0 / 24);
    v = fma(v, z, 1.0 / 6);
    v = fma(v, z, 0.5);
    v = fma(v, z, 1.0);
    v = fma(v, z, 1.0);
    v *= table[k & (kReqTable - 1)];
    return __hiloint2double(__double2hiint(v) + (k >> 6 << 20), __double2loint(v));
}
/* in 2^-43, to the nearest */
__device__ __forceinline__ uint64_t req_weight(const ReqRow &r, float x, const double *table) {
    const double v = fma(req_exp(r, x, table), (double)(1ull << kReqFraction), 4503599627370496.0);  // 2^52: the number is its low bits
    return (uint64_t)__double_as_longlong(v) & 0xFFFFFFFFFFFFFull;
}

__device__ __forceinline__ ReqRow req_row(const RequestArgs &a, int b, float m, float u) {
    ReqRow r;
    const float t = a.temperature ? a.temperature[b] : 1.0f;
    const float least = a.min_p ? a.min_p[b] : 0.0f, p = a.top_p ? a.top_p[b] : 1.0f;
    r.m = m;
    r.greedy = !(t > 0.0f);
    r.c64 = kReqTable * 1.4426950408889634 / (double)t;
    r.k = a.top_k ? a.top_k[b] : 0;
    if (r.k <= 0 || r.k >= a.vocab) r.k = 0;
    r.p = p < 1.0f ? fmax((double)p, 0.0) : 1.0;
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
    uint32_t ends[2];
    uint64_t before;
    uint32_t region;
    uint32_t rows[kReqWarps];
    double table[kReqTable];
    uint64_t list[kReqList];  // the elements around a cut, of the whole row
    uint32_t count;
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
    int32_t id;     // the last of those at it, or -1: not known
    uint64_t kept;  // weight of all that is left
};

/* The CTA's list of size (a power of two) numbers, largest first. */
template <int THREADS>
__device__ __forceinline__ void req_sort(uint64_t *list, int size) {
    for (int width = 2; width <= size; width <<= 1)
        for (int d = width >> 1; d; d >>= 1) {
            for (int i = threadIdx.x; i < size / 2; i += THREADS) {
                const int lo = 2 * i - (i & (d - 1)), up = lo + d;
                const uint64_t x = list[lo], y = list[up];
                if ((x < y) == ((lo & width) == 0)) list[lo] = y, list[up] = x;
            }
            __syncthreads();
        }
}

/* req_cut where few elements (n of the row) are in the range that holds the cut: every CTA sorts all of them. */
template <typename T>
__device__ ReqCut req_cut_list(const ReqSlice<T> &sl, ReqShared &s, const ReqRow &r, uint32_t lo, uint32_t hi, uint32_t n,
                               ReqSum above, bool by_weight, uint32_t want_n, uint64_t want_w, int &turn) {
    cg::cluster_group cluster = cg::this_cluster();
    const int me = cluster.block_rank(), nc = cluster.num_blocks(), tid = threadIdx.x;
    if (tid == 0) s.count = 0;
    __syncthreads();
    uint64_t *mine = s.all_w;  // what it held has been used
    for (int i = tid; i < sl.n; i += kReqThreads) {
        const uint32_t key = req_key(sl.at(i));
        if (key > lo && key <= hi) mine[atomicAdd(&s.count, 1u)] = (uint64_t)key << 32 | (0xFFFFFFFFu - (uint32_t)(sl.first + i));
    }
    __syncthreads();
    const uint32_t have = s.count;
    const uint64_t(*all)[2] = req_exchange(s, turn, have, 0);
    uint32_t at = 0;
    for (int c = 0; c < me; ++c) at += (uint32_t)all[c][0];
    for (int c = 0; c < nc; ++c) {
        uint64_t *to = cluster.map_shared_rank(&s, c)->list + at;
        for (uint32_t i = tid; i < have; i += kReqThreads) to[i] = mine[i];
    }
    cluster.sync();
    int size = 2;
    while (size < (int)n) size <<= 1;
    for (int i = n + tid; i < size; i += kReqThreads) s.list[i] = 0;
    __syncthreads();
    req_sort<kReqThreads>(s.list, size);
    constexpr int kEach = kReqList / kReqThreads;
    ReqSum in[kEach], sum = {0, 0};
    for (int i = 0; i < kEach; ++i) {
        const uint32_t j = tid * kEach + i;
        in[i] = j < n ? ReqSum{1, req_weight(r, req_unkey((uint32_t)(s.list[j] >> 32)), s.table)} : ReqSum{0, 0};
        sum = sum + in[i];
    }
    const ReqSum run = req_scan(s, sum);
    ReqSum before = {above.n + run.n - sum.n, above.w + run.w - sum.w};
    for (int i = 0; i < kEach; ++i) {
        const ReqSum after = before + in[i];
        const bool reached = by_weight ? after.w >= want_w : after.n >= want_n;
        const bool earlier = by_weight ? before.w >= want_w : before.n >= want_n;
        if (reached && !earlier) s.found_bin = tid * kEach + i, s.found_above = after;
        before = after;
    }
    __syncthreads();
    const uint64_t last = s.list[s.found_bin];
    return {(uint32_t)(last >> 32), 1, s.found_above, true, (int32_t)(0xFFFFFFFFu - (uint32_t)last), s.found_above.w};
}

/*
 * The cut at which the row's ids with keys in (lo, hi], largest first, reach
 * a count or (by_weight) a weight: a histogram of 1024 ranges of keys over the
 * range, then of the one that holds the cut, until ranges are single keys.
 * want_share: the weight is that share of all in the range.
 */
template <typename T>
__device__ ReqCut req_cut(const ReqSlice<T> &sl, ReqShared &s, const ReqRow &r, uint32_t lo, uint32_t hi, bool by_weight,
                          uint32_t want_n, double want_share, const uint64_t *all_weight, int &turn) {
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
    /*
     * The first histogram of a wide range goes by values, evenly between its ends: by keys, which are denser near
     * zero, most elements would meet in a few bins.
     */
    const float top = req_unkey(hi), scale = ((float)kReqBins - 0.5f) / (top - req_unkey(lo + 1));
    bool even = hi - lo > 64 * kReqBins && scale > 0.0f && scale < 3e38f;
    auto even_bin = [&](uint32_t key) { return min((uint32_t)((top - req_unkey(key)) * scale), (uint32_t)kReqBins - 1); };
    for (;;) {
        const uint32_t span = hi - lo;
        const int shift = span <= kReqBins ? 0 : 32 - __clz((span - 1) / kReqBins);
        for (int i = tid; i < kReqBins; i += kReqThreads) s.n[i] = s.lo[i] = s.hi[i] = 0;
        __syncthreads();
        for (int i = tid; i < sl.n; i += kReqThreads) {
            const float x = sl.at(i);
            const uint32_t key = req_key(x);
            if (key > lo && key <= hi) {
                const uint32_t bin = even ? even_bin(key) : (hi - key) >> shift;
                const uint64_t w = req_weight(r, x, s.table);
                atomicAdd(&s.n[bin], 1u);
                const uint32_t wl = (uint32_t)w, old = atomicAdd(&s.lo[bin], wl);
                const uint32_t wh = (uint32_t)(w >> 32) + (old + wl < old);
                if (wh) atomicAdd(&s.hi[bin], wh);
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
        if (bin == kReqBins) return {lo, 0, above + s.total, false, -1, 0};
        above = s.found_above;
        if (even) {
            /* the bin's keys: bins fall as keys rise, so both ends are found by halving */
            if (tid < 2) {
                uint32_t in = lo, out = hi;  // the largest key whose bin is bin (thread 0) or the next one (thread 1) at least
                if (even_bin(out) >= bin + tid) in = out;
                while (out - in > 1) {
                    const uint32_t mid = in + (out - in) / 2;
                    if (even_bin(mid) >= bin + tid) in = mid;
                    else out = mid;
                }
                s.ends[tid] = in;
            }
            __syncthreads();
            hi = s.ends[0], lo = s.ends[1];
            even = false;
            const uint32_t in = s.all_n[bin];
            if (in <= kReqList) return req_cut_list(sl, s, r, lo, hi, in, above, by_weight, want_n, want_w, turn);
            __syncthreads();
            continue;
        }
        if (shift == 0) {
            const uint32_t key = hi - bin, n = s.all_n[bin];
            __syncthreads();
            uint32_t ties = n;
            if (by_weight) {
                const uint64_t w = req_weight(r, req_unkey(key), s.table), need = want_w - above.w;
                ties = (uint32_t)min((uint64_t)n, (need + w - 1) / w);
            } else {
                ties = want_n - above.n;
            }
            return {key, ties, above, true, -1, above.w + ties * req_weight(r, req_unkey(key), s.table)};
        }
        hi -= bin << shift;
        lo = hi - lo > 1u << shift ? hi - (1u << shift) : lo;
        __syncthreads();
    }
}

/*
 * A cluster of CTAs to a row, each with a part of it in shared memory (read
 * from global memory each time where it does not fit): the largest logit, the
 * cut, the exact sums of every warp's region, and the region that the draw
 * ends in.  A row of 152,064 fp32 alone takes 14 us in a cluster of 16 where
 * nothing is cut (3.4 to load it, 4.7 for the weights' sums; a cluster of 8:
 * 20) and 35 where top-p cuts (5.7 for the histogram, 4 to add it up over the
 * cluster, 2.8 and 3.9 to collect and sort what is around the cut): latency,
 * and the issue of about 60 instructions an id.  A batch of rows that all come
 * here takes 4 to 5 us a row where something is cut and 1.8 where nothing is
 * (1024 rows of 152,064: 4.5 to 4.8 ms under top-p 0.9 with 6,000 to 17,000 ids
 * left, 4.3 under top-k 5000, 1.8 without filters): 45 % of the issue slots,
 * warps waiting at the cluster's barriers above all.
 */
template <typename T>
__device__ void req_sample_row(const RequestArgs &a, ReqShared &s, unsigned char *req_raw, int b, int &turn) {
    cg::cluster_group cluster = cg::this_cluster();
    const int me = cluster.block_rank(), nc = cluster.num_blocks();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

    ReqSlice<T> sl;
    sl.first = me * a.per;
    sl.n = max(0, min(a.per, a.vocab - sl.first));
    sl.global = static_cast<const T *>(a.logits) + (int64_t)b * a.ld + sl.first;
    sl.shared = reinterpret_cast<T *>(req_raw);
    sl.resident = a.resident;

    /* the row's largest logit */
    float top = -INFINITY;
    T *keep = reinterpret_cast<T *>(req_raw);
#pragma unroll 16
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
    const ReqRow r = req_row(a, b, m, a.u[b]);
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

    ReqCut cut = {r.floor - 1, 0, {0, 0}, false, -1, 0};
    if (r.k) cut = req_cut(sl, s, r, r.floor - 1, key, false, (uint32_t)r.k, 0.0, nullptr, turn);
    if (r.p < 1.0) {
        uint64_t all_weight = cut.above.w;
        if (cut.some) all_weight = cut.kept;
        const ReqCut by_p = req_cut(sl, s, r, cut.some ? cut.key - 1 : cut.key, key, true, 0, r.p, r.k ? &all_weight : nullptr, turn);
        if (by_p.some) cut = by_p;
    }

    /* of several ids at the cut, the lowest */
    int32_t cut_id = 0x7FFFFFFF;
    const int region = a.per / kReqWarps, begin = warp * region, end = min(sl.n, begin + region);
    if (cut.some && cut.id >= 0) {
        cut_id = cut.id;
    } else if (cut.some) {
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
        return k > cut.key || (cut.some && k == cut.key && sl.first + i <= cut_id) ? req_weight(r, x, s.table) : 0;
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
    uint64_t target = r.u >= 1.0f ? total : __umul64hi((uint64_t)((double)r.u * 18446744073709551616.0), total);
    if (target >= total) target = total - 1;
    if (target < before || target - before >= cta.w) return;  // in another CTA's part
    for (int w = 0; w < warp; ++w) before += s.warp[w].w;
    if (lane == 0 && before <= target && target - before < sum.w) s.region = warp, s.before = before;
    __syncthreads();
    /* the region that it ends in, some neighbouring elements to a thread */
    const int each = (region + kReqThreads - 1) / kReqThreads;
    const int from = s.region * region + tid * each, to = min(min(sl.n, (int)(s.region + 1) * region), from + each);
    uint64_t mine = 0;
    before = s.before;
    for (int i = from; i < to; ++i) mine += weight(i);
    before += req_scan(s, {0, mine}).w - mine;
    for (int i = from; i < to; ++i) {
        const uint64_t w = weight(i);
        if (before <= target && target < before + w) {
            a.ids[b] = sl.first + i;
            if (a.probs) a.probs[b] = (float)(req_exp(r, sl.at(i), s.table) * (double)(1ull << kReqFraction) / (double)total);
            if (a.counts) a.counts[b] = (int32_t)count;
        }
        before += w;
    }
}

/* what sample_pass_kernel says of a row: done, not taken (by its settings), or not settled */
enum PassStatus { kPassSettled, kPassSkipped, kPassUnsettled };
/* greatest logit; top-k; min-p; top-p alone; none of sample_pass_kernel's */
enum PassKind { kPassGreedy, kPassCount, kPassLeast, kPassShare, kPassNot };
constexpr int kPassTopK = 1024;  // largest top_k of sample_pass_kernel

/* What a row's settings come to before its largest logit is known. */
struct PassRow {
    PassKind kind;
    int k;
    float t, p, floor_t;  // floor = largest + floor_t (a little below, so that nothing is dropped too early)
    float c;              // log2(e) / T
};

__device__ __forceinline__ PassRow pass_row(const RequestArgs &a, int b) {
    PassRow r;
    const float t = a.temperature ? a.temperature[b] : 1.0f;
    const float least = a.min_p ? a.min_p[b] : 0.0f;
    r.p = a.top_p ? a.top_p[b] : 1.0f;
    r.k = a.top_k ? a.top_k[b] : 0;
    r.t = t;
    r.c = (float)(1.4426950408889634 / (double)t);
    r.floor_t = -30.0f * t;
    if (least > 0.0f) r.floor_t = fmaxf(r.floor_t, t * logf(fminf(least, 1.0f)) * 1.0001f);
    const bool plain = t >= 1e-3f && t <= 1e4f;  // what fp32 bounds below are made for
    if (!(t > 0.0f)) r.kind = kPassGreedy, r.k = 1, r.floor_t = 0.0f;
    else if (!plain) r.kind = kPassNot;
    else if (r.k > 0 && r.k <= kPassTopK) r.kind = kPassCount;
    else if (least > 0.0f && !(r.k > 0 && r.k < a.vocab)) r.kind = kPassLeast;
    else if (r.p < 1.0f && !(r.k > 0 && r.k < a.vocab)) r.kind = kPassShare;
    else r.kind = kPassNot;
    return r;
}
/*
 * The rows that sample_pass_kernel does not take, by their settings, as soon
 * as its last CTAs leave room, and then those that it could not settle.  The
 * clusters take them in turn.
 */
template <typename T>
__global__ void __launch_bounds__(kReqThreads) sample_requests_kernel(const __grid_constant__ RequestArgs a) {
    extern __shared__ __align__(16) unsigned char req_raw[];
    __shared__ ReqShared s;
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, n = cluster.num_blocks();
    const uint32_t me = blockIdx.x / n, clusters = gridDim.x / n;
    int turn = 0;
    req_table(s.table);
    cluster.sync();  // every CTA of the cluster is there before one writes into another's memory
    for (int after = 0; after < 2; ++after) {
        if (after) asm volatile("griddepcontrol.wait;" ::: "memory");
        uint32_t rank = 0;
        for (int at = 0; at < a.batch; at += kReqThreads) {
            bool mine = false;
            if (at + tid < a.batch) {
                mine = after ? a.status[at + tid] == kPassUnsettled : pass_row(a, at + tid).kind == kPassNot;
            }
            const uint32_t bits = __ballot_sync(0xFFFFFFFFu, mine);
            __syncthreads();
            if ((tid & 31) == 0) s.rows[tid >> 5] = bits;
            __syncthreads();
            for (int w = 0; w < kReqWarps; ++w)
                for (uint32_t left = s.rows[w]; left; left &= left - 1)
                    if (rank++ % clusters == me) {
                        req_sample_row<T>(a, s, req_raw, at + w * 32 + __ffs(left) - 1, turn);
                        __syncthreads();
                    }
        }
    }
}

/* ----------------------------------------------------- one pass over a row */

/*
 * The rows of a batch in one pass each.  A CTA (or each CTA of a cluster, a
 * part of the row each) reads its elements once and keeps those that may
 * still be left by the row's settings, from a filter that rises as more of
 * the row has been seen:
 *   top-k: the k-th largest so far;
 *   min-p: the largest so far + T ln(min_p);
 *   top-p: what has been dropped weighs at most a share of 1 - top_p of all
 *     that has been seen.  That is a bet on the rest of the row, and the row's
 *     end checks it: dropped ids are not left if they weigh at most 1 - top_p
 *     of the whole row together.
 * Then what was kept is sorted and the settings are applied to it with the
 * same whole-number weights as above.  Of what top-p rows dropped only the sum
 * of weights is needed, from fp32 exponentials; its error is bounded, and
 * where the bound leaves the cut open, as where a bet is lost or too much would have
 * to be kept, the row is marked for the kernel above.
 */
constexpr int kPassThreads = 256;
constexpr int kPassWarps = kPassThreads / 32;
constexpr int kPassEach = 16;     // elements of a thread's turn
constexpr int kPassKeep = 4096;   // kept at most
constexpr int kPassFull = kPassKeep / 4 * 3;  // and at most after the filter has risen
constexpr int kPassRises = 5;    // on the way; 3, 5 and 10 are within 2 % of each other in every case measured
constexpr int kPassBins = 1024;
constexpr int kPassSort = 2048;   // of those, at the end

struct PassArgs {
    RequestArgs r;
    int turns, step;  // turns of a warp's part of a row, taken in steps of step (no common divisor)
    bool order;       // the rows that take longest first
};

struct PassShared {
    uint32_t n[kPassBins];
    uint64_t warp[kPassWarps];
    double warp_d[kPassWarps];
    float warp_f[kPassWarps];
    uint32_t count;       // places taken in the list of what is kept
    uint32_t valid;       // and those that were filled, where it ran over
    uint32_t found, found_high;
    int full, lost, left;
    float u;
    double table[kReqTable];
    double top;
    double part_rest[kReqMaxCluster];  // of the cluster's parts: weights dropped,
    float part_rc[kReqMaxCluster];     // their reference,
    float part_f[kReqMaxCluster];      // and the filter
};

/* kept elements: key, then the lower id first */
__device__ __forceinline__ uint64_t pass_pack(float x, int id) {
    return (uint64_t)req_key(x + 0.0f) << 32 | (0xFFFFFFFFu - (uint32_t)id);
}
__device__ __forceinline__ float pass_x(uint64_t e) { return req_unkey((uint32_t)(e >> 32)); }
__device__ __forceinline__ int pass_id(uint64_t e) { return (int)(0xFFFFFFFFu - (uint32_t)e); }

__device__ __forceinline__ float pass_exp2(float t) {
    float w;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"(t));
    return w;
}

/* 16 bytes of a row as values */
template <typename T>
struct PassVec;
template <>
struct PassVec<float> {
    static constexpr int kPer = 4;
    static __device__ __forceinline__ void get(uint4 u, float *v) {
        v[0] = __uint_as_float(u.x), v[1] = __uint_as_float(u.y), v[2] = __uint_as_float(u.z), v[3] = __uint_as_float(u.w);
    }
    static __device__ __forceinline__ uint4 none() { return make_uint4(0xFF800000u, 0xFF800000u, 0xFF800000u, 0xFF800000u); }
};
template <>
struct PassVec<__nv_bfloat16> {
    static constexpr int kPer = 8;
    static __device__ __forceinline__ void get(uint4 u, float *v) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
    static __device__ __forceinline__ uint4 none() { return make_uint4(0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u); }
};
__device__ __forceinline__ uint4 pass_load(const uint4 *p) {
    uint4 u;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "l"(p));
    return u;
}

__device__ __forceinline__ float pass_max(PassShared &s, float v) {  // over the CTA's threads
    for (int d = 16; d; d >>= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, d));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s.warp_f[threadIdx.x >> 5] = v;
    __syncthreads();
    v = s.warp_f[0];
#pragma unroll
    for (int w = 1; w < kPassWarps; ++w) v = fmaxf(v, s.warp_f[w]);
    return v;
}
__device__ __forceinline__ double pass_sum(PassShared &s, double v) {
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s.warp_d[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int w = 0; w < kPassWarps; ++w) v += s.warp_d[w];
    return v;
}
/* inclusive running sum over the CTA's threads, the CTA's sum in all */
__device__ __forceinline__ uint64_t pass_scan(PassShared &s, uint64_t v, uint64_t &all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint64_t o = __shfl_up_sync(0xFFFFFFFFu, v, d);
        if (lane >= d) v += o;
    }
    __syncthreads();
    if (lane == 31) s.warp[warp] = v;
    __syncthreads();
    uint64_t before = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < kPassWarps; ++w) {
        if (w < warp) before += s.warp[w];
        all += s.warp[w];
    }
    return before + v;
}

/* a value that is not above the smallest that the temperature and min-p leave beside a largest logit of m */
__device__ __forceinline__ float pass_floor(const PassRow &r, float m) {
    const float f = m + r.floor_t;
    return fmaxf(f - fabsf(f) * 2e-7f - fabsf(m) * 2e-7f - 1e-37f, -3.402823466e38f);
}

/*
 * The row of place at, where rows with top-p alone or a large top-k come first
 * and the others after them: they take twice the others' time (1024 mixed
 * rows: 100 to 140 us against 50), and the last ones to start would end alone.
 */
__device__ __forceinline__ int pass_order(const RequestArgs &a, PassShared &s, int at) {
    const int each = (a.batch + kPassThreads - 1) / kPassThreads, from = threadIdx.x * each;
    auto slow = [&](int b) {
        const bool t = !a.temperature || a.temperature[b] > 0.0f, least = a.min_p && a.min_p[b] > 0.0f;
        const bool p = a.top_p && a.top_p[b] < 1.0f;
        const int k = a.top_k ? a.top_k[b] : 0;
        return t && (k > 0 ? k > kPassThreads : p && !least);
    };
    uint64_t mine = 0, all;
    for (int b = from; b < min(a.batch, from + each); ++b) mine += slow(b);
    const int before = (int)(pass_scan(s, mine, all) - mine);
    int place_slow = before, place = (int)all + min(from, a.batch) - before;
    for (int b = from; b < min(a.batch, from + each); ++b)
        if ((slow(b) ? place_slow++ : place++) == at) s.left = b;
    __syncthreads();
    const int b = s.left;
    __syncthreads();
    return b;
}

/*
 * Four CTAs to an SM leave a thread 64 registers, which do not hold the row's
 * state beside its end: 50 words of a thread are spilled and read again for
 * fp32 and 20 for bf16.  Of 1024 mixed rows of 152,064 fp32 one
 * takes about 53 us there: 3 for the first filter, 37 for the row (HBM, when
 * all of them are at it), 3 for a last rise where over 256 are kept, 1.7 to rank
 * them, 3 for weights, cuts and the walk; 8.5 for a rise on the way, which top-p
 * rows and large top-k need several of.  Of 1024 rows of 256,000 bf16 with top-p
 * alone one takes 97 us, 65 of them for the row, bound by instruction issue
 * (77 % of the slots, about 22 instructions an id: an exponential each, and
 * the kept ones).  For fp32 it is 54 % of the slots and half of the HBM's rate:
 * warps wait for loads and for what a row's end does in shared memory.
 */
template <typename T>
__global__ void __launch_bounds__(kPassThreads, 4) sample_pass_kernel(const __grid_constant__ PassArgs a) {
    extern __shared__ __align__(16) unsigned char req_raw[];
    uint64_t *keep = reinterpret_cast<uint64_t *>(req_raw);
    __shared__ PassShared s;
    cg::cluster_group cluster = cg::this_cluster();
    const int me = cluster.block_rank(), nc = cluster.num_blocks();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int b = a.order ? pass_order(a.r, s, blockIdx.x / nc) : blockIdx.x / nc;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    using V = PassVec<T>;
    constexpr int kVecs = kPassEach / V::kPer;
    const T *base = static_cast<const T *>(a.r.logits) + (int64_t)b * a.r.ld;
    const int vocab = a.r.vocab;
    const int head = min(vocab, (int)((16 - (reinterpret_cast<uintptr_t>(base) & 15)) & 15) / (int)sizeof(T));
    const int vecs = (vocab - head) / V::kPer;
    const uint4 *body = reinterpret_cast<const uint4 *>(base + head);
    /* a warp's part of the row: whole turns, so that a turn of the CTA is spread over the row */
    const int first = min((int64_t)vecs, (int64_t)(me * kPassWarps + warp) * a.turns * (32 * kVecs));
    const int last = min((int64_t)vecs, (int64_t)first + a.turns * (32 * kVecs));

    uint4 next[kVecs];
    auto load = [&](int turn) {
#pragma unroll
        for (int j = 0; j < kVecs; ++j) {
            const int v = first + turn * (32 * kVecs) + j * 32 + lane;
            next[j] = v < last ? pass_load(body + v) : V::none();
        }
    };
    int turn = 0, ahead = a.step < a.turns ? a.step : 0;  // the turn in x, and the one on its way
    load(0);
    const PassRow row = pass_row(a.r, b);
    if (row.kind == kPassNot) {
        if (me == 0 && tid == 0) a.r.status[b] = kPassSkipped;
        return;  // the whole cluster
    }
    if (tid == 0) s.u = a.r.u[b];
    req_table(s.table);

    if (tid == 0) s.count = 0, s.valid = kPassKeep, s.lost = s.full = 0;
    for (int i = tid; i < kPassBins; i += kPassThreads) s.n[i] = 0;

    float f = -3.402823466e38f;  // elements from f on are kept
    float rc = 0.0f;             // weights of what is dropped are 2^(x c - rc)
    bool weigh = false;
    double rest = 0.0;           // and their sum, of this thread
    float x[kPassEach];
#pragma unroll
    for (int j = 0; j < kVecs; ++j) V::get(next[j], x + j * V::kPer);
    if (a.turns > 1) load(ahead);

    /*
     * The filter that the histogram in s.n of elements from low to hi gives.
     * This CTA has seen 1 / grow of the row; dropped: what its dropped elements
     * weigh, hi's weight being 1.
     */
    auto edge = [&](float hi, float low, float scale, double dropped, double grow) -> float {
        /* counts in the low 14 bits, above them the weights of the bins (of their upper ends) in 2^-36 */
        constexpr int kEach = kPassBins / kPassThreads;
        uint64_t in[kEach], mine = 0, all;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int bin = tid * kEach + i;
            const uint32_t n = s.n[bin];
            in[i] = n;
            if (row.kind == kPassShare && n)
                in[i] += (uint64_t)((float)n * pass_exp2(-(float)bin / scale * row.c) * 6.8719477e10f) << 14;
            mine += in[i];
        }
        const uint64_t begin = pass_scan(s, mine, all) - mine;
        if (tid == 0) s.found = kPassBins, s.top = (double)(all >> 14);
        __syncthreads();
        const uint32_t need = row.kind == kPassCount ? (uint32_t)row.k : 4u;
        uint64_t run = begin;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const uint64_t after = run + in[i];
            if ((uint32_t)(run & 16383) < need && (uint32_t)(after & 16383) >= need) {
                if (row.kind == kPassCount) s.found = tid * kEach + i;
                else s.top = (double)(after >> 14);
            }
            run = after;
        }
        __syncthreads();
        if (row.kind == kPassShare) {
            /*
             * What will have been dropped in the end, as of the part seen so far, may be 3/4 (early on, 1/2) of 1 -
             * top_p of the row's weight; for that the 4 largest so far count once and the others for as much as the
             * part has seen.  The 24 largest of an early part stay: what lies below them is even enough to count on.
             * 1024 nucleus rows of 256,000 bf16 with the 8, 24 and 96 largest 292, 303 and 490 us; with shares of 1/4 and
             * 1/2, 1/2 and 3/4, 3/4 and 9/10 340, 303 and 292 (1024 mixed rows 216, 195 and 192).  A lower filter costs
             * work on each row, a higher one loses more bets where weights fall slowly.
             */
            const double weight = (double)(all >> 14), gone = dropped * 6.8719477e10, seen = weight + gone;
            const double row_weight = seen + (grow - 1.0) * (seen - s.top);
            const double may = (grow > 2.0 ? 0.5 : 0.75) * (1.0 - (double)row.p) * row_weight / grow - gone;
            const uint64_t want = may > 0.0 && may < weight ? (all >> 14) - (uint64_t)may : all >> 14;
            const uint32_t least = grow > 2.0 ? 24u : 1u;
            run = begin;
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                const uint64_t after = run + in[i];
                const bool reached = after >> 14 >= want && (uint32_t)(after & 16383) >= least;
                const bool earlier = run >> 14 >= want && (uint32_t)(run & 16383) >= least;
                if (reached && !earlier) s.found = tid * kEach + i;
                run = after;
            }
            __syncthreads();
        }
        if (s.found >= kPassBins - 1 || !(scale > 0.0f)) return -INFINITY;
        const float e = hi - (float)(s.found + 1) / scale;
        return e - fabsf(e) * 2e-7f - (hi - low) * 4e-7f;
    };

    /* the first filter, from the first turn */
    float lo;  // the smallest of that turn
    {
        float hi = -INFINITY;
        lo = INFINITY;
#pragma unroll
        for (int j = 0; j < kPassEach; ++j) {
            hi = fmaxf(hi, x[j]);
            lo = fminf(lo, x[j] > -INFINITY ? x[j] : INFINITY);
        }
        hi = pass_max(s, hi);
        if (hi > -INFINITY && hi < INFINITY) {
            f = pass_floor(row, hi);
            if (row.kind == kPassShare) weigh = true, rc = hi * row.c;
            if (row.kind == kPassCount || row.kind == kPassShare) {
                lo = -pass_max(s, -lo);
                const float low = fmaxf(f, lo), scale = hi > low ? ((float)kPassBins - 0.5f) / (hi - low) : 0.0f;
#pragma unroll
                for (int j = 0; j < kPassEach; ++j)
                    if (x[j] >= low) atomicAdd(&s.n[min((int)((hi - x[j]) * scale), kPassBins - 1)], 1u);
                __syncthreads();
                f = fmaxf(f, edge(hi, low, scale, 0.0, (double)a.turns * nc));
                if (row.kind == kPassShare && a.turns > 1) {
                    int many = 0;
#pragma unroll
                    for (int j = 0; j < kPassEach; ++j) many += x[j] >= f;
                    /* where a third has to be kept the list runs over again and again, and most such rows are lost in the end:
                     * 256 rows of normal logits of deviation 2 1318 us, 1354 without this; at a sixth rows are lost that
                     * could have been settled (1024 nucleus rows of 256,000 bf16 330 us, 303 at a third) */
                    if (pass_sum(s, (double)many) * 3.0 > kPassThreads * kPassEach) s.lost = 1;
                }
            }
        }
    }

    /* Raise the filter and drop what it drops. */
    auto raise = [&](double grow) {
        const int n = (int)min(s.count, s.valid);
        float hi = -INFINITY;
        for (int i = tid; i < n; i += kPassThreads) hi = fmaxf(hi, pass_x(keep[i]));
        hi = pass_max(s, hi);
        if (n == 0) return;
        if (!(hi < INFINITY)) {  // the kernel for every row
            s.lost = 1;
            return;
        }
        if (row.kind == kPassShare && !weigh) weigh = true, rc = hi * row.c;
        float f_new = fmaxf(pass_floor(row, hi), f);
        if (row.kind == kPassCount || row.kind == kPassShare) {
            const float low = lo < hi ? fmaxf(f_new, lo) : f_new, scale = hi > low ? ((float)kPassBins - 0.5f) / (hi - low) : 0.0f;
            for (int i = tid; i < kPassBins; i += kPassThreads) s.n[i] = 0;
            const double dropped =
                row.kind == kPassShare ? pass_sum(s, rest) * exp2((double)rc - (double)hi * (double)row.c) : 0.0;
            __syncthreads();
            for (int i = tid; i < n; i += kPassThreads) {
                const float v = pass_x(keep[i]);
                if (v >= low) atomicAdd(&s.n[min((int)((hi - v) * scale), kPassBins - 1)], 1u);
            }
            __syncthreads();
            f_new = fmaxf(f_new, edge(hi, low, scale, dropped, grow));
        }
        f = f_new;
        /* the kept ones move up; a turn's places are read before any of them is written */
        __syncthreads();
        if (tid == 0) s.count = 0, s.valid = kPassKeep, s.full = 0;
        for (int at = 0; at < n; at += 4 * kPassThreads) {
            uint64_t e[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int i = at + j * kPassThreads + tid;
                e[j] = i < n ? keep[i] : 0;  // 0 is below every key
            }
            __syncthreads();
            int mine = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float v = pass_x(e[j]);
                if (e[j] && v >= f) ++mine;
                else if (e[j] && weigh) rest += (double)pass_exp2(fmaf(v, row.c, -rc)), e[j] = 0;
                else e[j] = 0;
            }
            uint32_t to = mine ? atomicAdd(&s.count, (uint32_t)mine) : 0;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (e[j]) keep[to++] = e[j];
        }
        __syncthreads();
        if (tid == 0 && s.count > kPassFull) s.lost = 1;
        __syncthreads();
    };

    if (me == 0) {
        /* the row's ends beside whole vectors: at most 14 elements */
        const int tail = head + vecs * V::kPer;
        const int id = tid < head ? tid : tail + tid - head;
        const float v = id < vocab ? req_value(base[id]) : -INFINITY;
        if (tid < 16 && v >= f) keep[atomicAdd(&s.count, 1u)] = pass_pack(v, id);
        else if (weigh && tid < 16) rest += (double)pass_exp2(fmaf(v, row.c, -rc));
    }
    __syncthreads();

    /*
     * The row.  Warps go on by themselves; where the list runs over, all of
     * them meet to raise the filter, and those whose elements found no place
     * try again.
     */
    int done = 0, rises = 0;  // turns of this warp, rises of the filter on the way
    while (!s.lost) {
        while (done < a.turns) {
            const int full = *(volatile int *)&s.full;
            float most = x[0];
#pragma unroll
            for (int j = 1; j < kPassEach; ++j) most = fmaxf(most, x[j]);
            if (__any_sync(0xFFFFFFFFu, most >= f)) {
                uint32_t mask = 0;
#pragma unroll
                for (int j = 0; j < kPassEach; ++j) mask |= x[j] >= f ? 1u << j : 0u;
                bool again = false;
                if (mask) {
                    const uint32_t n = __popc(mask);
                    uint32_t at = atomicAdd(&s.count, n);
                    if (at + n <= kPassKeep) {
                        /* few of a thread's elements pass: the loop takes a turn or two, each choosing one of 16 registers */
                        for (uint32_t left = mask; left; left &= left - 1) {
                            const int j = __ffs(left) - 1;
                            float half[8];
#pragma unroll
                            for (int i = 0; i < 8; ++i) half[i] = j & 1 ? x[2 * i + 1] : x[2 * i];
#pragma unroll
                            for (int i = 0; i < 4; ++i) half[i] = j & 2 ? half[2 * i + 1] : half[2 * i];
#pragma unroll
                            for (int i = 0; i < 2; ++i) half[i] = j & 4 ? half[2 * i + 1] : half[2 * i];
                            const int v = first + turn * (32 * kVecs) + (j / V::kPer) * 32 + lane;
                            keep[at++] = pass_pack(j & 8 ? half[1] : half[0], head + v * V::kPer + j % V::kPer);
                        }
                    } else {  // from the first place that ran over on, none is filled
                        atomicMin(&s.valid, at);
                        s.full = 1;
                        again = true;
                    }
                }
                if (__any_sync(0xFFFFFFFFu, again) || weigh) {
#pragma unroll
                    for (int j = 0; j < kPassEach; ++j)
                        if (x[j] >= f && !again) x[j] = -INFINITY;  // kept: neither tried again nor dropped
                }
                if (__any_sync(0xFFFFFFFFu, again)) break;
            }
            if (weigh) {
                float w[kPassEach];
#pragma unroll
                for (int j = 0; j < kPassEach; ++j) w[j] = pass_exp2(fmaf(x[j], row.c, -rc));  // a NaN stays in the sum
#pragma unroll
                for (int d = kPassEach / 2; d; d >>= 1)
#pragma unroll
                    for (int j = 0; j < d; ++j) w[j] += w[j + d];
                rest += (double)w[0];
            }
            if (++done < a.turns) {
                turn = ahead;
#pragma unroll
                for (int j = 0; j < kVecs; ++j) V::get(next[j], x + j * V::kPer);
                ahead += a.step;
                if (ahead >= a.turns) ahead -= a.turns;
                if (done + 1 < a.turns) load(ahead);
            }
            if (full) break;
        }
        __syncthreads();
        if (!s.full) break;  // every warp is through
        raise(row.kind == kPassShare ? (double)a.turns * nc * kPassThreads / fmax(pass_sum(s, (double)done), 1.0) : 1.0);
        if (++rises == kPassRises && tid == 0) s.lost = 1;  // a row of many ids with some weight: not for one CTA
        __syncthreads();
        if (s.lost) break;
    }
    __syncthreads();

    /* the cluster's parts come together in the first one's memory, after a last rise so that little moves */
    if (nc > 1 && !s.lost && s.count > kPassKeep / 2 / nc) raise((double)nc);
    const double dropped = weigh ? pass_sum(s, rest) : 0.0;
    if (nc > 1) {
        __syncthreads();
        cluster.sync();  // every CTA of the cluster is there, and the first one has its own
        PassShared *to = cluster.map_shared_rank(&s, 0);
        uint64_t *to_keep = cluster.map_shared_rank(keep, 0);
        if (me != 0) {
            const int n = s.lost ? 0 : (int)s.count;
            if (tid == 0) {
                to->part_rest[me] = dropped;
                to->part_rc[me] = rc;
                to->part_f[me] = f;
                const uint32_t at = atomicAdd(&to->count, (uint32_t)n);
                s.left = (int)at;
                if (s.lost || at + n > kPassKeep) s.left = -1, to->lost = 1;
            }
            __syncthreads();
            if (s.left >= 0)
                for (int i = tid; i < n; i += kPassThreads) to_keep[s.left + i] = keep[i];
        }
        cluster.sync();
        if (me != 0) return;
    }
    if (s.lost) {
        if (tid == 0) a.r.status[b] = kPassUnsettled;
        return;
    }
    if (tid == 0) s.part_rest[0] = dropped, s.part_rc[0] = rc;
    __syncthreads();
    for (int c = 1; c < nc; ++c) f = fmaxf(f, s.part_f[c]);  // from here on every element of the row is kept
    int n = (int)s.count;
    if (n == 0) {
        if (tid == 0) {
            a.r.status[b] = kPassSettled;
            a.r.ids[b] = -1;
            if (a.r.probs) a.r.probs[b] = 0.0f;
            if (a.r.counts) a.r.counts[b] = 0;
        }
        return;
    }
    /* the parts' dropped weights, as of the row's largest logit */
    float hi = -INFINITY;
    for (int i = tid; i < n; i += kPassThreads) hi = fmaxf(hi, pass_x(keep[i]));
    hi = pass_max(s, hi);
    double gone = 0.0, gone_error = 0.0;
    if (row.kind == kPassShare) {
        double apart = 0.0;
        for (int c = 0; c < nc; ++c) {
            const double up = (double)s.part_rc[c] - (double)hi * (double)row.c;
            if (s.part_rest[c] != 0.0) gone += s.part_rest[c] * exp2(up), apart = fmax(apart, fabs(up));  // NaN too
        }
        /*
         * Against the sum of the definition's weights: an exponential is off by 2^-22 of itself, four additions by
         * 2^-24 each; the exponent's rounding by 2^-24 of it and that of log2(e) / T by as much (of the exponent from
         * the largest logit on, from which that of the part's reference lies apart).  Weights W over N ids have sum
         * W log2(1 / W) <= sum log2(N / sum).  Ids under the floor of 30 T are in it, at e^-30 each, weights below
         * 2^-126 of the reference's are not, and the definition's weights are rounded to 2^-43.
         */
        const double ids = (double)vocab;
        const double spread = gone > 0.0 ? log2(fmax(ids / gone, 2.0)) : 0.0;
        gone_error = gone * (ldexp(1.0, -21) + 0.6932 * (spread * 2.0 + apart) * ldexp(1.0, -24)) * 1.01 +
                     ids * (1e-13 + ldexp(1.0, -43));
        if (!(gone < 1e7)) {  // the reference was too far below, or there is a NaN
            if (tid == 0) a.r.status[b] = kPassUnsettled;
            return;
        }
    }
    if (!(hi < INFINITY)) {
        if (tid == 0) a.r.status[b] = kPassUnsettled;
        return;
    }
    /* one more rise for a shorter sort */
    if (n > kPassThreads) {
        const double other = gone;
        if (row.kind == kPassShare) {
            /* the parts' weights as one thread's, of one reference */
            weigh = true;
            rc = hi * row.c;
            rest = tid == 0 ? gone * exp2((double)hi * (double)row.c - (double)rc) : 0.0;
        }
        raise(1.0);
        n = (int)s.count;
        if (row.kind == kPassShare) {
            gone = pass_sum(s, rest) * exp2((double)rc - (double)hi * (double)row.c);
            /* exponents of 44 at most: ids are above the floor of 30 T */
            gone_error += fmax(gone - other, 0.0) * (ldexp(1.0, -21) + 0.6932 * 2.0 * 44.0 * ldexp(1.0, -24)) * 1.01 + gone * 1e-14;
        }
        __syncthreads();
    }
    if (s.lost || n > kPassSort) {
        if (tid == 0) a.r.status[b] = kPassUnsettled;
        return;
    }
    /*
     * In order, largest first: each thread counts what is larger than its
     * element, or where they are more than threads, a sort.
     */
    uint64_t *list = keep, *weights = keep + kPassSort;
    if (n <= kPassThreads) {
        list = keep + kPassSort, weights = keep;
        if (tid < n) {
            const uint64_t e = keep[tid];
            int larger = 0;
#pragma unroll 4
            for (int i = 0; i < n; ++i) larger += keep[i] > e;
            list[larger] = e;
        }
        __syncthreads();
    } else {
        int size = 2 * kPassThreads;
        while (size < n) size <<= 1;
        for (int i = n + tid; i < size; i += kPassThreads) keep[i] = 0;
        __syncthreads();
        req_sort<kPassThreads>(keep, size);
    }
    const ReqRow r = req_row(a.r, b, hi, s.u);
    if (r.greedy) {
        if (tid == 0) {
            a.r.status[b] = kPassSettled;
            a.r.ids[b] = pass_id(list[0]);
            if (a.r.probs) a.r.probs[b] = 1.0f;
            if (a.r.counts) a.r.counts[b] = 1;
        }
        return;
    }
    /* what is left by the temperature, min-p and top-k is a beginning of the order */
    const int most = r.k ? min(n, r.k) : n;
    int left = 0;
    for (int at = 0; at < most; at += kPassThreads) {
        const int i = at + tid;
        const bool in = i < most && (uint32_t)(list[i] >> 32) >= r.floor;
        if (in) weights[i] = req_weight(r, pass_x(list[i]), s.table);
        left += __syncthreads_count(in);
    }
    if (r.p < 1.0) {
        const int each = (left + kPassThreads - 1) / kPassThreads, from = min(left, tid * each), to = min(left, from + each);
        uint64_t mine = 0, all;
        for (int i = from; i < to; ++i) mine += weights[i];
        const uint64_t end = pass_scan(s, mine, all);
        uint64_t want[2];
        for (int side = 0; side < 2; ++side) {
            const double d = side ? gone + gone_error : fmax(gone - gone_error, 0.0);
            const uint64_t total = all + (row.kind == kPassShare ? (uint64_t)(d * (double)(1ull << kReqFraction)) + side : 0);
            const uint64_t share = (uint64_t)(r.p * 18446744073709551616.0);
            want[side] = __umul64hi(share, total) + (share * total != 0);
            if (want[side] == 0) want[side] = 1;
        }
        if (tid == 0) s.found = s.found_high = 0;
        __syncthreads();
        uint64_t run = end - mine;
        for (int i = from; i < to; ++i) {
            const uint64_t after = run + weights[i];
            if (run < want[0] && after >= want[0]) s.found = (uint32_t)i + 1;
            if (run < want[1] && after >= want[1]) s.found_high = (uint32_t)i + 1;
            run = after;
        }
        __syncthreads();
        left = (int)s.found;
        /* open within the error, or a lost bet: the row's other ids weigh too much, or some come before the cut */
        if (s.found != s.found_high || left == 0 || (row.kind == kPassShare && !(pass_x(list[left - 1]) >= f))) {
            if (tid == 0) a.r.status[b] = kPassUnsettled;
            return;
        }
    }
    /* the walk in the order of ids: each thread adds up what lies before its element, or after a sort */
    uint64_t before = 0, total = 0;
    int at = tid, end = min(left, tid + 1);
    if (left <= kPassThreads) {
        const uint32_t id = tid < left ? (uint32_t)list[tid] : 0;  // the larger, the earlier
#pragma unroll 4
        for (int i = 0; i < left; ++i) {
            const uint64_t w = weights[i];
            total += w;
            before += (uint32_t)list[i] > id ? w : 0;
        }
    } else {
        int size = 2 * kPassThreads;
        while (size < left) size <<= 1;
        for (int i = tid; i < size; i += kPassThreads) list[i] = i < left ? list[i] << 32 | list[i] >> 32 : 0;
        __syncthreads();
        req_sort<kPassThreads>(list, size);
        for (int i = tid; i < left; i += kPassThreads) {
            list[i] = list[i] << 32 | list[i] >> 32;
            weights[i] = req_weight(r, pass_x(list[i]), s.table);
        }
        __syncthreads();
        const int each = (left + kPassThreads - 1) / kPassThreads;
        at = min(left, tid * each), end = min(left, at + each);
        uint64_t mine = 0;
        for (int i = at; i < end; ++i) mine += weights[i];
        before = pass_scan(s, mine, total) - mine;
    }
    uint64_t target = r.u >= 1.0f ? total : __umul64hi((uint64_t)((double)r.u * 18446744073709551616.0), total);
    if (target >= total) target = total - 1;
    for (; at < end; ++at) {
        if (before <= target && target - before < weights[at]) {
            a.r.status[b] = kPassSettled;
            a.r.ids[b] = pass_id(list[at]);
            if (a.r.probs)
                a.r.probs[b] = (float)(req_exp(r, pass_x(list[at]), s.table) * (double)(1ull << kReqFraction) / (double)total);
            if (a.r.counts) a.r.counts[b] = left;
        }
        before += weights[at];
    }
}

}  // namespace noel
