/*
 * Host side of the 8-bit projections (include/noel_int8.h).
 */
#include "noel_int8.h"

#include <atomic>
#include <deque>
#include <map>
#include <mutex>

#include "host.h"
#include "int8.cuh"
#include "noel_lmhead.h"

using namespace noel;

namespace {

/*
 * Products that gave up, counted on the device and never cleared there: a
 * count for each stream, and the first one for calls that a graph has captured
 * (it may be replayed on any stream) and for streams that come when the others
 * are taken.  A check compares with what its stream was last told, so that
 * none takes another stream's report.
 */
constexpr int kCounts = 1024;
__device__ unsigned g_i8_failed[kCounts];

struct StreamWaits {
    int count = 0;                  // index of its count; 0: no product yet, or the common one
    unsigned told = 0, told_common = 0;
};
struct DeviceWaits {
    unsigned *counts = nullptr;
    int taken = 1;
    bool common = false;            // something may be in the common count
    std::map<const void *, StreamWaits> streams;
};
std::mutex g_waits_mu;
std::deque<DeviceWaits> g_waits;

/* what stands for a stream among the threads: the two names of the default one are one, the thread's own is each thread's */
const void *stream_key(cudaStream_t s) {
    static thread_local char mine;
    return s == cudaStreamPerThread ? &mine : s == cudaStreamLegacy ? nullptr : static_cast<const void *>(s);
}

/* with the lock held */
int device_waits(DeviceWaits **out) {
    int dev = 0;
    CUDA_TRY(cudaGetDevice(&dev));
    if ((int)g_waits.size() <= dev) g_waits.resize(dev + 1);
    DeviceWaits &d = g_waits[dev];
    if (!d.counts) {
        void *p = nullptr;
        CUDA_TRY(cudaGetSymbolAddress(&p, g_i8_failed));
        d.counts = static_cast<unsigned *>(p);
    }
    *out = &d;
    return NOEL_OK;
}

/* where a product on the stream counts that it gave up */
int failed_count(cudaStream_t s, unsigned **count) {
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    CUDA_TRY(cudaStreamIsCapturing(s, &cap));
    std::lock_guard<std::mutex> lk(g_waits_mu);
    DeviceWaits *d = nullptr;
    const int r = device_waits(&d);
    if (r) return r;
    int at = 0;
    if (cap == cudaStreamCaptureStatusNone) {
        StreamWaits &w = d->streams[stream_key(s)];
        if (!w.count && d->taken < kCounts) w.count = d->taken++;
        at = w.count;
    }
    if (!at) d->common = true;
    *count = d->counts + at;
    return NOEL_OK;
}

using EncodeFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                              const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

int encode_fn(EncodeFn *out) {
    static std::atomic<EncodeFn> known{nullptr};  // the same for every device and thread
    EncodeFn fn = known.load(std::memory_order_acquire);
    if (!fn) {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult found;
        CUDA_TRY(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found));
        if (found != cudaDriverEntryPointSuccess || !p) return fail(NOEL_ERR_CUDA, "cuTensorMapEncodeTiled is not there");
        fn = reinterpret_cast<EncodeFn>(p);
        known.store(fn, std::memory_order_release);
    }
    *out = fn;
    return NOEL_OK;
}

/* rows of bytes, copied box_rows x 128 columns at a time; zeros beyond them */
int byte_map(CUtensorMap *m, const void *base, int rows, int cols, size_t ld, int box_rows) {
    EncodeFn encode = nullptr;
    const int r = encode_fn(&encode);
    if (r) return r;
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld};
    const cuuint32_t box[2] = {(cuuint32_t)kI8Line, (cuuint32_t)box_rows}, each[2] = {1, 1};
    const CUresult e = encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(base), dims, strides, box, each,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (e != CUDA_SUCCESS) return fail(NOEL_ERR_CUDA, "cuTensorMapEncodeTiled: %d (%d x %d, pitch %zu)", (int)e, rows, cols, ld);
    return NOEL_OK;
}

/* tokens and rows of a product: the kernel steps over both in 32 bits, by tiles of 256 */
constexpr int kMostRows = 0x7FFFFFFF - 512;

bool misaligned(const void *p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to != 0; }

int cast_args(const void *x, int type, size_t ldx, int rows, int cols, const void *q, size_t ldq, const float *scale,
              I8CastArgs *out) {
    if (type != NOEL_HEAD_F32 && type != NOEL_HEAD_F16 && type != NOEL_HEAD_BF16)
        return fail(NOEL_ERR_UNSUPPORTED, "type %d (F32 0, F16 1, BF16 30)", type);
    if (rows < 0 || cols <= 0) return fail(NOEL_ERR_INVALID_ARG, "rows %d / cols %d", rows, cols);
    if (cols > NOEL_I8_MAX_COLS) return fail(NOEL_ERR_TOO_LARGE, "cols %d (1..%d)", cols, NOEL_I8_MAX_COLS);
    if (ldx < (size_t)cols || ldq < (size_t)cols || ldq % 16)
        return fail(NOEL_ERR_INVALID_ARG, "cols %d: ldx %zu / ldq %zu (multiple of 16)", cols, ldx, ldq);
    const size_t es = type == NOEL_HEAD_F32 ? 4 : 2;
    if (misaligned(x, es) || misaligned(q, 16) || misaligned(scale, 4))
        return fail(NOEL_ERR_INVALID_ARG, "x aligned to its elements, q to 16 bytes and scale to 4 wanted");
    if (rows > 0 && (!x || !q || !scale)) return fail(NOEL_ERR_INVALID_ARG, "x, q and scale are required");
    I8CastArgs a{};
    a.x = x, a.ldx = (int64_t)ldx, a.rows = rows, a.cols = cols;
    a.vec = !misaligned(x, 16) && (rows == 1 || ldx * es % 16 == 0);
    a.ldq = (int64_t)ldq;
    a.scale = const_cast<float *>(scale);
    a.q = static_cast<int8_t *>(const_cast<void *>(q));
    *out = a;
    return NOEL_OK;
}

int cast_launch(const I8CastArgs &a, int type, cudaStream_t s) {
    if (type == NOEL_HEAD_F32) i8_cast_kernel<kI8F32><<<a.rows, kI8CastThreads, 0, s>>>(a);
    else if (type == NOEL_HEAD_F16) i8_cast_kernel<kI8F16><<<a.rows, kI8CastThreads, 0, s>>>(a);
    else i8_cast_kernel<kI8BF16><<<a.rows, kI8CastThreads, 0, s>>>(a);
    CUDA_TRY(cudaGetLastError());
    return NOEL_OK;
}

struct Product {
    const int8_t *a, *w;
    size_t lda, ldw;
    I8Args args;
    int dtype;
};

int product_args(const int8_t *a, size_t lda, const float *a_scale, int tokens, const int8_t *w, size_t ldw,
                 const float *w_scale, int rows, int cols, void *y, int dtype, size_t ldy, Product *out) {
    if (dtype != NOEL_DTYPE_F32 && dtype != NOEL_DTYPE_BF16) return fail(NOEL_ERR_UNSUPPORTED, "dtype %d (F32 0, BF16 1)", dtype);
    if (tokens < 0 || rows < 0 || cols <= 0)
        return fail(NOEL_ERR_INVALID_ARG, "tokens %d / rows %d / cols %d", tokens, rows, cols);
    if (cols > NOEL_I8_MAX_COLS) return fail(NOEL_ERR_TOO_LARGE, "cols %d (1..%d)", cols, NOEL_I8_MAX_COLS);
    if (tokens > kMostRows || rows > kMostRows)
        return fail(NOEL_ERR_TOO_LARGE, "tokens %d / rows %d (up to %d)", tokens, rows, kMostRows);
    if (lda < (size_t)cols || lda % 16 || ldw < (size_t)cols || ldw % 16 || ldy < (size_t)rows)
        return fail(NOEL_ERR_INVALID_ARG, "cols %d: lda %zu / ldw %zu (multiples of 16); rows %d: ldy %zu", cols, lda, ldw, rows, ldy);
    if (misaligned(a, 16) || misaligned(w, 16)) return fail(NOEL_ERR_INVALID_ARG, "a and w must be 16-byte aligned");
    if (misaligned(a_scale, 4) || misaligned(w_scale, 4) || misaligned(y, dtype == NOEL_DTYPE_F32 ? 4 : 2))
        return fail(NOEL_ERR_INVALID_ARG, "scales must be 4-byte aligned and y aligned to its elements");
    if (lda >> 40 || ldw >> 40) return fail(NOEL_ERR_TOO_LARGE, "lda %zu / ldw %zu", lda, ldw);
    if (tokens > 0 && rows > 0 && (!a || !a_scale || !w || !w_scale || !y))
        return fail(NOEL_ERR_INVALID_ARG, "a, w, their scales and y are required");
    Product p{};
    p.a = a, p.w = w, p.lda = lda, p.ldw = ldw, p.dtype = dtype;
    p.args.a_scale = a_scale, p.args.w_scale = w_scale, p.args.y = y, p.args.ldy = (int64_t)ldy;
    p.args.tokens = tokens, p.args.rows = rows, p.args.cols = cols;
    *out = p;
    return NOEL_OK;
}

template <int NT, bool PAIR, typename OUT>
int product_launch(const Product &p, const I8Args &args, int groups, bool dependent, cudaStream_t s) {
    CUtensorMap mw, mp, ma;
    int r = byte_map(&mw, p.w, args.rows, args.cols, p.ldw, kI8RowsCta);
    if (!r) r = byte_map(&mp, p.w, args.rows, args.cols, p.ldw, kI8Box);
    if (!r) r = byte_map(&ma, p.a, args.tokens, args.cols, p.lda, PAIR ? NT / 2 : NT);
    if (!r) r = dynamic_smem((const void *)i8_product_kernel<NT, PAIR, OUT>, i8_smem(NT, PAIR));
    if (r) return r;
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3(PAIR ? 2 * groups : groups);
    lc.blockDim = dim3(kI8Threads);
    lc.dynamicSmemBytes = i8_smem(NT, PAIR);
    lc.stream = s;
    cudaLaunchAttribute at[2];
    int n = 0;
    if (dependent) {
        at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (PAIR) {
        at[n].id = cudaLaunchAttributeClusterDimension;
        at[n].val.clusterDim.x = 2;
        at[n].val.clusterDim.y = at[n].val.clusterDim.z = 1;
        ++n;
    }
    lc.attrs = at;
    lc.numAttrs = n;
    CUDA_TRY(cudaLaunchKernelEx(&lc, i8_product_kernel<NT, PAIR, OUT>, mw, mp, ma, args));
    CUDA_TRY(cudaGetLastError());
    return NOEL_OK;
}

template <int NT, bool PAIR>
int product_tile(const Product &p, bool dependent, cudaStream_t s) {
    int sms = 0;
    int r = device_sms(&sms);
    I8Args args = p.args;
    if (!r) r = failed_count(s, &args.failed);
    if (r) return r;
    args.wait_ns = wait_limit_ns();
    args.stall = take_stall();
    const int most = PAIR ? sms / 2 : sms, tile = PAIR ? 2 * kI8RowsCta : kI8RowsCta;
    const int64_t token_tiles = ((int64_t)args.tokens + NT - 1) / NT;
    int64_t groups;
    args.ranges = token_tiles == 1;
    if (args.ranges) groups = ((int64_t)args.rows + 31) / 32;
    else groups = token_tiles * (((int64_t)args.rows + tile - 1) / tile);
    if (groups > most) groups = most;
    return p.dtype == NOEL_DTYPE_F32 ? product_launch<NT, PAIR, float>(p, args, (int)groups, dependent, s)
                                     : product_launch<NT, PAIR, __nv_bfloat16>(p, args, (int)groups, dependent, s);
}

/*
 * Tiles by the number of tokens alone, made for matrices whose weights' stream
 * counts.  152,064 rows of 4096, in us with tiles of 16, 32, 64, 128 and 256:
 * 16 tokens 112 110 113 116 160; 17 tokens 128 110 113 117 172; 33 tokens 185
 * 130 108 113 118; 65 tokens 303 186 133 117 123; 129 tokens 535 304 189 194
 * 133; 300 tokens with 64, 128 and 256: 310 281 222; 2048 with 128 and 256: 1468
 * 962.  Matrices of few rows would want narrower tiles, which give more groups:
 * 4096 rows, 64 tokens 13.5 13.4 15.8 18.5 17.9, 200 tokens 28.5 21.4 15.2 17.7
 * 20.7, 300 tokens with 64, 128 and 256: 22.3 18.6 19.9; from 768 tokens on 256
 * is best there too (128 31.0, 256 21.9).  1024 rows: within 3 us of each other.
 */
int product(const Product &p, bool dependent, cudaStream_t s) {
    const int t = p.args.tokens;
    if (t <= 16) return product_tile<16, false>(p, dependent, s);
    if (t <= 32) return product_tile<32, false>(p, dependent, s);
    if (t <= 64) return product_tile<64, true>(p, dependent, s);
    if (t <= 128) return product_tile<128, true>(p, dependent, s);
    return product_tile<256, true>(p, dependent, s);
}

size_t cast_pitch(int cols) { return ((size_t)cols + 15) / 16 * 16; }

}  // namespace

int noel::i8_wait_failed(cudaStream_t s, bool *failed) {
    *failed = false;
    const unsigned *own = nullptr, *common = nullptr;
    {
        std::lock_guard<std::mutex> lk(g_waits_mu);
        DeviceWaits *d = nullptr;
        const int r = device_waits(&d);
        if (r) return r;
        const auto it = d->streams.find(stream_key(s));
        if (it != d->streams.end() && it->second.count) own = d->counts + it->second.count;
        if (d->common) common = d->counts;
    }
    unsigned now = 0, now_common = 0;
    if (own) CUDA_TRY(cudaMemcpyAsync(&now, own, sizeof(now), cudaMemcpyDeviceToHost, s));
    if (common) CUDA_TRY(cudaMemcpyAsync(&now_common, common, sizeof(now_common), cudaMemcpyDeviceToHost, s));
    if (!own && !common) return NOEL_OK;
    CUDA_TRY(cudaStreamSynchronize(s));
    std::lock_guard<std::mutex> lk(g_waits_mu);
    DeviceWaits *d = nullptr;
    const int r = device_waits(&d);
    if (r) return r;
    StreamWaits &w = d->streams[stream_key(s)];
    *failed = (own && now != w.told) || (common && now_common != w.told_common);
    if (own) w.told = now;
    if (common) w.told_common = now_common;
    return NOEL_OK;
}

extern "C" int noel_i8_cast(const void *d_x, int type, size_t ldx, int rows, int cols, int8_t *d_q, size_t ldq,
                            float *d_scale, void *stream) try {
    I8CastArgs a{};
    int r = cast_args(d_x, type, ldx, rows, cols, d_q, ldq, d_scale, &a);
    if (r) return r;
    if (rows == 0) return ok();
    int sms = 0;
    r = device_sms(&sms);
    if (!r) r = cast_launch(a, type, static_cast<cudaStream_t>(stream));
    return r ? r : ok();
} catch (...) {
    return fail(NOEL_ERR_CUDA, "host memory");
}

extern "C" int noel_i8_product(const int8_t *d_a, size_t lda, const float *d_a_scale, int tokens, const int8_t *d_w,
                               size_t ldw, const float *d_w_scale, int rows, int cols, void *d_y, int dtype, size_t ldy,
                               void *stream) try {
    Product p{};
    int r = product_args(d_a, lda, d_a_scale, tokens, d_w, ldw, d_w_scale, rows, cols, d_y, dtype, ldy, &p);
    if (r) return r;
    if (tokens == 0 || rows == 0) return ok();
    r = product(p, false, static_cast<cudaStream_t>(stream));
    return r ? r : ok();
} catch (...) {
    return fail(NOEL_ERR_CUDA, "host memory");
}

extern "C" size_t noel_i8_linear_workspace_bytes(int tokens, int cols) {
    if (tokens <= 0 || cols <= 0 || cols > NOEL_I8_MAX_COLS) return 0;
    return (size_t)tokens * (cast_pitch(cols) + sizeof(float));
}

extern "C" int noel_i8_linear(const void *d_x, int type, size_t ldx, int tokens, const int8_t *d_w, size_t ldw,
                              const float *d_w_scale, int rows, int cols, void *d_y, int dtype, size_t ldy, void *d_work,
                              size_t work_bytes, void *stream) try {
    if (misaligned(d_work, 16)) return fail(NOEL_ERR_INVALID_ARG, "scratch must be 16-byte aligned");
    const size_t need = noel_i8_linear_workspace_bytes(tokens, cols);
    if (need > 0 && (!d_work || work_bytes < need))
        return fail(NOEL_ERR_INVALID_ARG, "scratch of %zu bytes, %zu wanted", d_work ? work_bytes : 0, need);
    const size_t ldq = cols > 0 ? cast_pitch(cols) : 0;
    int8_t *q = static_cast<int8_t *>(d_work);
    float *scale = reinterpret_cast<float *>(q + (tokens > 0 ? (size_t)tokens * ldq : 0));
    I8CastArgs a{};
    Product p{};
    int r = cast_args(d_x, type, ldx, tokens, cols, q, ldq, scale, &a);
    if (!r) r = product_args(q, ldq, scale, tokens, d_w, ldw, d_w_scale, rows, cols, d_y, dtype, ldy, &p);
    if (r) return r;
    if (tokens == 0 || rows == 0) return ok();
    int sms = 0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    r = device_sms(&sms);
    if (!r) r = cast_launch(a, type, s);
    if (!r) r = product(p, true, s);
    return r ? r : ok();
} catch (...) {
    return fail(NOEL_ERR_CUDA, "host memory");
}
