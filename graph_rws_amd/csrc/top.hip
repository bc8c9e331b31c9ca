// The k largest logits of each row with their classes (gfx950): the teacher's
// side of distillation from top logits.
//
// Every logit becomes a 64-bit key, (order-preserving bits of the value,
// complement of the class), so keys are distinct, a larger key is a larger
// logit, and of equal logits the lowest class comes first.  -0 equals +0 and
// a NaN is larger than everything, as in torch's sort.
//
// A work-group streams a row (or one of several stretches of it, when there
// are few rows) and keeps in LDS the keys above a running bound; when the
// buffer might overflow, it finds the k-th largest key bit by bit, drops the
// rest and raises the bound to it.  The row is read once.
#include "grws_internal.h"

namespace grws {
namespace {

constexpr int kT = 256;          // threads of a work-group
constexpr int kMaxK = 1024;
constexpr int kVec = 8;          // logits a thread takes per step
constexpr int kCap = kMaxK + kT * kVec;  // keys in LDS
constexpr int kPer = kCap / kT;

__device__ __forceinline__ uint32_t order_bits(float x) {
    if (x != x) return 0xffffffffu;
    const uint32_t u = __float_as_uint(x == 0.f ? 0.f : x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ uint64_t key_of(float x, uint32_t cls) {
    return ((uint64_t)order_bits(x) << 32) | (uint32_t)~cls;
}

struct Pool {
    uint64_t keys[kCap];
    int32_t count;
    int32_t waves[2][kT / kWave];
};

// Number of the work-group's threads' keys that are >= bound.
__device__ __forceinline__ int count_from(const uint64_t (&mine)[kPer], uint64_t bound, Pool& p, int turn) {
    int c = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) c += __builtin_popcountll(__ballot(mine[i] >= bound));
    if ((threadIdx.x & 63) == 0) p.waves[turn][threadIdx.x >> 6] = c;
    __syncthreads();
    c = 0;
#pragma unroll
    for (int w = 0; w < kT / kWave; ++w) c += p.waves[turn][w];
    return c;
}

// Keeps the k largest keys of the pool (all, when there are no more) and
// returns the k-th (0 when there are fewer).  Keys are distinct and not 0.
__device__ __forceinline__ uint64_t keep_best(Pool& p, int k) {
    __syncthreads();
    const int n = p.count;
    uint64_t mine[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int at = i * kT + threadIdx.x;
        mine[i] = at < n ? p.keys[at] : 0;
    }
    if (n < k) return 0;
    uint64_t bound = 0;
    for (int bit = 63; bit >= 0; --bit) {
        const uint64_t trial = bound | (1ull << bit);
        if (count_from(mine, trial, p, bit & 1) >= k) bound = trial;
    }
    __syncthreads();  // every thread has its keys and the last counts
    if (threadIdx.x == 0) p.count = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const bool in = mine[i] >= bound && mine[i] != 0;
        const uint64_t b = __ballot(in);
        int at = 0;
        if ((threadIdx.x & 63) == 0 && b) at = atomicAdd(&p.count, __builtin_popcountll(b));
        at = __shfl(at, 0, kWave) + __builtin_popcountll(b & lanemask_lt());
        if (in) p.keys[at] = mine[i];
    }
    __syncthreads();
    return bound;
}

// Offers every thread's kVec keys (0: none) to the pool.
__device__ __forceinline__ void offer(Pool& p, const uint64_t (&x)[kVec], int k, uint64_t& bound) {
    __syncthreads();
    if (p.count + kT * kVec > kCap) bound = keep_best(p, k);  // uniform: the count is read after the barrier
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
        const bool in = x[i] > bound;
        const uint64_t b = __ballot(in);
        if (!b) continue;
        int at = 0;
        if ((threadIdx.x & 63) == 0) at = atomicAdd(&p.count, __builtin_popcountll(b));
        at = __shfl(at, 0, kWave) + __builtin_popcountll(b & lanemask_lt());
        if (in) p.keys[at] = x[i];
    }
}

// The pool's keys, largest first, by counting the larger ones.
template <typename T>
__device__ __forceinline__ void write_best(Pool& p, int k, const T* row, T* values, int32_t* index) {
    keep_best(p, k);
    __syncthreads();
    const int n = p.count < k ? p.count : k;
    for (int a = threadIdx.x; a < n; a += kT) {
        const uint64_t key = p.keys[a];
        int rank = 0;
        for (int b = 0; b < n; ++b) rank += p.keys[b] > key;
        const uint32_t cls = ~(uint32_t)key;
        index[rank] = (int32_t)cls;
        values[rank] = row[cls];
    }
}

template <typename T, bool FINAL>
__global__ __launch_bounds__(kT) void top_rows_kernel(const T* __restrict__ logits, int64_t ld, int32_t classes,
                                                      int32_t k, int32_t stretch, T* __restrict__ values,
                                                      int32_t* __restrict__ index, uint64_t* __restrict__ best) {
    __shared__ Pool p;
    const int64_t r = blockIdx.x;
    const T* row = logits + r * ld;
    const int32_t c0 = (int32_t)blockIdx.y * stretch;
    const int32_t c1 = classes - c0 < stretch ? classes : c0 + stretch;
    if (threadIdx.x == 0) p.count = 0;
    uint64_t bound = 0;
    for (int32_t c = c0; c < c1; c += kT * kVec) {
        const int32_t at = c + (int32_t)threadIdx.x * kVec;
        uint64_t x[kVec];
        if (at + kVec <= c1) {
            T v[kVec];
            __builtin_memcpy(v, row + at, sizeof(v));  // rows of any alignment
#pragma unroll
            for (int i = 0; i < kVec; ++i) x[i] = key_of(to_float(v[i]), (uint32_t)(at + i));
        } else {
#pragma unroll
            for (int i = 0; i < kVec; ++i)
                x[i] = at + i < c1 ? key_of(to_float(row[at + i]), (uint32_t)(at + i)) : 0;
        }
        offer(p, x, k, bound);
    }
    if constexpr (FINAL) {
        write_best(p, k, row, values + r * k, index + r * k);
    } else {
        keep_best(p, k);
        __syncthreads();
        uint64_t* out = best + (r * gridDim.y + blockIdx.y) * k;
        const int n = p.count;
        for (int a = threadIdx.x; a < k; a += kT) out[a] = a < n ? p.keys[a] : 0;
    }
}

// Joins the stretches of a row: `count` keys (0: none), the k largest.
template <typename T>
__global__ __launch_bounds__(kT) void top_join_kernel(const T* __restrict__ logits, int64_t ld,
                                                      const uint64_t* __restrict__ best, int64_t count, int32_t k,
                                                      T* __restrict__ values, int32_t* __restrict__ index) {
    __shared__ Pool p;
    const int64_t r = blockIdx.x;
    if (threadIdx.x == 0) p.count = 0;
    uint64_t bound = 0;
    for (int64_t c = 0; c < count; c += kT * kVec) {
        uint64_t x[kVec];
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            const int64_t at = c + i * kT + threadIdx.x;
            x[i] = at < count ? best[r * count + at] : 0;
        }
        offer(p, x, k, bound);
    }
    write_best(p, k, logits + r * ld, values + r * k, index + r * k);
}

// Stretches of a row: one when the rows alone fill the chip (4 work-groups
// on each of 256 CUs), else as many as that takes, of at least 4,096 logits
// and 4 k.
int32_t stretches(int64_t rows, int64_t classes, int64_t k) {
    int64_t n = (1024 + rows - 1) / rows;
    const int64_t least = 4 * k > 4096 ? 4 * k : 4096;
    const int64_t most = classes / least;
    if (n > most) n = most;
    return n < 1 ? 1 : (int32_t)n;
}

}  // namespace
}  // namespace grws

using namespace grws;

extern "C" size_t grws_top_logits_workspace_bytes(int64_t rows, int64_t classes, int32_t k) {
    if (rows <= 0 || classes <= 0 || k <= 0) return 0;
    const int32_t n = stretches(rows, classes, k);
    if (n == 1) return 0;
    Sizer s;
    s.take<uint64_t>((size_t)rows * n * k);
    return s.used;
}

extern "C" int grws_top_logits(const void* logits, int32_t dtype, int64_t ld, int64_t rows, int64_t classes,
                               int32_t k, void* values, int32_t* index, void* workspace, size_t workspace_bytes,
                               void* stream_) {
    clear_error();
    hipStream_t stream = as_stream(stream_);
    if (dtype != GRWS_F32 && dtype != GRWS_F16 && dtype != GRWS_BF16)
        return set_error(GRWS_E_DTYPE, "top_logits: unsupported dtype %d", dtype);
    GRWS_CHECK_ARG(rows >= 0 && rows <= INT32_MAX && classes > 0 && classes <= INT32_MAX - 65536 && ld >= classes,
                   "top_logits: bad sizes");
    GRWS_CHECK_ARG(k >= 1 && k <= kMaxK && k <= classes, "top_logits: k must be 1..min(classes, 1024)");
    if (rows == 0) return GRWS_OK;
    GRWS_CHECK_ARG(logits && values && index, "top_logits: null pointer");
    const int32_t n = stretches(rows, classes, k);
    Carver cv(workspace, workspace_bytes);
    uint64_t* best = n > 1 ? cv.take<uint64_t>((size_t)rows * n * k) : nullptr;
    if (!cv.ok)
        return set_error(GRWS_E_CAPACITY, "top_logits: workspace too small (%zu < %zu)", workspace_bytes, cv.used);
    const int32_t stretch = (int32_t)((classes + n - 1) / n);
    const dim3 grid((unsigned)rows, (unsigned)n);
#define GRWS_TOP(T)                                                                                                \
    do {                                                                                                           \
        const T* x = static_cast<const T*>(logits);                                                                \
        T* v = static_cast<T*>(values);                                                                            \
        if (n == 1) {                                                                                              \
            hipLaunchKernelGGL((top_rows_kernel<T, true>), grid, dim3(kT), 0, stream, x, ld, (int32_t)classes, k,  \
                               stretch, v, index, best);                                                           \
        } else {                                                                                                   \
            hipLaunchKernelGGL((top_rows_kernel<T, false>), grid, dim3(kT), 0, stream, x, ld, (int32_t)classes, k, \
                               stretch, v, index, best);                                                           \
            GRWS_LAUNCH_CHECK();                                                                                   \
            hipLaunchKernelGGL(top_join_kernel<T>, dim3((unsigned)rows), dim3(kT), 0, stream, x, ld, best,         \
                               (int64_t)n * k, k, v, index);                                                       \
        }                                                                                                          \
    } while (0)
    if (dtype == GRWS_F32) GRWS_TOP(float);
    else if (dtype == GRWS_F16) GRWS_TOP(_Float16);
    else GRWS_TOP(__hip_bfloat16);
#undef GRWS_TOP
    GRWS_LAUNCH_CHECK();
    return GRWS_OK;
}
