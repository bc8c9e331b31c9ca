// The k largest logits of each row with their classes (gfx950): the teacher's
// side of distillation from top logits.
//
// A work-group streams a row (or one of several stretches of it, when there
// are few rows) and keeps in LDS the keys above a running bound; the row is
// read once.  The first bound is the k-th largest of the threads' maxima over
// the first 8,192 logits (at least k logits reach it); of random logits about
// 1% pass it, so a row of 50,021 leaves some 450 keys for k = 64, of which
// the k largest are found digit by digit (8 bits, an LDS histogram each) and
// ordered by counting.  When the pool overflows (k > 128, rising rows, ties)
// the k largest are found in between and the bound is raised to the k-th.
#include "top_pool.h"

namespace grws {
namespace {

template <int MAXK, typename T>
__device__ __forceinline__ void write_best(Pool<MAXK>& p, int k, int bits, int class_bits, const T* row, T* values,
                                           int32_t* index) {
    put_best(p, k, bits, class_bits, [&](int at, int32_t cls) {
        index[at] = cls;
        values[at] = row[cls];
    });
}

template <typename T, bool FINAL, int MAXK>
__global__ __launch_bounds__(kT, MAXK <= kSmallK ? 8 : 5) void top_rows_kernel(
    const T* __restrict__ logits, int64_t ld, int32_t classes, int32_t class_bits, int32_t k, int32_t stretch,
                                                      T* __restrict__ values, int32_t* __restrict__ index,
                                                      uint64_t* __restrict__ best) {
    constexpr int VB = sizeof(T) * 8, CAP = Sizes<MAXK>::CAP, OFFER = Sizes<MAXK>::OFFER;
    struct Vec {
        uint32_t w[kVec * sizeof(T) / 4];
    };
    __shared__ Pool<MAXK> p;
    const int64_t r = blockIdx.x;
    const T* row = logits + r * ld;
    const int32_t c0 = (int32_t)blockIdx.y * stretch;
    const int32_t c1 = classes - c0 < stretch ? classes : c0 + stretch;
    const int bits = VB + class_bits;
    const uint64_t low = (1ull << class_bits) - 1;
    if (threadIdx.x == 0) p.count = 0;
    uint64_t bound = 0;
    float least = -INFINITY;  // the bound's logit: smaller ones are not looked at
    for (int32_t c = c0; c < c1; c += kChunk) {
        // load i of a thread: logits c + 2,048 i + 8 thread + 0..7
        Vec v[kLoads];
        const int32_t at = c + (int32_t)threadIdx.x * kVec;
        const bool whole = c + kChunk <= c1;  // uniform
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int32_t f = at + i * kT * kVec;
            if (whole || f + kVec <= c1) {
                __builtin_memcpy(&v[i], row + f, sizeof(Vec));  // rows of any alignment
            } else {
                T x[kVec];
#pragma unroll
                for (int e = 0; e < kVec; ++e) x[e] = f + e < c1 ? row[f + e] : from_float<T>(0.f);
                __builtin_memcpy(&v[i], x, sizeof(Vec));
            }
        }
        auto get = [&](int i) -> T {
            const uint32_t w = v[i / kVec].w[(i % kVec) * (int)sizeof(T) / 4];
            if constexpr (sizeof(T) == 2) return __builtin_bit_cast(T, (uint16_t)(w >> (16 * (i & 1))));
            else return __builtin_bit_cast(T, w);
        };
        auto cls = [&](int i) { return at + (i / kVec) * kT * kVec + i % kVec; };
        // a candidate is read again (few are, from the L1 or L2) instead of
        // holding 32 keys in registers
        auto key = [&](int i) {
            const int32_t x = cls(i);
            return ((uint64_t)order_of<T>(row[x]) << class_bits) | (low - (uint32_t)x);
        };
        if (c == c0 && k <= kT / 2 && c1 - c0 >= 4 * kT) {  // uniform
            uint32_t most = 0;
#pragma unroll
            for (int i = 0; i < kMine; ++i)
                if (cls(i) < c1) {
                    const uint32_t o = order_of<T>(get(i));
                    most = o > most ? o : most;
                }
            const uint32_t o = first_bound(p, most, k, VB);
            if (o > 0) {
                bound = ((uint64_t)o << class_bits) - 1;
                least = value_of<T>(o);
            }
        }
        uint32_t mask = 0;
#pragma unroll
        for (int i = 0; i < kMine; ++i)
            if (!(to_float(get(i)) < least) && (whole || cls(i) < c1)) mask |= 1u << i;
        // room for the wave's candidates; what does not fit shows in the count
        __syncthreads();
        const int before = p.count;
        __syncthreads();
        const int mine = __builtin_popcount(mask);
        int incl = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(incl, d, kWave);
            if ((int)(threadIdx.x & 63) >= d) incl += o;
        }
        int base = 0;
        if ((threadIdx.x & 63) == 63 && incl) base = atomicAdd(&p.count, incl);
        base = __shfl(base, 63, kWave) + incl - mine;
        if (base + mine <= CAP) {
#pragma unroll 1
            for (uint32_t m = mask; m; m &= m - 1) {
                const uint64_t x = key(__builtin_ctz(m));
                // a logit equal to the bound's, of a later class, keeps its place as an empty key
                p.keys[base++] = x > bound ? x : 0;
            }
        }
        __syncthreads();
        if (p.count > CAP) {  // uniform: again, a few a thread at a time
            __syncthreads();
            if (threadIdx.x == 0) p.count = before;
#pragma unroll 1
            for (int i = 0; i < kMine; i += OFFER) {
                uint64_t x[OFFER];
#pragma unroll
                for (int e = 0; e < OFFER; ++e) x[e] = (mask >> (i + e)) & 1 ? key(i + e) : 0;
                offer(p, x, k, bits, bound);
            }
            if (bound > 0) least = value_of<T>((uint32_t)((bound + 1) >> class_bits));
        }
    }
    if constexpr (FINAL) {
        write_best(p, k, bits, class_bits, row, values + r * k, index + r * k);
    } else {
        keep_best(p, k, bits);
        __syncthreads();
        uint64_t* out = best + (r * gridDim.y + blockIdx.y) * k;
        const int n = p.count < k ? p.count : k;
        for (int a = threadIdx.x; a < k; a += kT) out[a] = a < n ? p.keys[a] : 0;
    }
}

// Short rows and small k: a wave holds a row in its registers and takes the
// largest key k times (a local maximum, six exchanges, and the owner drops
// it).  Bound by those exchanges, 0.15 us each; a work-group a row spends
// 9 us in its 20 barriers on 1,024 rows of 172 classes.
constexpr int kWaveClasses = 1024;
constexpr int kWaveK = 16;

template <typename T, int PER>
__global__ __launch_bounds__(kT) void top_wave_kernel(const T* __restrict__ logits, int64_t ld, int64_t rows,
                                                      int32_t classes, int32_t class_bits, int32_t k,
                                                      T* __restrict__ values, int32_t* __restrict__ index) {
    const int lane = threadIdx.x & 63;
    const int64_t r = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6);
    if (r >= rows) return;  // uniform over the wave
    const T* row = logits + r * ld;
    const uint64_t low = (1ull << class_bits) - 1;
    uint64_t key[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int c = i * 64 + lane;
        key[i] = c < classes ? ((uint64_t)order_of<T>(row[c]) << class_bits) | (low - (uint32_t)c) : 0;
    }
    for (int a = 0; a < k; ++a) {
        uint64_t m = key[0];
#pragma unroll
        for (int i = 1; i < PER; ++i) m = key[i] > m ? key[i] : m;
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) {
            const uint64_t o = __shfl_xor((unsigned long long)m, d, kWave);
            m = o > m ? o : m;
        }
        const int c = (int)(low - (m & low));
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (key[i] == m) {  // one lane's: keys are distinct
                key[i] = 0;
                index[r * k + a] = c;
                values[r * k + a] = row[c];
            }
    }
}

// Joins the stretches of a row: `count` keys (0: none), the k largest.
template <typename T, int MAXK>
__global__ __launch_bounds__(kT) void top_join_kernel(const T* __restrict__ logits, int64_t ld,
                                                      const uint64_t* __restrict__ best, int64_t count,
                                                      int32_t class_bits, int32_t k, T* __restrict__ values,
                                                      int32_t* __restrict__ index) {
    __shared__ Pool<MAXK> p;
    const int64_t r = blockIdx.x;
    if (threadIdx.x == 0) p.count = 0;
    const int bits = (int)sizeof(T) * 8 + class_bits;
    uint64_t bound = 0;
    constexpr int OFFER = Sizes<MAXK>::OFFER;
    for (int64_t c = 0; c < count; c += kT * OFFER) {
        uint64_t x[OFFER];
#pragma unroll
        for (int i = 0; i < OFFER; ++i) {
            const int64_t at = c + i * kT + threadIdx.x;
            x[i] = at < count ? best[r * count + at] : 0;
        }
        offer(p, x, k, bits, bound);
    }
    write_best(p, k, bits, class_bits, logits + r * ld, values + r * k, index + r * k);
}

constexpr int64_t kMostRows = 1 << 23;  // of a launch (they need no stretches)

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
    int32_t class_bits = 1;
    while ((1ll << class_bits) < classes) ++class_bits;
    if (rows > kMostRows) {  // a work-group of 256 a row: 2^32 threads are not launched
        const size_t e = dtype_size(dtype);
        for (int64_t r = 0; r < rows; r += kMostRows)
            GRWS_TRY(grws_top_logits(static_cast<const char*>(logits) + r * ld * e, dtype, ld,
                                     rows - r < kMostRows ? rows - r : kMostRows, classes, k,
                                     static_cast<char*>(values) + r * k * e, index + r * k, workspace,
                                     workspace_bytes, stream_));
        return GRWS_OK;
    }
    if (classes <= kWaveClasses && k <= kWaveK) {
        const dim3 blocks((unsigned)((rows + kWaves - 1) / kWaves));
#define GRWS_TOP_WAVE(T, PER)                                                                                    \
    hipLaunchKernelGGL((top_wave_kernel<T, PER>), blocks, dim3(kT), 0, stream, static_cast<const T*>(logits), ld, \
                       rows, (int32_t)classes, class_bits, k, static_cast<T*>(values), index)
#define GRWS_TOP_ROWS(T)                             \
    do {                                             \
        if (classes <= 256) GRWS_TOP_WAVE(T, 4);     \
        else GRWS_TOP_WAVE(T, 16);                   \
    } while (0)
        if (dtype == GRWS_F32) GRWS_TOP_ROWS(float);
        else if (dtype == GRWS_F16) GRWS_TOP_ROWS(_Float16);
        else GRWS_TOP_ROWS(__hip_bfloat16);
#undef GRWS_TOP_ROWS
#undef GRWS_TOP_WAVE
        GRWS_LAUNCH_CHECK();
        return GRWS_OK;
    }
    const int32_t n = stretches(rows, classes, k);
    Carver cv(workspace, workspace_bytes);
    uint64_t* best = n > 1 ? cv.take<uint64_t>((size_t)rows * n * k) : nullptr;
    if (!cv.ok)
        return set_error(GRWS_E_CAPACITY, "top_logits: workspace too small (%zu < %zu)", workspace_bytes, cv.used);
    const int32_t stretch = (int32_t)((classes + n - 1) / n);
    const dim3 grid((unsigned)rows, (unsigned)n);
#define GRWS_TOP_K(T, MAXK)                                                                                        \
    do {                                                                                                           \
        const T* x = static_cast<const T*>(logits);                                                                \
        T* v = static_cast<T*>(values);                                                                            \
        if (n == 1) {                                                                                              \
            hipLaunchKernelGGL((top_rows_kernel<T, true, MAXK>), grid, dim3(kT), 0, stream, x, ld,                 \
                               (int32_t)classes, class_bits, k, stretch, v, index, best);                          \
        } else {                                                                                                   \
            hipLaunchKernelGGL((top_rows_kernel<T, false, MAXK>), grid, dim3(kT), 0, stream, x, ld,                \
                               (int32_t)classes, class_bits, k, stretch, v, index, best);                          \
            GRWS_LAUNCH_CHECK();                                                                                   \
            hipLaunchKernelGGL((top_join_kernel<T, MAXK>), dim3((unsigned)rows), dim3(kT), 0, stream, x, ld, best, \
                               (int64_t)n * k, class_bits, k, v, index);                                           \
        }                                                                                                          \
    } while (0)
#define GRWS_TOP(T)                                \
    do {                                           \
        if (k <= kSmallK) GRWS_TOP_K(T, kSmallK);  \
        else GRWS_TOP_K(T, kMaxK);                 \
    } while (0)
    if (dtype == GRWS_F32) GRWS_TOP(float);
    else if (dtype == GRWS_F16) GRWS_TOP(_Float16);
    else GRWS_TOP(__hip_bfloat16);
#undef GRWS_TOP
#undef GRWS_TOP_K
    GRWS_LAUNCH_CHECK();
    return GRWS_OK;
}
