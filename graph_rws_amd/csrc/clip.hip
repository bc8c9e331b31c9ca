// The global norm of many gradients, and clipping by it (gfx950): the end of
// every training step.
//
//   norm = |scale| sqrt(sum over the tensors of g^2)
//   out  = g scale min(1, max_norm / (norm + 1e-6))
//
// Squares are summed in 64 bits (f32 gradients of 1e-23 or 1e19 have squares
// that 32 bits do not hold, and 5e8 of them a sum that 32 bits round): the
// 64-bit multiply-add runs at the f32 rate here, and the pass stays bound by
// HBM (5.4e8 bf16: 166 us, 6.5 TB/s; clipped into f32 another 575, 5.6 TB/s read
// and written; in place 548 in all, where a norm and a scaling a tensor take
// 2,090).  Two launches of up to kTensors tensors each: the first leaves a
// partial sum per work-group, the second adds those up in its every
// work-group (in one order, so all agree and the same inputs give the same
// bits) and scales.
#include "grws_internal.h"

#include <algorithm>
#include <memory>
#include <new>

namespace grws {
namespace {

constexpr int kT = 256;        // threads of a work-group
constexpr int kChunk = 8192;   // elements of a work-group's step
constexpr int kTensors = 64;   // of a launch: what fits into its arguments
constexpr int kBlocks = 1024;  // work-groups of a launch: 4 a CU (5.4e8 bf16 with 512: 827 us against 741)
// What the last cache (256 MB) keeps for the second pass, or with the outputs
// for what follows; beyond it loads and stores go past the caches (of 5e8 bf16
// the squares 164 us against 180, of 5e7 f32 norm and clipping 92 against 106).
constexpr int64_t kCached = (int64_t)192 << 20;

struct Tensors {
    const void* src[kTensors];
    void* dst[kTensors];
    int64_t size[kTensors];
    int64_t first[kTensors + 1];  // chunks before the tensor
    uint8_t src_dt[kTensors], dst_dt[kTensors];
    int32_t count;
};

template <typename T, int N>
struct Vec {
    T x[N];
};

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2), aligned(2)));

// elements at.. of x, zeros from `size` on; any alignment.  ONCE: past the
// caches.
template <bool ONCE, int N, typename T>
__device__ __forceinline__ Vec<T, N> load_vec(const T* x, int64_t at, int64_t size) {
    typedef std::conditional_t<N * sizeof(T) % 16 == 0, u32x4_t, u32x2_t> W;
    constexpr int C = N * sizeof(T) / sizeof(W);
    Vec<T, N> v;
    if (at + N <= size) {
        W w[C];
#pragma unroll
        for (int i = 0; i < C; ++i) {
            const W* p = reinterpret_cast<const W*>(x + at) + i;
            if constexpr (ONCE) w[i] = __builtin_nontemporal_load(p);
            else w[i] = *p;
        }
        __builtin_memcpy(&v, w, sizeof(v));
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) v.x[e] = at + e < size ? x[at + e] : from_float<T>(0.f);
    }
    return v;
}

__device__ __forceinline__ double block_sum(double s, double* red) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) s += __shfl_xor(s, d, kWave);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    s = 0.0;
#pragma unroll
    for (int w = 0; w < kT / kWave; ++w) s += red[w];
    return s;
}

// The tensor of chunk c.
__device__ __forceinline__ int tensor_of(const Tensors& a, int64_t c) {
    int lo = 0, hi = a.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.first[mid] <= c) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// use(tensor, first element of the chunk) for every gridDim-th chunk (the
// work-groups read neighbouring memory; runs of it a work-group: 772 us against
// 741 for 5e8 bf16); the dtype of a chunk is uniform.
template <typename F>
__device__ __forceinline__ void for_chunks(const Tensors& a, F use) {
    const int64_t n = a.first[a.count];
    if (blockIdx.x >= n) return;
    int t = tensor_of(a, blockIdx.x);
    for (int64_t c = blockIdx.x; c < n; c += gridDim.x) {
        while (c >= a.first[t + 1]) ++t;
        use(t, (c - a.first[t]) * kChunk);
    }
}

template <bool ONCE, typename T>
__device__ __forceinline__ double squares(const void* src, int64_t from, int64_t size) {
    constexpr int N = 16 / sizeof(T), LOADS = kChunk / (kT * N);
    const T* x = static_cast<const T*>(src);
    Vec<T, N> v[LOADS];
#pragma unroll
    for (int l = 0; l < LOADS; ++l) v[l] = load_vec<ONCE, N>(x, from + ((int64_t)l * kT + threadIdx.x) * N, size);
    double s = 0.0;
#pragma unroll
    for (int l = 0; l < LOADS; ++l)
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const double g = (double)to_float(v[l].x[e]);
            s = __builtin_fma(g, g, s);
        }
    return s;
}

template <bool ONCE>
__global__ __launch_bounds__(kT) void clip_squares_kernel(Tensors a, double* __restrict__ part) {
    __shared__ double red[kT / kWave];
    double s = 0.0;
    for_chunks(a, [&](int t, int64_t from) {
        if (a.src_dt[t] == GRWS_F32) s += squares<ONCE, float>(a.src[t], from, a.size[t]);
        else if (a.src_dt[t] == GRWS_F16) s += squares<ONCE, _Float16>(a.src[t], from, a.size[t]);
        else s += squares<ONCE, __hip_bfloat16>(a.src[t], from, a.size[t]);
    });
    s = block_sum(s, red);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}

__device__ __forceinline__ double norm_of(const double* __restrict__ part, int parts, const float* scale,
                                          double* red) {
    double s = 0.0;
    for (int k = threadIdx.x; k < parts; k += kT) s += part[k];
    s = sqrt(block_sum(s, red));
    return scale ? fabs((double)*scale) * s : s;
}

__global__ __launch_bounds__(kT) void clip_norm_kernel(const double* __restrict__ part, int parts,
                                                       const float* scale, float* __restrict__ norm) {
    __shared__ double red[kT / kWave];
    const double n = norm_of(part, parts, scale, red);
    if (threadIdx.x == 0) *norm = (float)n;
}

// keep = f tail.  Beside gradients near the largest float keep may lie below the
// smallest normal one, where f32 has few bits or none: then f is 2^126 of it
// (the product stays finite) and tail takes that off.
struct Factor {
    float f, tail;
};

__device__ __forceinline__ Factor factor_of(double keep) {
    const bool low = fabs(keep) < 0x1p-126;
    return Factor{(float)(low ? keep * 0x1p126 : keep), low ? 0x1p-126f : 1.f};
}

// (A lane stores 16 bytes next to its neighbour's, so it reads 8 of 16-bit
// gradients that go to f32.)
template <bool ONCE, typename T, typename O>
__device__ __forceinline__ void scale_chunk(const void* src, void* dst, int64_t from, int64_t size, Factor f) {
    constexpr int N = 16 / sizeof(O), LOADS = kChunk / (kT * N);
    const T* x = static_cast<const T*>(src);
    O* o = static_cast<O*>(dst);
    Vec<T, N> v[LOADS];
#pragma unroll
    for (int l = 0; l < LOADS; ++l) v[l] = load_vec<ONCE, N>(x, from + ((int64_t)l * kT + threadIdx.x) * N, size);
#pragma unroll
    for (int l = 0; l < LOADS; ++l) {
        const int64_t at = from + ((int64_t)l * kT + threadIdx.x) * N;
        Vec<O, N> w;
#pragma unroll
        for (int e = 0; e < N; ++e) w.x[e] = from_float<O>(to_float(v[l].x[e]) * f.f * f.tail);
        if (at + N <= size) {
            u32x4_t x4;
            __builtin_memcpy(&x4, &w, sizeof(w));
            u32x4_t* p = reinterpret_cast<u32x4_t*>(o + at);
            if constexpr (ONCE) __builtin_nontemporal_store(x4, p);
            else *p = x4;
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (at + e < size) o[at + e] = w.x[e];
        }
    }
}

// A factor of exactly one leaves gradients that are clipped in place as they
// are (in_place), without reading them a second time.
template <bool ONCE>
__global__ __launch_bounds__(kT) void clip_scale_kernel(Tensors a, const double* __restrict__ part, int parts,
                                                        float max_norm, const float* scale, int32_t in_place,
                                                        float* __restrict__ norm) {
    __shared__ double red[kT / kWave];
    double n = norm_of(part, parts, scale, red);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
    if ((float)n == INFINITY) n = INFINITY;  // what f32 does not hold clips as it is returned
    double keep = (double)max_norm / (n + 1e-6);
    if (keep > 1.0) keep = 1.0;  // (a NaN stays)
    if (scale) keep *= (double)*scale;
    const Factor f = factor_of(keep);
    if (in_place && f.f == 1.f && f.tail == 1.f) return;  // uniform
    for_chunks(a, [&](int t, int64_t from) {
        const void* x = a.src[t];
        void* o = a.dst[t];
        const int64_t size = a.size[t];
        const int s = a.src_dt[t], d = a.dst_dt[t];
        if (d == s) {
            if (s == GRWS_F32) scale_chunk<ONCE, float, float>(x, o, from, size, f);
            else if (s == GRWS_F16) scale_chunk<ONCE, _Float16, _Float16>(x, o, from, size, f);
            else scale_chunk<ONCE, __hip_bfloat16, __hip_bfloat16>(x, o, from, size, f);
        } else if (s == GRWS_F16) {
            scale_chunk<ONCE, _Float16, float>(x, o, from, size, f);
        } else {
            scale_chunk<ONCE, __hip_bfloat16, float>(x, o, from, size, f);
        }
    });
}

bool known(int32_t dt) { return dt == GRWS_F32 || dt == GRWS_F16 || dt == GRWS_BF16; }

// Whether an output shares memory with another output, or with a gradient
// that is not its own (which would be read before and after it is written).
// Ranges in the order of their beginnings: a written one may not begin before
// all others have ended, a read one not before the written ones have.
struct Range {
    uintptr_t lo, hi;
    bool written;
};

int check_apart(const void* const* grads, const int32_t* dtypes, const int64_t* sizes, void* const* outs,
                const int32_t* out_dtypes, int32_t count) {
    std::unique_ptr<Range[]> r(new (std::nothrow) Range[2 * (size_t)count]);
    if (!r) return set_error(GRWS_E_CAPACITY, "clip: out of host memory");
    size_t n = 0;
    for (int32_t i = 0; i < count; ++i) {
        if (sizes[i] == 0) continue;
        const uintptr_t g = reinterpret_cast<uintptr_t>(grads[i]), o = reinterpret_cast<uintptr_t>(outs[i]);
        r[n++] = Range{o, o + sizes[i] * dtype_size(out_dtypes ? out_dtypes[i] : dtypes[i]), true};
        if (g != o) r[n++] = Range{g, g + sizes[i] * dtype_size(dtypes[i]), false};
    }
    std::sort(r.get(), r.get() + n, [](const Range& a, const Range& b) { return a.lo < b.lo; });
    uintptr_t any = 0, written = 0;
    for (size_t i = 0; i < n; ++i) {
        // (of two that begin together either order finds the overlap)
        GRWS_CHECK_ARG(r[i].lo >= (r[i].written ? any : written), "clip: tensors overlap, or one is listed twice");
        any = std::max(any, r[i].hi);
        if (r[i].written) written = std::max(written, r[i].hi);
    }
    return GRWS_OK;
}

// Calls use(Tensors, its work-groups) for the tensors, kTensors of them at a
// time; empty ones are left out.
template <typename F>
int for_launches(const void* const* grads, const int32_t* dtypes, const int64_t* sizes, void* const* outs,
                 const int32_t* out_dtypes, int32_t count, F use) {
    Tensors a;
    a.count = 0;
    a.first[0] = 0;
    for (int32_t i = 0; i <= count; ++i) {
        if (a.count == kTensors || (i == count && a.count > 0)) {
            const int64_t chunks = a.first[a.count];
            GRWS_TRY(use(a, (unsigned)(chunks < kBlocks ? chunks : kBlocks)));
            a.count = 0;
        }
        if (i == count) break;
        if (sizes[i] == 0) continue;
        const int t = a.count++;
        a.src[t] = grads[i];
        a.dst[t] = outs ? outs[i] : nullptr;
        a.src_dt[t] = (uint8_t)dtypes[i];
        a.dst_dt[t] = (uint8_t)(out_dtypes ? out_dtypes[i] : dtypes[i]);
        a.size[t] = sizes[i];
        a.first[t + 1] = a.first[t] + (sizes[i] + kChunk - 1) / kChunk;
    }
    return GRWS_OK;
}

}  // namespace
}  // namespace grws

using namespace grws;

extern "C" size_t grws_clip_workspace_bytes(int32_t count) {
    Sizer s;
    s.take<double>((size_t)((count > 0 ? count : 0) + kTensors) / kTensors * kBlocks);
    return s.used;
}

extern "C" int grws_clip_grads(const void* const* grads, const int32_t* dtypes, const int64_t* sizes,
                               void* const* outs, const int32_t* out_dtypes, int32_t count, float max_norm,
                               const float* scale, float* norm, void* workspace, size_t workspace_bytes,
                               void* stream_) {
    clear_error();
    hipStream_t stream = as_stream(stream_);
    GRWS_CHECK_ARG(count >= 0 && (count == 0 || (grads && dtypes && sizes)), "clip: null lists");
    GRWS_CHECK_ARG(norm || outs, "clip: nothing to compute");
    GRWS_CHECK_ARG(!outs || max_norm >= 0.f, "clip: max_norm must not be negative");
    int32_t in_place = 1;
    int64_t bytes = 0, all_bytes = 0;
    for (int32_t i = 0; i < count; ++i) {
        const int32_t d = out_dtypes ? out_dtypes[i] : dtypes[i];
        if (!known(dtypes[i]) || !known(d))
            return set_error(GRWS_E_DTYPE, "clip: unsupported dtype %d", known(dtypes[i]) ? d : dtypes[i]);
        if (d != dtypes[i] && d != GRWS_F32)
            return set_error(GRWS_E_DTYPE, "clip: an output has its gradient's dtype or is f32");
        GRWS_CHECK_ARG(sizes[i] >= 0, "clip: negative size");
        if (sizes[i] == 0) continue;
        GRWS_CHECK_ARG(grads[i] && (!outs || outs[i]), "clip: null tensor");
        bytes += sizes[i] * (int64_t)dtype_size(dtypes[i]);
        all_bytes += sizes[i] * (int64_t)(dtype_size(dtypes[i]) + (outs ? dtype_size(d) : 0));
        if (outs && outs[i] != grads[i]) in_place = 0;
        GRWS_CHECK_ARG(!outs || outs[i] != grads[i] || d == dtypes[i], "clip: in place is in one dtype");
    }
    if (outs) GRWS_TRY(check_apart(grads, dtypes, sizes, outs, out_dtypes, count));
    Carver cv(workspace, workspace_bytes);
    double* part = cv.take<double>((size_t)(count + kTensors) / kTensors * kBlocks);
    if (!cv.ok) return set_error(GRWS_E_CAPACITY, "clip: workspace too small (%zu < %zu)", workspace_bytes, cv.used);
    int parts = 0;
    GRWS_TRY(for_launches(grads, dtypes, sizes, outs, out_dtypes, count, [&](const Tensors& a, unsigned blocks) -> int {
        double* to = part + parts;
        if (bytes > kCached) hipLaunchKernelGGL(clip_squares_kernel<true>, dim3(blocks), dim3(kT), 0, stream, a, to);
        else hipLaunchKernelGGL(clip_squares_kernel<false>, dim3(blocks), dim3(kT), 0, stream, a, to);
        GRWS_LAUNCH_CHECK();
        parts += (int)blocks;
        return GRWS_OK;
    }));
    if (!outs || parts == 0) {
        if (norm) {
            hipLaunchKernelGGL(clip_norm_kernel, dim3(1), dim3(kT), 0, stream, part, parts, scale, norm);
            GRWS_LAUNCH_CHECK();
        }
        return GRWS_OK;
    }
    float* first = norm;
    return for_launches(grads, dtypes, sizes, outs, out_dtypes, count, [&](const Tensors& a, unsigned blocks) -> int {
        if (all_bytes > kCached)
            hipLaunchKernelGGL(clip_scale_kernel<true>, dim3(blocks), dim3(kT), 0, stream, a, part, parts, max_norm,
                               scale, in_place, first);
        else
            hipLaunchKernelGGL(clip_scale_kernel<false>, dim3(blocks), dim3(kT), 0, stream, a, part, parts, max_norm,
                               scale, in_place, first);
        GRWS_LAUNCH_CHECK();
        first = nullptr;
        return GRWS_OK;
    });
}
