// The pool of the largest keys of a row, which top.hip and logp.hip find top
// logits with (gfx950).
//
// Every logit becomes a 64-bit key, the order-preserving bits of the value
// above the complement of the class, so keys are distinct, a larger key is a
// larger logit, and of equal logits the lowest class comes first.  -0 equals
// +0 and a NaN is larger than everything, as in torch's sort.
#pragma once

#include "grws_internal.h"

namespace grws {
namespace {

constexpr int kT = 256;          // threads of a work-group
constexpr int kWaves = kT / kWave;
constexpr int kMaxK = 1024;
constexpr int kVec = 8;          // logits of a load (two loads of f32)
constexpr int kLoads = 4;        // loads a thread has in flight
constexpr int kMine = kVec * kLoads;
constexpr int kChunk = kT * kMine;  // logits of a step
constexpr int kSmallK = 128;

// Keys in LDS, and keys a thread offers at a time where they might not fit:
// for k up to MAXK they take k + kT OFFER at most.  The small pool (11 KB, 64
// registers) lets 8 work-groups onto a CU where the large one lets 5: 308 ->
// 225 us for 64 of 8,192 x 50,021 bf16.
template <int MAXK>
struct Sizes {
    static constexpr int CAP = MAXK <= kSmallK ? 1024 : 3 * 1024;
    static constexpr int OFFER = MAXK <= kSmallK ? 2 : 8;
    static constexpr int PER = CAP / kT;
    static_assert(MAXK + kT * OFFER <= CAP, "an offer has to fit");
};

// Order-preserving bits of a logit: 16 for the 16-bit types, 32 for f32.
template <typename T>
__device__ __forceinline__ uint32_t order_of(T x) {
    constexpr uint32_t SIGN = sizeof(T) == 2 ? 0x8000u : 0x80000000u;
    constexpr uint32_t ALL = SIGN | (SIGN - 1);
    uint32_t u;
    if constexpr (sizeof(T) == 2) u = __builtin_bit_cast(uint16_t, x);
    else u = __builtin_bit_cast(uint32_t, x);
    const float f = to_float(x);
    if (f != f) return ALL;
    if (f == 0.f) u = 0;
    return u & SIGN ? ~u & ALL : u | SIGN;
}

// The logit with these order bits (a NaN for the largest).
template <typename T>
__device__ __forceinline__ float value_of(uint32_t o) {
    constexpr uint32_t SIGN = sizeof(T) == 2 ? 0x8000u : 0x80000000u;
    constexpr uint32_t ALL = SIGN | (SIGN - 1);
    const uint32_t u = o & SIGN ? o & (SIGN - 1) : ~o & ALL;
    if constexpr (sizeof(T) == 2) return to_float(__builtin_bit_cast(T, (uint16_t)u));
    else return __uint_as_float(u);
}

template <int MAXK>
struct Pool {
    uint64_t keys[Sizes<MAXK>::CAP];
    int32_t hist[2][256];
    uint32_t most[kT];  // the threads' maxima
    uint32_t first;     // the first bound's order bits
    int32_t count;
};

// The need-th largest bin from the top: the digit, the keys in it, and how
// many of them are needed.  Every wave works it out for itself.
__device__ __forceinline__ int find_digit(const int32_t* hist, int& need, int& in_bin) {
    const int lane = threadIdx.x & 63;
    int c[4], sum = 0;  // lane 0 holds the four largest digits
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        c[j] = hist[255 - 4 * lane - j];
        sum += c[j];
    }
    int incl = sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(incl, d, kWave);
        if (lane >= d) incl += o;
    }
    const int l = __builtin_ctzll(__ballot(incl >= need));
    int above = __shfl(incl - sum, l, kWave);
    int digit = 0, in = 0;
    bool found = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int x = __shfl(c[j], l, kWave);
        if (!found) {
            if (above + x >= need) {
                found = true;
                digit = 255 - 4 * l - j;
                in = x;
            } else {
                above += x;
            }
        }
    }
    need -= above;
    in_bin = in;
    return digit;
}

// Keeps the k largest keys of the pool, of `bits` bits (all, when there are
// no more), and returns a bound that exactly they reach (0: all).
template <int MAXK>
__device__ __forceinline__ uint64_t keep_best(Pool<MAXK>& p, int k, int bits) {
    constexpr int PER = Sizes<MAXK>::PER;
    __syncthreads();
    const int n = p.count;
    if (n <= k) return 0;  // uniform over the work-group
    uint64_t mine[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int at = i * kT + threadIdx.x;
        mine[i] = at < n ? p.keys[at] : 0;
    }
    p.hist[0][threadIdx.x] = 0;
    uint64_t bound = 0;
    int need = k, turn = 0;
    for (int shift = (bits + 7) / 8 * 8 - 8; shift >= 0; shift -= 8, turn ^= 1) {
        __syncthreads();  // this histogram is clear, the last one read
        p.hist[turn ^ 1][threadIdx.x] = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            // of the keys with the bound's digits above
            if (mine[i] != 0 && ((mine[i] ^ bound) >> shift) < 256)
                atomicAdd(&p.hist[turn][(mine[i] >> shift) & 255], 1);
        }
        __syncthreads();
        int in_bin;
        const int digit = find_digit(p.hist[turn], need, in_bin);
        bound |= (uint64_t)digit << shift;
        if (in_bin == need) break;  // the whole bin is in
    }
    if (threadIdx.x == 0) p.count = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const bool in = mine[i] >= bound && mine[i] != 0;
        const uint64_t b = __ballot(in);
        if (!b) continue;  // uniform over the wave
        int at = 0;
        if ((threadIdx.x & 63) == 0) at = atomicAdd(&p.count, __builtin_popcountll(b));
        at = __shfl(at, 0, kWave) + __builtin_popcountll(b & lanemask_lt());
        if (in) p.keys[at] = mine[i];
    }
    __syncthreads();
    return bound;
}

// Offers every thread's N keys (0: none) to the pool, which has room for
// them or is cut to its best.  `bound`: keys up to it are not wanted.
template <int MAXK, int N>
__device__ __forceinline__ void offer(Pool<MAXK>& p, const uint64_t (&x)[N], int k, int bits, uint64_t& bound) {
    static_assert(N == Sizes<MAXK>::OFFER, "keys of an offer");
    __syncthreads();
    if (p.count + kT * N > Sizes<MAXK>::CAP) {  // uniform: the count is read after the barrier
        const uint64_t b = keep_best(p, k, bits);
        if (b > 0 && b - 1 > bound) bound = b - 1;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const bool in = x[i] > bound;
        const uint64_t b = __ballot(in);
        if (!b) continue;
        int at = 0;
        if ((threadIdx.x & 63) == 0) at = atomicAdd(&p.count, __builtin_popcountll(b));
        at = __shfl(at, 0, kWave) + __builtin_popcountll(b & lanemask_lt());
        if (in) p.keys[at] = x[i];
    }
}

// put(place, class) for the pool's k largest, by counting the larger ones.
template <int MAXK, typename F>
__device__ __forceinline__ void put_best(Pool<MAXK>& p, int k, int bits, int class_bits, F put) {
    keep_best(p, k, bits);
    __syncthreads();
    const int n = p.count < k ? p.count : k;
    const uint64_t low = (1ull << class_bits) - 1;
    for (int a = threadIdx.x; a < n; a += kT) {
        const uint64_t key = p.keys[a];
        int rank = 0;
        for (int b = 0; b < n; ++b) rank += p.keys[b] > key;
        put(rank, (int32_t)(low - (key & low)));
    }
}

// put(place, key) for the pool's k largest, by counting the larger ones: of few
// keys all of them, without finding the k-th first.
template <int MAXK, typename F>
__device__ __forceinline__ void put_ranked(Pool<MAXK>& p, int k, int bits, F put) {
    __syncthreads();
    int n = p.count;
    if (n > kT) {  // uniform
        keep_best(p, k, bits);
        __syncthreads();
        n = p.count < k ? p.count : k;
    }
    for (int a = threadIdx.x; a < n; a += kT) {
        const uint64_t key = p.keys[a];
        int rank = 0;
#pragma unroll 8
        for (int b = 0; b < n; ++b) rank += p.keys[b] > key;
        if (key != 0 && rank < k) put(rank, key);
    }
}

// The first bound: order bits that at least k of the threads' maxima reach
// (their upper 16 bits; the first wave, 4 maxima a lane).
template <int MAXK>
__device__ __forceinline__ uint32_t first_bound(Pool<MAXK>& p, uint32_t most, int k, int value_bits) {
    p.most[threadIdx.x] = most;
    __syncthreads();
    if (threadIdx.x < kWave) {
        uint32_t m[kWaves];
#pragma unroll
        for (int j = 0; j < kWaves; ++j) m[j] = p.most[threadIdx.x + j * kWave];
        uint32_t bound = 0;
        for (int bit = value_bits - 1; bit >= value_bits - 16; --bit) {
            const uint32_t trial = bound | (1u << bit);
            int c = 0;
#pragma unroll
            for (int j = 0; j < kWaves; ++j) c += __builtin_popcountll(__ballot(m[j] >= trial));
            if (c >= k) bound = trial;
        }
        if (threadIdx.x == 0) p.first = bound;
    }
    __syncthreads();
    return p.first;
}

// A V from any address.  ONCE: what does not fit into the last cache goes past
// them (8,192 x 50,048 bf16 forward 126 us against 141; of 16,384 x 5,003, which
// do fit, 51 against 46).
template <bool ONCE, typename V>
__device__ __forceinline__ V load_vec(const void* p) {
    static_assert(sizeof(V) % 16 == 0, "whole loads");
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4), aligned(2)));
    u32x4 w[sizeof(V) / 16];
#pragma unroll
    for (int i = 0; i < (int)(sizeof(V) / 16); ++i)
        if constexpr (ONCE) w[i] = __builtin_nontemporal_load(static_cast<const u32x4*>(p) + i);
        else w[i] = static_cast<const u32x4*>(p)[i];
    V v;
    __builtin_memcpy(&v, w, sizeof(V));
    return v;
}

// Elements before the first that lies at a whole 16 bytes, of `most`.  (Loads of
// 16 bytes that do not take twice the time: 4,099 rows of 100,003 bf16, every
// other one at an odd element, 219 us against 186.)
template <typename T>
__device__ __forceinline__ int32_t before_aligned(const T* p, int32_t most) {
    const int32_t n = (int32_t)((0 - reinterpret_cast<uintptr_t>(p)) & 15) / (int32_t)sizeof(T);
    return n < most ? n : most;
}

// A work-group's step through a row: load i of a thread has the logits from
// at + 2,048 i on, kVec of them; where those go past the end, the last kVec of
// the row, of which the first are not its own (rows have kVec logits or more).
template <typename T>
struct Chunk {
    struct Vec {
        uint32_t w[kVec * sizeof(T) / 4];
    };
    Vec v[kLoads];
    int32_t at, c1;
    bool whole;  // uniform

    // logits c.. of a stretch that ends at `end`
    template <bool ONCE>
    __device__ __forceinline__ void load(const T* row, int32_t c, int32_t end) {
        at = c + (int32_t)threadIdx.x * kVec;
        c1 = end;
        whole = c + kChunk <= c1;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) v[i] = load_vec<ONCE, Vec>(row + from(i));
    }
    // first class of load i
    __device__ __forceinline__ int32_t from(int i) const {
        const int32_t f = at + i * kT * kVec;
        return whole || f + kVec <= c1 ? f : c1 - kVec;
    }
    __device__ __forceinline__ T get(int i) const {
        const uint32_t w = v[i / kVec].w[(i % kVec) * (int)sizeof(T) / 4];
        if constexpr (sizeof(T) == 2) return __builtin_bit_cast(T, (uint16_t)(w >> (16 * (i & 1))));
        else return __builtin_bit_cast(T, w);
    }
    __device__ __forceinline__ int32_t cls(int i) const { return from(i / kVec) + i % kVec; }
    __device__ __forceinline__ bool in(int i) const { return whole || cls(i) >= at + i / kVec * kT * kVec; }
};

// Offers a step's logits to the pool.  c0: the stretch's first class; bound:
// keys up to it are not wanted; least: the bound's logit, smaller ones are not
// looked at (they begin as 0 and -inf).
template <int MAXK, typename T>
__device__ __forceinline__ void offer_chunk(Pool<MAXK>& p, const Chunk<T>& v, const T* row, int32_t c, int32_t c0,
                                            int32_t c1, int32_t class_bits, int32_t k, uint64_t& bound,
                                            float& least) {
    constexpr int VB = sizeof(T) * 8, CAP = Sizes<MAXK>::CAP, OFFER = Sizes<MAXK>::OFFER;
    const int bits = VB + class_bits;
    const uint64_t low = (1ull << class_bits) - 1;
    // a candidate is read again (few are, from the L1 or L2) instead of
    // holding 32 keys in registers
    auto key = [&](int i) {
        const int32_t x = v.cls(i);
        return ((uint64_t)order_of<T>(row[x]) << class_bits) | (low - (uint32_t)x);
    };
    if (c == c0 && k <= kT / 2 && c1 - c0 >= 4 * kT) {  // uniform
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < kMine; ++i)
            if (v.in(i)) {
                const uint32_t o = order_of<T>(v.get(i));
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
        if (!(to_float(v.get(i)) < least) && v.in(i)) mask |= 1u << i;
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

}  // namespace
}  // namespace grws
