// Log probabilities of given classes, entropy and top alternatives of rows of
// logits in memory, and their gradient (gfx950).
//
//   m the largest z, u_v = (z_v - m) log2(e) / T, s = sum 2^u, t = sum 2^u u
//   ln p_v = (z_v - m) / T - ln s        logp_j = ln p_cj
//   H = ln s - ln2 t / s
//   dz_v = (sum_j a_j [v = c_j] - p_v (A + b (ln p_v + H))) / T
// with a_j the upstream gradient of logp_j, b that of H, A the sum of a_j.
// t <= 0 and s >= 1, so H adds two terms of one sign and nothing cancels.
//
// Forward: one pass.  Every thread keeps its own (m, s, t) and moves them to a
// new m when some of its logits are larger (rare after the first steps); the
// work-group joins them at the end, in a fixed order.  Few rows are cut into
// stretches and joined, short ones take a wave each.  Bound by HBM: 8,192 x
// 50,048 bf16 124 us, 6.6 TB/s (a bare read 7.1); an element takes 9 of the
// vector unit's slots, 4 of them for the exponential, 90 us in all.
// Backward: the logits are read again and the gradient written, 8,192 x 50,048
// bf16 320 us, 5.1 TB/s (a copy 5.0).
#include "logp.h"
#include "top_pool.h"

namespace grws {
namespace {

// The classes whose log probabilities are asked for: k a row; a negative
// one asks for nothing (0), one past the last is an error (NaN).
struct Given {
    const void* index;
    int32_t k, i64;
    __device__ __forceinline__ int64_t at(int64_t r, int j) const {
        return i64 ? static_cast<const int64_t*>(index)[r * k + j]
                   : (int64_t) static_cast<const int32_t*>(index)[r * k + j];
    }
};

struct Outputs {
    float* logp;      // [rows k]
    float* entropy;   // [rows]
    float2* saved;    // [rows]: m, s; or NULL
    float* top_logp;  // [rows top]
    int32_t* top_index;
};

// The factors of T: c1 = log2(e) / T.
struct Scale {
    float c1, inv_t;
};

// What a row's statistics say of logit z (in natural units: a mask of the
// type's lowest value stays finite).
struct Row {
    float m, l2, inv_t;  // largest logit, log2 s
    __device__ __forceinline__ float logp(float z) const { return at_most_zero(fmaf(z - m, inv_t, -kLn2 * l2)); }
};

__device__ __forceinline__ Row row_of(const Stats& a, const Scale& sc) {
    return Row{a.m, a.m == -INFINITY ? __int_as_float(0x7fc00000) : log2f(a.s), sc.inv_t};
}

// A thread's first given class and its logit, asked for before the pass over
// the row: two reads that follow one another.
struct Early {
    int64_t cls;
    float z;
};

template <typename T>
__device__ __forceinline__ Early early_given(const T* row, int64_t r, int32_t classes, const Given& g, int sub) {
    Early e{-1, 0.f};
    if (sub < g.k) e.cls = g.at(r, sub);
    if (e.cls >= 0 && e.cls < classes) e.z = to_float(row[e.cls]);
    return e;
}

// The row's outputs, `lanes` threads of which this is `sub`.
template <typename T>
__device__ __forceinline__ void put_row(const Stats& a, const Scale& sc, const T* row, int64_t r, int32_t classes,
                                        const Given& g, Early e, const Outputs& o, int sub, int lanes) {
    const Row q = row_of(a, sc);
    for (int j = sub; j < g.k; j += lanes) {
        if (j != sub) e = early_given(row, r, classes, g, j);
        float v = 0.f;
        if (e.cls >= classes) v = __int_as_float(0x7fc00000);
        else if (e.cls >= 0) v = q.logp(e.z);
        o.logp[r * g.k + j] = v;
    }
    if (sub != 0) return;
    o.entropy[r] = q.l2 != q.l2 ? q.l2 : entropy_of(a);
    if (o.saved) o.saved[r] = make_float2(q.m, a.s);
}

// The pool's alternatives; a key holds its logit.
template <typename T, int MAXK>
__device__ __forceinline__ void put_top(Pool<MAXK>& p, const Row& q, int64_t r, int32_t class_bits, int32_t top,
                                        const Outputs& o) {
    const uint64_t low = (1ull << class_bits) - 1;
    put_ranked(p, top, (int)sizeof(T) * 8 + class_bits, [&](int at, uint64_t key) {
        o.top_index[r * top + at] = (int32_t)(low - (key & low));
        o.top_logp[r * top + at] = q.logp(value_of<T>((uint32_t)(key >> class_bits)));
    });
}

// What a thread has added: s and t against ref, the rounded m c1, and what that
// rounding took; or against m c1 itself, where that is far from zero: ref is
// +inf then, so that the first pass over the logits leaves a t that is not a
// number, and the second has the differences.
struct Running {
    Stats a = no_stats();
    float ref = 0.f;

    // what ref's rounding took
    __device__ __forceinline__ float past(float c1) const {
        return fabsf(a.m) == INFINITY || fabsf(ref) == INFINITY ? 0.f : fmaf(-a.m, c1, ref);
    }
    // Adds N logits; the largest of them.
    template <int N>
    __device__ __forceinline__ float add(const float (&z)[N], float c1) {
        float m = z[0];
#pragma unroll
        for (int i = 1; i < N; ++i) m = fmaxf(m, z[i]);
        if (m > a.m) {
            const float d = (a.m - m) * c1 + past(c1);
            a.m = m;
            ref = is_far(m, c1) ? INFINITY : m * c1;
            move(a, d - past(c1));
        }
        const float s = a.s, t = a.t;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float u = fmaf(z[i], c1, -ref), e = __builtin_amdgcn_exp2f(u);
            a.s += e;
            a.t = fmaf(e, u, a.t);
        }
        if (a.t != a.t && a.s == a.s) {  // a zero times an infinity: again
            a.s = s;
            a.t = t;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float u = ref == INFINITY ? (z[i] - a.m) * c1 : fmaf(z[i], c1, -ref);
                const float e = __builtin_amdgcn_exp2f(u);
                a.s += e;
                a.t = fmaf(e, reach(u), a.t);
            }
        }
        return m;
    }
    // Adds a step's logits; the largest of them.
    template <typename T>
    __device__ __forceinline__ float add(const Chunk<T>& v, float c1) {
        float m = -INFINITY;
        if (v.whole) {
            // in halves: fewer registers, so one wave more a SIMD
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float z[kMine / 2];
#pragma unroll
                for (int i = 0; i < kMine / 2; ++i) z[i] = to_float(v.get(h * (kMine / 2) + i));
                m = fmaxf(m, add(z, c1));
            }
            return m;
        }
#pragma unroll
        for (int l = 0; l < kLoads; ++l) {
            if (v.at - (int)(threadIdx.x & 63) * kVec + l * kT * kVec >= v.c1) break;  // nothing of the wave's: uniform
            float z[kVec];
#pragma unroll
            for (int e = 0; e < kVec; ++e) z[e] = v.in(l * kVec + e) ? to_float(v.get(l * kVec + e)) : -INFINITY;
            m = fmaxf(m, add(z, c1));
        }
        return m;
    }
    // against m c1 itself
    __device__ __forceinline__ Stats stats(float c1) {
        move(a, past(c1));
        return a;
    }
};

// Where the alternatives of small `top` are: every thread leaves the largest
// logit of each of its runs of steps, at least `top` threads' largest
// reach a first bound, and only runs that reach it are looked at again.  So the
// pass over the row has no barrier and no candidates (8,192 x 50,021 bf16 with
// 16 alternatives: 151 us, 470 with a pool that every step offers to).
template <typename T>
struct Runs {
    typedef std::conditional_t<sizeof(T) == 2, uint16_t, uint32_t> Order;
    static constexpr int GROUPS = 32 / sizeof(T);  // of a thread: 8 KB a work-group
    Order most[GROUPS][kT];
};

template <typename T, int MAXK>
__device__ __forceinline__ void offer_runs(Pool<MAXK>& p, Runs<T>& runs, int32_t groups, int32_t steps, const T* row,
                                           int32_t first, int32_t end, int32_t class_bits, int32_t top) {
    constexpr int VB = sizeof(T) * 8, OFFER = Sizes<MAXK>::OFFER, GROUPS = Runs<T>::GROUPS;
    constexpr uint32_t ALL = VB == 16 ? 0xffffu : 0xffffffffu;
    const uint64_t low = (1ull << class_bits) - 1;
    uint32_t order[GROUPS], mine = 0;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
        order[g] = g < groups ? runs.most[g][threadIdx.x] : 0;
        mine = order[g] > mine ? order[g] : mine;
    }
    // (a NaN, or an infinity whose sum is one, stands for the largest: where
    // they are the bound, all runs are looked at)
    uint32_t reach = top <= kT / 2 ? first_bound(p, mine, top, VB) : 0;
    if ((reach >> (VB - 16)) >= (ALL >> (VB - 16))) reach = 0;
    __syncthreads();
    if (threadIdx.x == 0) p.first = 0;
    __syncthreads();
    uint32_t in = 0;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g)
        if (g < groups && order[g] >= reach) in |= 1u << g;
    uint16_t* chosen = reinterpret_cast<uint16_t*>(runs.most);  // every thread has read its runs
    if (in) {
        int at = (int)atomicAdd(&p.first, (uint32_t)__builtin_popcount(in));
        for (uint32_t m = in; m; m &= m - 1) chosen[at++] = (uint16_t)(__builtin_ctz(m) * kT + (int)threadIdx.x);
    }
    __syncthreads();
    uint64_t bound = reach > 0 ? ((uint64_t)reach << class_bits) - 1 : 0;
    const int32_t run = steps * kMine;
    const int64_t count = (int64_t)p.first * run;
    for (int64_t c = 0; c < count; c += kT * OFFER) {
        uint64_t x[OFFER];
#pragma unroll
        for (int e = 0; e < OFFER; ++e) {
            const int64_t at = c + e * kT + (int)threadIdx.x;
            x[e] = 0;
            if (at < count) {
                const int32_t k = (int32_t)(at / run), i = (int32_t)(at - (int64_t)k * run);  // logit i of the run
                const int64_t step = (int64_t)(chosen[k] / kT) * steps * kChunk + (int64_t)(i / kVec) * kT * kVec;
                const int64_t cls = first + step + chosen[k] % kT * kVec + i % kVec;
                if (cls < end) x[e] = ((uint64_t)order_of<T>(row[cls]) << class_bits) | (low - (uint32_t)cls);
            }
        }
        offer(p, x, top, VB + class_bits, bound);
    }
}

// A work-group a row, or a stretch of one (FINAL false: its statistics and
// keys go to `part` and `best`).  MAXK 0: no alternatives.
template <typename T, bool FINAL, int MAXK, bool ONCE>
__global__ __launch_bounds__(kT) void logp_rows_kernel(const T* __restrict__ logits, int64_t ld, int64_t r0,
                                                       int32_t classes, int32_t class_bits, int32_t top,
                                                       int32_t stretch, Scale sc, Given g, Outputs o,
                                                       float4* __restrict__ part, uint64_t* __restrict__ best) {
    constexpr bool RUNS = MAXK == kSmallK;
    __shared__ Pool<MAXK ? MAXK : 1> p;
    __shared__ std::conditional_t<RUNS, Runs<T>, int> runs;
    __shared__ float sm[kWaves], ss[kWaves], st[kWaves];
    const int64_t r = r0 + blockIdx.x;
    const T* row = logits + r * ld;
    const int32_t first = (int32_t)blockIdx.y * stretch;
    const int32_t end = classes - first < stretch ? classes : first + stretch;
    const int bits = (int)sizeof(T) * 8 + class_bits;
    uint64_t bound = 0;
    float least = -INFINITY;
    Running sum;
    Early early{-1, 0.f};
    if constexpr (FINAL) early = early_given(row, r, classes, g, threadIdx.x);
    // what lies before a whole 16 bytes: a logit a thread
    const int32_t head = end > first ? before_aligned(row + first, end - first) : 0, begin = first + head;
    if ((int32_t)threadIdx.x < head) {
        const float z[1] = {to_float(row[first + threadIdx.x])};
        sum.add(z, sc.c1);
    }
    const int32_t all_steps = end > begin ? (end - begin + kChunk - 1) / kChunk : 0;
    const int32_t steps = (all_steps + Runs<T>::GROUPS - 1) / Runs<T>::GROUPS;  // of a run
    float run = -INFINITY;
    int32_t group = 0, left = steps;
    if constexpr (MAXK) {
        __syncthreads();
        if ((int32_t)threadIdx.x < head)
            p.keys[threadIdx.x] = ((uint64_t)order_of<T>(row[first + threadIdx.x]) << class_bits) |
                                  (((1ull << class_bits) - 1) - (uint32_t)(first + threadIdx.x));
        if (threadIdx.x == 0) p.count = head;
        __syncthreads();
    }
    for (int32_t c = begin; c < end; c += kChunk) {
        Chunk<T> v;
        v.template load<ONCE>(row, c, end);
        const float m = sum.add(v, sc.c1);
        if constexpr (RUNS) {
            run = fmaxf(run, m);
            if (--left == 0 || c + kChunk >= end) {
                runs.most[group++][threadIdx.x] = order_of<T>(from_float<T>(sum.a.s == sum.a.s ? run : sum.a.s));
                run = -INFINITY;
                left = steps;
            }
        } else if constexpr (MAXK) {
            offer_chunk<MAXK>(p, v, row, c, begin, end, class_bits, top, bound, least);
        }
    }
    Stats a = join_wave(sum.stats(sc.c1), sc.c1);
    if ((threadIdx.x & 63) == 0) {
        sm[threadIdx.x >> 6] = a.m;
        ss[threadIdx.x >> 6] = a.s;
        st[threadIdx.x >> 6] = a.t;
    }
    __syncthreads();
    a = Stats{sm[0], ss[0], st[0]};
#pragma unroll
    for (int w = 1; w < kWaves; ++w) a = join(a, Stats{sm[w], ss[w], st[w]}, sc.c1);
    if constexpr (RUNS) offer_runs<T>(p, runs, group, steps, row, begin, end, class_bits, top);
    if constexpr (FINAL) {
        put_row(a, sc, row, r, classes, g, early, o, threadIdx.x, kT);
        if constexpr (MAXK) {
            put_top<T>(p, row_of(a, sc), r, class_bits, top, o);
        }
    } else {
        const int64_t at = blockIdx.x * (int64_t)gridDim.y + blockIdx.y;
        if (threadIdx.x == 0) part[at] = make_float4(a.m, a.s, a.t, 0.f);
        if constexpr (MAXK) {
            for (int j = threadIdx.x; j < top; j += kT) best[at * top + j] = 0;  // (a barrier follows)
            put_ranked(p, top, bits, [&](int j, uint64_t key) { best[at * top + j] = key; });
        }
    }
}

// Joins the stretches of a row.
template <typename T, int MAXK>
__global__ __launch_bounds__(kT) void logp_join_kernel(const T* __restrict__ logits, int64_t ld, int64_t r0,
                                                       int32_t classes, int32_t class_bits, int32_t top,
                                                       int32_t stretches, Scale sc, Given g, Outputs o,
                                                       const float4* __restrict__ part,
                                                       const uint64_t* __restrict__ best) {
    __shared__ Pool<MAXK ? MAXK : 1> p;
    const int64_t r = r0 + blockIdx.x;
    const T* row = logits + r * ld;
    const Early early = early_given(row, r, classes, g, threadIdx.x);
    Stats a = no_stats();
    // every wave joins them all, in one order
    for (int w = threadIdx.x & 63; w < stretches; w += 64) {
        const float4 x = part[blockIdx.x * (int64_t)stretches + w];
        a = join(a, Stats{x.x, x.y, x.z}, sc.c1);
    }
    a = join_wave(a, sc.c1);
    put_row(a, sc, row, r, classes, g, early, o, threadIdx.x, kT);
    if constexpr (MAXK) {
        if (threadIdx.x == 0) p.count = 0;
        constexpr int OFFER = Sizes<MAXK>::OFFER;
        const int bits = (int)sizeof(T) * 8 + class_bits;
        const int64_t count = (int64_t)stretches * top;
        uint64_t bound = 0;
        if (top <= kT / 2) {  // what `top` of the threads' largest keys reach
            constexpr int VB = sizeof(T) * 8;
            uint32_t most = 0;
            for (int64_t c = threadIdx.x; c < count; c += kT) {
                const uint32_t x = (uint32_t)(best[blockIdx.x * count + c] >> class_bits);
                most = x > most ? x : most;
            }
            const uint32_t reach = first_bound(p, most, top, VB);
            if (reach > 0) bound = ((uint64_t)reach << class_bits) - 1;
        }
        for (int64_t c = 0; c < count; c += kT * OFFER) {
            uint64_t x[OFFER];
#pragma unroll
            for (int i = 0; i < OFFER; ++i) {
                const int64_t at = c + i * kT + threadIdx.x;
                x[i] = at < count ? best[blockIdx.x * count + at] : 0;
            }
            offer(p, x, top, bits, bound);
        }
        put_top<T>(p, row_of(a, sc), r, class_bits, top, o);
    }
}

// Short rows: a wave holds a row in its registers; the alternatives as in
// top_wave_kernel, the largest key `top` times.
constexpr int kWaveClasses = 1024;
constexpr int kWaveTop = 16;

template <typename T, int PER>
__global__ __launch_bounds__(kT) void logp_wave_kernel(const T* __restrict__ logits, int64_t ld, int64_t r0,
                                                       int64_t rows,
                                                       int32_t classes, int32_t class_bits, int32_t top, Scale sc,
                                                       Given g, Outputs o) {
    const int lane = threadIdx.x & 63;
    const int64_t r = r0 + (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6);
    if (r >= rows) return;  // uniform over the wave
    const T* row = logits + r * ld;
    const Early early = early_given(row, r, classes, g, lane);
    T x[PER];
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int c = i * 64 + lane;
        x[i] = c < classes ? row[c] : from_float<T>(-INFINITY);
        m = fmaxf(m, to_float(x[i]));
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor(m, d, kWave));
    Stats a{m, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < PER; ++i) add(a, to_float(x[i]), m == -INFINITY ? 0.f : m, sc.c1);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        a.s += __shfl_xor(a.s, d, kWave);
        a.t += __shfl_xor(a.t, d, kWave);
    }
    put_row(a, sc, row, r, classes, g, early, o, lane, 64);
    if (top == 0) return;
    const Row q = row_of(a, sc);
    const uint64_t low = (1ull << class_bits) - 1;
    uint64_t key[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int c = i * 64 + lane;
        key[i] = c < classes ? ((uint64_t)order_of<T>(x[i]) << class_bits) | (low - (uint32_t)c) : 0;
    }
    for (int n = 0; n < top; ++n) {
        uint64_t best = key[0];
#pragma unroll
        for (int i = 1; i < PER; ++i) best = key[i] > best ? key[i] : best;
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) {
            const uint64_t other = __shfl_xor((unsigned long long)best, d, kWave);
            best = other > best ? other : best;
        }
        const int c = (int)(low - (best & low));
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (key[i] == best) {  // one lane's: keys are distinct
                key[i] = 0;
                o.top_index[r * top + n] = c;
                o.top_logp[r * top + n] = q.logp(to_float(x[i]));
            }
    }
}

// ---------------------------------------------------------------------------
// the gradient
// ---------------------------------------------------------------------------
struct Upstream {
    const float* dlogp;     // [rows k], or NULL: zeros
    const float* dentropy;  // [rows], or NULL: zeros
};

// The sum of a_j of a row's given classes, `LANES` lanes of a wave together.
__device__ __forceinline__ float given_sum(const Given& g, const Upstream& up, int64_t r, int32_t classes, int lane) {
    float s = 0.f;
    if (!up.dlogp) return s;
    for (int j = lane; j < g.k; j += 64) {
        const int64_t c = g.at(r, j);
        if (c >= 0 && c < classes) s += up.dlogp[r * g.k + j];
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) s += __shfl_xor(s, d, kWave);
    return s;
}

// dz of a logit that is not given: -p (A + b (ln p + H)) / T.  A row of
// nothing but -inf (s of 0) has no p: zeros, so that it can be left out of a
// loss.  NaN beside them, which m does not show, is in s and f: NaN everywhere.
struct Slope {
    float m, c1, f, k, b2;  // f = -1 / (s T), k = A + b (H - ln s), b2 = b ln2
    __device__ __forceinline__ float of(float z) const {
        if (m == -INFINITY) return f == f ? 0.f : f;  // uniform
        const float u = (z - m) * c1;
        return __builtin_amdgcn_exp2f(u) * f * fmaf(b2, reach(u), k);
    }
};

template <bool ONCE, typename V>
__device__ __forceinline__ void store_vec(void* p, const V& v) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4), aligned(2)));
    u32x4 w[sizeof(V) / 16];
    __builtin_memcpy(w, &v, sizeof(V));
#pragma unroll
    for (int i = 0; i < (int)(sizeof(V) / 16); ++i) {
        if constexpr (ONCE) __builtin_nontemporal_store(w[i], static_cast<u32x4*>(p) + i);
        else static_cast<u32x4*>(p)[i] = w[i];
    }
}

// 16 bytes a thread at a time of a stretch of one row (ONE), or of four rows, a
// wave each (1,024 rows of 172: 5 us).  Given classes are put in place after the
// rest: the wave's stores (ONE: the work-group's, behind a barrier) have left
// before the same places are written again.  (Rows that begin inside 16 bytes
// are read and written as they lie: beginning at a whole 16 took 362 us against
// 351 for 4,099 x 100,003 bf16.)
template <typename T, bool ONE, bool ONCE>
__global__ __launch_bounds__(kT) void logp_grad_kernel(const T* __restrict__ logits, int64_t ld, int64_t r0,
                                                       int64_t rows, int32_t classes, int32_t stretch, float c1,
                                                       float inv_t, Given g, Upstream up,
                                                       const float2* __restrict__ saved,
                                                       const float* __restrict__ entropy, T* __restrict__ out,
                                                       int64_t ldo) {
    constexpr int N = ONE ? kT : 64;  // threads of a row
    const int sub = ONE ? threadIdx.x : threadIdx.x & 63;
    const int64_t r = r0 + (ONE ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6));
    if (r >= rows) return;  // uniform over the row's threads
    const int32_t first = (int32_t)blockIdx.y * stretch;
    const int32_t end = classes - first < stretch ? classes : first + stretch;
    const T* row = logits + r * ld;
    T* to = out + r * ldo;
    const float2 s = saved[r];
    const float b = up.dentropy ? up.dentropy[r] : 0.f;
    const float A = given_sum(g, up, r, classes, threadIdx.x & 63);
    const Slope f{s.x, c1, -inv_t / s.y, up.dentropy ? fmaf(b, entropy[r] - kLn2 * log2f(s.y), A) : A, b * kLn2};
    constexpr int E = 16 / sizeof(T);  // a lane's 16 bytes lie next to its neighbour's
    struct Vec {
        T x[E];
    };
    for (int32_t c = first + sub * E; c < end; c += N * E) {
        if (c + E <= end) {
            Vec v = load_vec<ONCE, Vec>(row + c);
#pragma unroll
            for (int e = 0; e < E; ++e) v.x[e] = from_float<T>(f.of(to_float(v.x[e])));
            store_vec<ONCE>(to + c, v);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (c + e < end) to[c + e] = from_float<T>(f.of(to_float(row[c + e])));
        }
    }
    if (!up.dlogp || f.m == -INFINITY) return;  // uniform
    __threadfence_block();
    if constexpr (ONE) __syncthreads();
    for (int j = sub; j < g.k; j += N) {
        const int64_t c = g.at(r, j);
        if (c < first || c >= end) continue;
        float a = up.dlogp[r * g.k + j];
        bool again = false;  // an earlier entry has the class: it adds this one
        for (int o = 0; o < j && !again; ++o) again = g.at(r, o) == c;
        if (again) continue;
        for (int o = j + 1; o < g.k; ++o)
            if (g.at(r, o) == c) a += up.dlogp[r * g.k + o];
        to[c] = from_float<T>(fmaf(a, inv_t, f.of(to_float(row[c]))));
    }
}

constexpr int64_t kMostBlocks = 1 << 23;  // of a launch: 2^31 threads
constexpr int32_t kGradStretch = kChunk;

// Work-groups of the rows left, a wave a row, in one launch.
unsigned wave_blocks(int64_t rows) {
    const int64_t n = (rows + kWaves - 1) / kWaves;
    return (unsigned)(n < kMostBlocks ? n : kMostBlocks);
}

// Stretches of a row: as many as it takes to fill the chip when there are few
// rows, of at least 2,048 logits and 4 `top`.
int32_t stretches(int64_t rows, int64_t classes, int64_t top) {
    int64_t n = (1024 + rows - 1) / rows;
    const int64_t least = 4 * top > 2048 ? 4 * top : 2048;
    const int64_t most = classes / least;
    if (n > most) n = most;
    return n < 1 ? 1 : (int32_t)n;
}

// Whether logits are read past the caches: those that do not fit into the last
// one (256 MB), where the backward would find them.
bool streams(int64_t bytes) { return bytes > ((int64_t)192 << 20); }

bool by_wave(int64_t classes, int64_t top) { return classes <= kWaveClasses && top <= kWaveTop; }

int check(const char* what, int32_t dtype, int64_t ld, int64_t rows, int64_t classes, int32_t k, float temperature) {
    if (dtype != GRWS_F32 && dtype != GRWS_F16 && dtype != GRWS_BF16)
        return set_error(GRWS_E_DTYPE, "%s: unsupported dtype %d", what, dtype);
    GRWS_CHECK_ARG(rows >= 0 && rows <= INT32_MAX && classes > 0 && classes <= INT32_MAX - 65536 && ld >= classes,
                   "%s: bad sizes", what);
    GRWS_CHECK_ARG(k >= 1 && k <= 1024, "%s: 1 to 1024 given classes a row", what);
    GRWS_CHECK_ARG(temperature > 0.f && temperature < INFINITY && kLog2e / temperature < INFINITY,
                   "%s: the temperature must be positive", what);
    return GRWS_OK;
}

int32_t bits_of(int64_t classes) {
    int32_t b = 1;
    while ((1ll << b) < classes) ++b;
    return b;
}

template <typename T>
int forward(const T* x, int64_t ld, int64_t rows, int32_t classes, int32_t top, const Scale& sc, const Given& g,
            const Outputs& o, float4* part, uint64_t* best, hipStream_t stream) {
    const int32_t cb = bits_of(classes);
    if (by_wave(classes, top)) {
        for (int64_t r0 = 0; r0 < rows; r0 += kMostBlocks * kWaves) {
            const dim3 grid(wave_blocks(rows - r0));
            if (classes <= 256)
                hipLaunchKernelGGL((logp_wave_kernel<T, 4>), grid, dim3(kT), 0, stream, x, ld, r0, rows, classes, cb,
                                   top, sc, g, o);
            else
                hipLaunchKernelGGL((logp_wave_kernel<T, 16>), grid, dim3(kT), 0, stream, x, ld, r0, rows, classes, cb,
                                   top, sc, g, o);
            GRWS_LAUNCH_CHECK();
        }
        return GRWS_OK;
    }
    const int32_t n = stretches(rows, classes, top);
    const bool once = streams(rows * classes * (int64_t)sizeof(T));
    const int32_t stretch = (int32_t)(((int64_t)classes + n - 1) / n + 63) / 64 * 64;  // (the last may be empty)
    for (int64_t r0 = 0; r0 < rows; r0 += kMostBlocks) {  // (with several stretches there are fewer than 1,024 rows)
        const dim3 grid((unsigned)(rows - r0 < kMostBlocks ? rows - r0 : kMostBlocks), (unsigned)n);
#define GRWS_LOGP(MAXK)                                                                                              \
    do {                                                                                                             \
        if (n == 1) {                                                                                                \
            if (once && MAXK != kMaxK)                                                                               \
                hipLaunchKernelGGL((logp_rows_kernel<T, true, MAXK, MAXK != kMaxK>), grid, dim3(kT), 0, stream, x,   \
                                   ld, r0, classes, cb, top, stretch, sc, g, o, part, best);                         \
            else                                                                                                     \
                hipLaunchKernelGGL((logp_rows_kernel<T, true, MAXK, false>), grid, dim3(kT), 0, stream, x, ld, r0,   \
                                   classes, cb, top, stretch, sc, g, o, part, best);                                 \
        } else {                                                                                                     \
            hipLaunchKernelGGL((logp_rows_kernel<T, false, MAXK, false>), grid, dim3(kT), 0, stream, x, ld, r0,      \
                               classes, cb, top, stretch, sc, g, o, part, best);                                     \
            GRWS_LAUNCH_CHECK();                                                                                     \
            hipLaunchKernelGGL((logp_join_kernel<T, MAXK>), dim3(grid.x), dim3(kT), 0, stream, x, ld, r0, classes,   \
                               cb, top, n, sc, g, o, part, best);                                                    \
        }                                                                                                            \
    } while (0)
        if (top == 0) GRWS_LOGP(0);
        else if (top <= kSmallK) GRWS_LOGP(kSmallK);
        else GRWS_LOGP(kMaxK);
#undef GRWS_LOGP
        GRWS_LAUNCH_CHECK();
    }
    return GRWS_OK;
}

template <typename T>
int backward(const T* x, int64_t ld, int64_t rows, int32_t classes, float c1, float inv_t, const Given& g,
             const Upstream& up, const float2* saved, const float* entropy, T* out, int64_t ldo, hipStream_t stream) {
    if (classes <= kWaveClasses) {
        for (int64_t r0 = 0; r0 < rows; r0 += kMostBlocks * kWaves) {
            hipLaunchKernelGGL((logp_grad_kernel<T, false, false>), dim3(wave_blocks(rows - r0)), dim3(kT), 0, stream,
                               x, ld, r0, rows, classes, classes, c1, inv_t, g, up, saved, entropy, out, ldo);
            GRWS_LAUNCH_CHECK();
        }
        return GRWS_OK;
    }
    // (at most 2^15 stretches of a row: a grid's second dimension ends at 2^16)
    const int64_t pieces = ((int64_t)classes + kGradStretch - 1) / kGradStretch;
    const int32_t stretch = kGradStretch * (int32_t)((pieces + 32767) / 32768);
    const int64_t n = ((int64_t)classes + stretch - 1) / stretch;
    const int64_t most = kMostBlocks / n < 1 ? 1 : kMostBlocks / n;
    const bool once = streams(rows * classes * (int64_t)sizeof(T));
    for (int64_t r0 = 0; r0 < rows; r0 += most) {
        const dim3 grid((unsigned)(rows - r0 < most ? rows - r0 : most), (unsigned)n);
#define GRWS_LOGP_GRAD(ONCE)                                                                                         \
    hipLaunchKernelGGL((logp_grad_kernel<T, true, ONCE>), grid, dim3(kT), 0, stream, x, ld, r0, rows, classes,       \
                       stretch, c1, inv_t, g, up, saved, entropy, out, ldo)
        if (once) GRWS_LOGP_GRAD(true);
        else GRWS_LOGP_GRAD(false);
#undef GRWS_LOGP_GRAD
        GRWS_LAUNCH_CHECK();
    }
    return GRWS_OK;
}

}  // namespace
}  // namespace grws

using namespace grws;

extern "C" size_t grws_log_probs_workspace_bytes(int64_t rows, int64_t classes, int32_t top) {
    if (rows <= 0 || classes <= 0 || top < 0 || by_wave(classes, top)) return 0;
    const int32_t n = stretches(rows, classes, top);
    if (n == 1) return 0;
    Sizer s;
    s.take<float4>((size_t)rows * n);
    s.take<uint64_t>((size_t)rows * n * top);
    return s.used;
}

extern "C" int grws_log_probs_fwd(const void* logits, int32_t dtype, int64_t ld, int64_t rows, int64_t classes,
                                  const void* index, int32_t index_is_i64, int32_t k, int32_t top, float temperature,
                                  float* logp, float* entropy, float* saved, float* top_logp, int32_t* top_index,
                                  void* workspace, size_t workspace_bytes, void* stream_) {
    clear_error();
    hipStream_t stream = as_stream(stream_);
    GRWS_TRY(check("log_probs", dtype, ld, rows, classes, k, temperature));
    GRWS_CHECK_ARG(top >= 0 && top <= kMaxK && top <= classes, "log_probs: top must be 0..min(classes, 1024)");
    if (rows == 0) return GRWS_OK;
    GRWS_CHECK_ARG(logits && index && logp && entropy && (top == 0 || (top_logp && top_index)),
                   "log_probs: null pointer");
    const int32_t n = by_wave(classes, top) ? 1 : stretches(rows, classes, top);
    Carver cv(workspace, workspace_bytes);
    float4* part = n > 1 ? cv.take<float4>((size_t)rows * n) : nullptr;
    uint64_t* best = n > 1 ? cv.take<uint64_t>((size_t)rows * n * top) : nullptr;
    if (!cv.ok)
        return set_error(GRWS_E_CAPACITY, "log_probs: workspace too small (%zu < %zu)", workspace_bytes, cv.used);
    const Given g{index, k, index_is_i64};
    const Outputs o{logp, entropy, reinterpret_cast<float2*>(saved), top_logp, top_index};
    const Scale sc{kLog2e / temperature, 1.f / temperature};
#define GRWS_LOGP_FWD(T)                                                                                         \
    return forward(static_cast<const T*>(logits), ld, rows, (int32_t)classes, top, sc, g, o, part, best, stream)
    if (dtype == GRWS_F32) GRWS_LOGP_FWD(float);
    if (dtype == GRWS_F16) GRWS_LOGP_FWD(_Float16);
    GRWS_LOGP_FWD(__hip_bfloat16);
#undef GRWS_LOGP_FWD
}

extern "C" int grws_log_probs_bwd(const void* logits, int32_t dtype, int64_t ld, int64_t rows, int64_t classes,
                                  const void* index, int32_t index_is_i64, int32_t k, float temperature,
                                  const float* saved, const float* entropy, const float* dlogp,
                                  const float* dentropy, void* grad, int64_t ldg, void* stream_) {
    clear_error();
    hipStream_t stream = as_stream(stream_);
    GRWS_TRY(check("log_probs", dtype, ld, rows, classes, k, temperature));
    GRWS_CHECK_ARG(ldg >= classes, "log_probs: bad sizes");
    if (rows == 0) return GRWS_OK;
    GRWS_CHECK_ARG(logits && index && saved && entropy && grad, "log_probs: null pointer");
    const Given g{index, k, index_is_i64};
    const Upstream up{dlogp, dentropy};
    const float c1 = kLog2e / temperature;
#define GRWS_LOGP_BWD(T)                                                                                     \
    return backward(static_cast<const T*>(logits), ld, rows, (int32_t)classes, c1, 1.f / temperature, g, up, \
                    reinterpret_cast<const float2*>(saved), entropy, static_cast<T*>(grad), ldg, stream)
    if (dtype == GRWS_F32) GRWS_LOGP_BWD(float);
    if (dtype == GRWS_F16) GRWS_LOGP_BWD(_Float16);
    GRWS_LOGP_BWD(__hip_bfloat16);
#undef GRWS_LOGP_BWD
}
