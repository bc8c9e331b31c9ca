// What log probabilities and entropies take of a row's logits, for logp.hip and
// head.hip (gfx950).  With T a temperature, m the largest of some logits and
// u_v = (z_v - m) log2(e) / T:
//   s = sum 2^u, t = sum 2^u u,    ln sum exp(z / T) = m / T + ln s
//   entropy = ln s - ln2 t / s     (t <= 0 and s >= 1: two terms of one sign)
#pragma once

#include "grws_internal.h"

namespace grws {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// (m, s, t) of some of a row's logits; nothing of them: m = -inf, s = t = 0.
struct Stats {
    float m, s, t;
};

__device__ __forceinline__ Stats no_stats() { return Stats{-INFINITY, 0.f, 0.f}; }

// 2^u u and 2^d (s d + t) below -200 are zero: infinities would leave NaN
__device__ __forceinline__ float reach(float u) { return fmaxf(u, -200.f); }

// s and t seen from a larger m, d = (old m - new m) log2(e) / T further down
// (-inf where there was nothing)
__device__ __forceinline__ void move(Stats& a, float d) {
    d = reach(d);
    const float f = __builtin_amdgcn_exp2f(d);
    a.t = fmaf(d, a.s, a.t) * f;
    a.s *= f;
}

__device__ __forceinline__ Stats join(Stats a, Stats b, float c1) {
    // a NaN logit shows in s; largest values are compared without it
    const float m = fmaxf(a.m, b.m);
    if (m == -INFINITY) return Stats{m, a.s + b.s, a.t + b.t};  // zeros, or NaN
    move(a, (a.m - m) * c1);
    move(b, (b.m - m) * c1);
    return Stats{m, a.s + b.s, a.t + b.t};
}

__device__ __forceinline__ void add(Stats& a, float z, float m, float c1) {
    const float u = (z - m) * c1, e = __builtin_amdgcn_exp2f(u);
    a.s += e;
    a.t = fmaf(e, reach(u), a.t);
}

// Roundings leave no log probability above zero and no entropy below it (a NaN
// stays).
__device__ __forceinline__ float at_most_zero(float x) { return x > 0.f ? 0.f : x; }

__device__ __forceinline__ float entropy_of(const Stats& a) {
    const float h = kLn2 * (log2f(a.s) - a.t / a.s);
    return h < 0.f ? 0.f : h;
}

// The exponentials are 2^(z c1 - ref), ref the rounded m c1 of a largest logit
// m, and what that rounding took is put back.  Where m c1 is 2^30 or more (masks
// of -1e30, temperatures next to zero) the rounding alone can be 2^6 and soon
// is more than an exponent: there they are 2^((z - m) c1).
__device__ __forceinline__ bool is_far(float m, float c1) {
    return fabsf(m * c1) >= 1073741824.f && fabsf(m) != INFINITY;
}

// The wave's, in every lane: the largest m first, then sums against it.
__device__ __forceinline__ Stats join_wave(Stats a, float c1) {
    float m = a.m;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor(m, d, kWave));
    if (m != -INFINITY) move(a, (a.m - m) * c1);
    a.m = m;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        a.s += __shfl_xor(a.s, d, kWave);
        a.t += __shfl_xor(a.t, d, kWave);
    }
    return a;
}

}  // namespace
}  // namespace grws
