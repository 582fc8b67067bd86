// rotary.hpp -- the angles of rotary positions, shared by the rotation itself
// (rotary.hip) and the cache that keys are rotated into (kv_cache.hip).
//
// Pair i of a head at position p turns by p * freq[i].  Far positions make the
// product large (a few 10^5 turns), so it is formed and reduced in 64 bits: to
// quarter turns f in [-1/2, 1/2] and their number, then a Taylor series in x = f pi / 2.
#pragma once

#include "common.hpp"

namespace dit {
namespace rotary {

struct Quarter {
    double f;  // quarter turns left, in [-1/2, 1/2]
    int n;     // whole quarter turns, mod 4
};

__device__ __forceinline__ Quarter quarter(int pos, float freq) {
    // 2 / pi in two parts: the second is what the first rounds off.
    constexpr double kHi = 0.63661977236758138, kLo = -3.9357353350364971e-17;
    constexpr double kWhole = 6755399441055744.0;  // 1.5 2^52: a sum with it ends in the nearest whole number
    const double t = (double)pos * (double)freq;
    const double w = __builtin_fma(t, kHi, kWhole), q = w - kWhole;
    Quarter r;
    r.f = __builtin_fma(t, kLo, __builtin_fma(t, kHi, -q));
    r.n = (int)(uint32_t)__double_as_longlong(w) & 3;
    return r;
}

// Whole quarter turns put back: (cos, sin) of x + n pi / 2.
template <typename F>
__device__ __forceinline__ void unfold(int n, F co, F si, F mul, F* c, F* s) {
    const F a = (n & 1) ? si : co, b = (n & 1) ? co : si;
    *c = ((n + 1) & 2) ? -a * mul : a * mul;
    *s = (n & 2) ? -b * mul : b * mul;
}

// In 32 bits from the angle on, which is rounded once (off by 2^-25 at most; the terms left out are below 2e-9): off by
// 2^-23 of mul at most.  Over every fp32 angle up to pi / 4, with the angle's and the factor's rounding at their worst, 2^-23.04
// for the cosine and 2^-23.22 for the sine; where mul is a power of two 2^-23.70 and 2^-23.95.  (An angle that is itself
// a product in 32 bits, off by up to 1.3 2^-24, made 2^-22.89.)
__device__ __forceinline__ void cos_sin(int pos, float freq, float mul, float* c, float* s) {
    const Quarter r = quarter(pos, freq);
    const float x = (float)(r.f * 1.5707963267948966), y = x * x;
    float co = __builtin_fmaf(y, -1.f / 3628800, 1.f / 40320);
    co = __builtin_fmaf(y, co, -1.f / 720);
    co = __builtin_fmaf(y, co, 1.f / 24);
    co = __builtin_fmaf(y, co, -0.5f);
    co = __builtin_fmaf(y, co, 1.f);
    float si = __builtin_fmaf(y, 1.f / 362880, -1.f / 5040);
    si = __builtin_fmaf(y, si, 1.f / 120);
    si = __builtin_fmaf(y, si, -1.f / 6);
    si = __builtin_fmaf(y * x, si, x);
    unfold(r.n, co, si, mul, c, s);
}

// In 64 bits (terms left out below 1e-15), for what is rounded to few bits right after: a
// value next to a border between two codes falls on the side that it belongs to.
__device__ __forceinline__ void cos_sin(int pos, float freq, double mul, double* c, double* s) {
    const Quarter r = quarter(pos, freq);
    const double x = r.f * 1.5707963267948966, y = x * x;
    double co = __builtin_fma(y, -1. / 87178291200., 1. / 479001600);
    co = __builtin_fma(y, co, -1. / 3628800);
    co = __builtin_fma(y, co, 1. / 40320);
    co = __builtin_fma(y, co, -1. / 720);
    co = __builtin_fma(y, co, 1. / 24);
    co = __builtin_fma(y, co, -0.5);
    co = __builtin_fma(y, co, 1.);
    double si = __builtin_fma(y, -1. / 1307674368000., 1. / 6227020800.);
    si = __builtin_fma(y, si, -1. / 39916800);
    si = __builtin_fma(y, si, 1. / 362880);
    si = __builtin_fma(y, si, -1. / 5040);
    si = __builtin_fma(y, si, 1. / 120);
    si = __builtin_fma(y, si, -1. / 6);
    si = __builtin_fma(y * x, si, x);
    unfold(r.n, co, si, mul, c, s);
}

// The 2 W elements a thread rotates: runs of W at a and b.  Halves: run b holds the partners of
// run a, pair e of the unit is (a[e], b[e]).  Pairs: each run holds W / 2 of them, (2 e, 2 e + 1), and
// run b follows run a, or lies `apart` units of W on (so that a wave's loads are whole rows).  Units
// behind the rotated part of halves are in order too.
template <int W>
struct Unit {
    int a, b;
    int pa, pb;  // pairs of the head: the unit's first, and its W/2th
    __device__ __forceinline__ Unit(int u, int rot, bool half, int apart = 0) {
        const bool split = half && 2 * W * u < rot;
        a = split || (!half && apart) ? W * u : 2 * W * u;
        b = split ? a + rot / 2 : !half && apart ? a + W * apart : a + W;
        pa = half ? W * u : a / 2;
        pb = half ? pa + W / 2 : b / 2;
    }
    __device__ __forceinline__ int pair(int e) const { return e < W / 2 ? pa + e : pb + e - W / 2; }
};

// Without branches: the frequencies are on their way together, and what is behind the rotated part
// is selected, never computed (0 times an infinity).
template <typename F, int W>
struct Angles {
    F c[W], s[W];
    float f[W];
    bool on[W];
    // Before the loads of what is rotated: results come in the order of the loads.  freq: a word that can
    // be read, also where nothing is rotated.
    __device__ __forceinline__ Angles(const float* freq, const Unit<W>& at, int rot) {
#pragma unroll
        for (int e = 0; e < W; ++e) {
            on[e] = 2 * at.pair(e) < rot;
            f[e] = freq[max(min(at.pair(e), rot / 2 - 1), 0)];
        }
    }
    __device__ __forceinline__ void set(int pos, F mul) {
#pragma unroll
        for (int e = 0; e < W; ++e) cos_sin(pos, f[e], mul, &c[e], &s[e]);
    }
    template <bool HALF>
    __device__ __forceinline__ void turn_as(F (&v)[2 * W], F sign) const {
#pragma unroll
        for (int e = 0; e < W; ++e) {
            F &x = HALF ? v[e] : v[2 * e], &y = HALF ? v[W + e] : v[2 * e + 1];
            const F si = s[e] * sign, x1 = x * c[e] - y * si, y1 = y * c[e] + x * si;
            x = on[e] ? x1 : x;
            y = on[e] ? y1 : y;
        }
    }
    // v: run a, then run b.
    __device__ __forceinline__ void turn(F (&v)[2 * W], bool half, F sign) const {
        if (half) turn_as<true>(v, sign);
        else turn_as<false>(v, sign);
    }
};

// Unit u of up to ITER heads of one token, whose angles are worked out once: x(i) is where the i-th
// head is read if has(i), y(i) where it is written.
template <typename T, int ITER, typename H, typename X, typename Y>
__device__ __forceinline__ void turn_heads(int pos, const float* freq, int u, int units, int rot, bool half, float mul, float sign, H has, X x,
                                           Y y) {
    constexpr int W = Io<T>::EPV;
    const Unit<W> at(u, rot, half, units);
    Angles<float, W> w(freq, at, rot);
    uint4 raw[ITER][2];
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        if (!has(i)) continue;
        const T* p = x(i);
        raw[i][0] = ld_stream(p + at.a);
        raw[i][1] = ld_stream(p + at.b);
    }
    w.set(pos, mul);
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        if (!has(i)) continue;
        T* p = y(i);
        float v[2 * W];
        Io<T>::unpack(raw[i][0], v);
        Io<T>::unpack(raw[i][1], v + W);
        w.turn(v, half, sign);
        st_stream(p + at.a, Io<T>::pack(v));
        st_stream(p + at.b, Io<T>::pack(v + W));
    }
}

}  // namespace rotary
}  // namespace dit
