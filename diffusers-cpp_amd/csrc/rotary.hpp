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
    const double t = (double)pos * (double)freq;
    const double q = rint(t * kHi);
    Quarter r;
    r.f = __builtin_fma(t, kLo, __builtin_fma(t, kHi, -q));
    r.n = (int)(q - 4.0 * floor(q * 0.25));
    return r;
}

// Whole quarter turns put back: (cos, sin) of x + n pi / 2.
template <typename F>
__device__ __forceinline__ void unfold(int n, F co, F si, F mul, F* c, F* s) {
    const F a = (n & 1) ? si : co, b = (n & 1) ? co : si;
    *c = ((n + 1) & 2) ? -a * mul : a * mul;
    *s = (n & 2) ? -b * mul : b * mul;
}

// In 32 bits: the terms left out are below 2e-9 of the result.
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

// The 16 elements a thread rotates: two runs of 8 at a and b.  Halves: run b holds the
// partners of run a, pair e of the unit is (a[e], b[e]), and pair 8 u + e of the head.  Pairs:
// the 16 are in order, pair e is (2 e, 2 e + 1).  Units behind the rotated part are in order too.
struct Unit {
    int a, b;
    __device__ __forceinline__ Unit(int u, int rot, bool half) {
        const bool split = half && 16 * u < rot;
        a = split ? 8 * u : 16 * u;
        b = split ? 8 * u + rot / 2 : 16 * u + 8;
    }
};

template <typename F>
struct Angles {
    F c[8], s[8];
    __device__ __forceinline__ void set(int pos, const float* freq, int u, int rot, F mul) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            c[e] = mul;
            s[e] = 0;
            if (2 * (8 * u + e) < rot) cos_sin(pos, freq[8 * u + e], mul, &c[e], &s[e]);
        }
    }
    // v: run a, then run b.  Elements behind the rotated part stay as they are.
    __device__ __forceinline__ void turn(F (&v)[16], int u, int rot, bool half, F sign) const {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (2 * (8 * u + e) >= rot) continue;
            const F si = s[e] * sign;
            F x = half ? v[e] : v[2 * e], y = half ? v[8 + e] : v[2 * e + 1];
            const F x1 = x * c[e] - y * si, y1 = y * c[e] + x * si;
            if (half) {
                v[e] = x1;
                v[8 + e] = y1;
            } else {
                v[2 * e] = x1;
                v[2 * e + 1] = y1;
            }
        }
    }
};

}  // namespace rotary
}  // namespace dit
