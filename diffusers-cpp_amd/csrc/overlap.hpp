// overlap.hpp -- whether two strided operands share memory, in plain C++ that the C
// entries (rotary.hip, kv_cache.hip, kv_attention.hip) and a host program can build.
#pragma once

#include <stdint.h>

namespace dit {

// Runs of `run` bytes at base + sum of i_k step_k, 0 <= i_k < n_k.
struct Strided {
    typedef __int128 wide;  // strides below 2^42 bytes times sizes below 2^30
    wide base, run;
    int dims;
    wide n[3], step[3];
    // `count` dimensions of n elements and `strides` (in elements of es bytes) of rows of `width` elements.
    Strided(const void* p, int es, int count, const int64_t* sizes, const int64_t* strides, int64_t width)
        : base((uintptr_t)p), run((wide)width * es), dims(0) {
        for (int i = 0; i < count; ++i) {  // by their steps, those of one element, or of one element repeated, left out
            if (sizes[i] == 1 || strides[i] == 0) continue;
            int at = dims++;
            for (; at > 0 && step[at - 1] > (wide)strides[i] * es; --at) {
                n[at] = n[at - 1];
                step[at] = step[at - 1];
            }
            n[at] = sizes[i];
            step[at] = (wide)strides[i] * es;
        }
        while (dims > 0 && step[0] == run) {  // one run after the other
            run *= n[0];
            drop(0);
        }
        for (int i = 1; i < dims;) {  // one row of runs after the other
            if (step[i] != step[i - 1] * n[i - 1]) {
                ++i;
                continue;
            }
            n[i - 1] *= n[i];
            drop(i);
        }
    }
    bool same_as(const Strided& o) const {
        bool same = base == o.base && run == o.run && dims == o.dims;
        for (int i = 0; same && i < dims; ++i) same = n[i] == o.n[i] && step[i] == o.step[i];
        return same;
    }

private:
    void drop(int i) {
        --dims;
        for (; i < dims; ++i) {
            n[i] = n[i + 1];
            step[i] = step[i + 1];
        }
    }
};

// True where a byte of a is shown to be one of b.  What lies apart is known at once; where the two are interleaved,
// the distance of any two runs is b.base - a.base + sum of d_k step_k for whole d_k in a range each: the longest
// range is solved, the others are tried, up to 4096 of them (rows of one buffer leave none to try, nor do heads in turn).
inline bool share_memory(const Strided& a, const Strided& b) {
    typedef Strided::wide wide;
    wide a_end = a.base + a.run, b_end = b.base + b.run;
    for (int i = 0; i < a.dims; ++i) a_end += a.step[i] * (a.n[i] - 1);
    for (int i = 0; i < b.dims; ++i) b_end += b.step[i] * (b.n[i] - 1);
    if (a.base >= b_end || b.base >= a_end) return false;
    wide step[7] = {1}, lo[7] = {0}, hi[7] = {0}, tried[7] = {0};  // the first: none, where there is no other
    int dims = 1;
    for (int i = 0; i < a.dims; ++i, ++dims) {
        step[dims] = a.step[i];
        lo[dims] = -(a.n[i] - 1);
        hi[dims] = 0;
    }
    for (int i = 0; i < b.dims; ++i) {
        int at = 1;
        while (at < dims && step[at] != b.step[i]) ++at;
        if (at == dims) {
            step[dims] = b.step[i];
            lo[dims] = hi[dims] = 0;
            ++dims;
        }
        hi[at] += b.n[i] - 1;
    }
    auto floor_div = [](wide x, wide y) { return x / y - (x % y < 0); };
    // Whether a distance within (-b.run, a.run) is base + a multiple of `by` that lies in [lo, hi].
    auto meets = [&](wide base, wide by, wide lo, wide hi) {
        const wide first = floor_div(-b.run - base, by) + 1, last = floor_div(a.run - 1 - base, by);
        return (first < lo ? lo : first) <= (last > hi ? hi : last);
    };
    // Any distance is a multiple of the steps' common divisor from the bases' one: heads in turn are apart by that alone.
    wide common = 0;
    for (int i = 1; i < dims; ++i)
        for (wide x = step[i]; x;) {
            const wide y = common % x;
            common = x;
            x = y;
        }
    const wide any = (wide)1 << 100;
    if (common && !meets(b.base - a.base, common, -any, any)) return false;
    int most = 0;
    for (int i = 0; i < dims; ++i)
        if (step[i] > 0 && hi[i] - lo[i] > hi[most] - lo[most]) most = i;
    // 0, 1, -1, 2, -2 .. until one side is done, then the rest of the other: runs of like indices meet soonest.
    auto d_of = [&](int i) {
        const wide c = tried[i], both = -lo[i] < hi[i] ? -lo[i] : hi[i];
        if (c <= 2 * both) return c % 2 ? (c + 1) / 2 : -(c / 2);
        return hi[i] > -lo[i] ? c - both : both - c;
    };
    for (int tries = 0; tries < 4096; ++tries) {
        wide x = b.base - a.base;
        for (int i = 0; i < dims; ++i) x += i == most ? 0 : d_of(i) * step[i];
        if (meets(x, step[most], lo[most], hi[most])) return true;
        int i = 0;
        for (; i < dims; ++i) {
            if (i == most) continue;
            if (++tried[i] <= hi[i] - lo[i]) break;
            tried[i] = 0;
        }
        if (i == dims) return false;
    }
    return false;
}

}  // namespace dit
