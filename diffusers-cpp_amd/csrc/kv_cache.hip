// kv_cache.hip -- appending to a paged key/value cache: k rotated on the way, k and v rounded
// to e4m3 with a power of two for each page and head (or to bf16), q rotated beside them.
//
// A workgroup takes one page of one head of k or of v: a page's scale needs all of the page's
// new tokens, which fit its registers (16 elements a thread and pass).  They are read once; the
// largest size over the workgroup gives the scale; then codes go out, k's as they lie, v's
// turned over in LDS.
// q's rows (and nothing else of the call) need no page: a wave takes one token of them.
#include <float.h>
#include <math.h>

#include "kv_cache.hpp"
#include "overlap.hpp"
#include "rotary.hpp"

namespace dit {
namespace kv {
namespace {

struct Args {
    Cache c;
    Seqs s;
    const void* k;
    const void* v;
    const void* q;
    void* q_out;
    int64_t ks[2], vs[2], qs[2], os[2];
    int32_t heads;
    const int32_t* pos;
    const float* freq;
    float mul;
    int32_t rot, half;
    int32_t units, per_pass;         // 16-element units a row; tokens a pass of a workgroup
    FastDiv unit_div;
    int32_t q_units, slots;          // q: units of two vectors a row; heads side by side in a wave
    FastDiv q_unit_div;
    int32_t threads;                 // of a workgroup
    int32_t kv_blocks;               // workgroups before q's
    int32_t q_chunks;                // waves a row of q
    FastDiv head_div, chunk_div;
    int32_t quads_per_pass;          // v: fours of tokens a pass
    FastDiv quad_div;                // by the fours of dims of a row
    int32_t lds_row;                 // words a dim's row of v takes in LDS
};

constexpr int kScaleLow = 1;   // 2^-126
constexpr int kBias = 127;

// The least power of two, plus 127, by which 448 = 0.875 2^9 reaches m 2^x (m in [1/2, 1)).
__device__ __forceinline__ int scale_of(float most) {
    if (!(most > 0.f)) return kScaleLow;
    const int x = __builtin_amdgcn_frexp_expf(most);
    const float m = __builtin_amdgcn_frexp_mantf(most);
    return max(x - 9 + (m > 0.875f) + kBias, kScaleLow);
}

__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= FLT_MAX; }

// A 64-bit value as 32 bits rounded to odd: rounding that again to fewer bits gives what the value itself would.
__device__ __forceinline__ float to_odd(double d) {
    const float f = (float)d;
    if ((double)f == d || !finite(f)) return f;
    uint32_t u = __float_as_uint(f);
    if (fabs((double)f) > fabs(d)) --u;
    return __uint_as_float(u | 1u);
}

// A value that is not finite is held as NaN: the conversion would have the largest code for infinities.
__device__ __forceinline__ float tame(float x) { return finite(x) ? x : __builtin_nanf(""); }

__device__ __forceinline__ float power(int scale) { return __uint_as_float((uint32_t)scale << 23); }

// Codes times 2^-shift, rounded again.
__device__ __forceinline__ uint32_t again(uint32_t w, int shift) {
    float v[4];
    from_e4m3x4(w, v);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = __builtin_amdgcn_ldexpf(v[e], -shift);
    return to_e4m3x4(v[0], v[1], v[2], v[3], 1.f);
}

// The largest size of N values, and whether all are finite: sizes of others do not count, which a second look sees to.
struct Most {
    float top = 0.f, zero = 0.f;  // zero: 0 while all are finite, then NaN
    template <int N>
    __device__ __forceinline__ void take(const float (&v)[N]) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            top = fmaxf(top, fabsf(v[e]));
            zero = __builtin_fmaf(v[e], 0.f, zero);
        }
    }
    __device__ __forceinline__ bool tame() const { return zero == 0.f; }
    template <int N>
    __device__ __forceinline__ void take_finite(const float (&v)[N]) {
#pragma unroll
        for (int e = 0; e < N; ++e) top = fmaxf(top, finite(v[e]) ? fabsf(v[e]) : 0.f);
    }
};

template <typename T>
__device__ __forceinline__ void load8(const T* p, float* v) {
#pragma unroll
    for (int n = 0; n < 8 / Io<T>::EPV; ++n) Io<T>::load(p + n * Io<T>::EPV, v + n * Io<T>::EPV);
}

template <typename T>
__device__ void rotate_q(const Args& a) {
    const uint32_t wave = (blockIdx.x - a.kv_blocks) * (a.threads >> 6) + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int row = (int)fdiv(wave, a.chunk_div), chunk = (int)(wave - (uint32_t)row * a.q_chunks);
    if (row >= a.s.rows) return;
    const Found of = find_seq(a.s, row, [](int start, int) { return start; });
    if (of.b < 0) return;
    const Seq q = of.seq(a.s);
    if (row - q.row >= q.n) return;
    const int slot = (int)fdiv(lane, a.q_unit_div), u = (int)lane - slot * a.q_units;
    if (slot >= a.slots) return;
    const int p = a.pos ? a.pos[row] : q.past + row - q.row;
    const int first = chunk * 4 * a.slots + slot;
    rotary::turn_heads<T, 4>(
        p, a.freq, u, a.q_units, a.rot, a.half, a.mul, 1.f,
        [&](int i) { return first + i * a.slots < a.heads; },
        [&](int i) { return reinterpret_cast<const T*>(a.q) + row * a.qs[0] + (first + i * a.slots) * a.qs[1]; },
        [&](int i) { return reinterpret_cast<T*>(a.q_out) + row * a.os[0] + (first + i * a.slots) * a.os[1]; });
}

// The largest of the workgroup's `most`.
__device__ __forceinline__ float most_of_all(float most, float* of) {
#pragma unroll
    for (int o = 32; o; o >>= 1) most = fmaxf(most, __shfl_xor(most, o, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) of[threadIdx.x >> 6] = most;
    __syncthreads();
    most = of[0];
    for (uint32_t w = 1; w < blockDim.x >> 6; ++w) most = fmaxf(most, of[w]);
    return most;
}

template <typename E>
__device__ __forceinline__ uint4 stored8(const float (&x)[8], float scale) {
    if constexpr (sizeof(E) == 1) {
        return make_uint4(to_e4m3x4(x[0], x[1], x[2], x[3], scale), to_e4m3x4(x[4], x[5], x[6], x[7], scale), 0, 0);
    } else {
        return Io<bf16>::pack(x);
    }
}
template <typename E>
__device__ __forceinline__ void store8(uint8_t* y, uint4 w) {
    if constexpr (sizeof(E) == 1) *reinterpret_cast<uint2*>(y) = make_uint2(w.x, w.y);
    else *reinterpret_cast<uint4*>(y) = w;
}

// The scale of a page whose new values reach `most`, and by how much its earlier codes shrink.
__device__ __forceinline__ int page_scale(float most, int before, bool has_before, int* grown) {
    const int scale = scale_of(most);
    *grown = has_before && scale > before ? scale - before : 0;
    return has_before ? max(scale, before) : scale;
}

// k of one page and head.  Rotated in 32 bits, as values +- tol; only pairs of which an end is stored as another
// code than the other end (one of ten thousand with e4m3) are rotated in 64 bits after all, and so is the page
// where its scale is in doubt: what is stored is always the value's own rounding.
template <typename T, typename E, int NP>
__device__ __forceinline__ void append_k(const Args& a, const PageItem& it, int row0, int page, int h, float* of) {
    constexpr bool F8 = sizeof(E) == 1;
    const int tid = threadIdx.x, dim = a.c.dim, first = it.first, last = it.last;
    const int t0 = (int)fdiv((uint32_t)tid, a.unit_div), u = tid - t0 * a.units;
    const rotary::Unit<8> at(u, a.rot, a.half);
    const T* src = reinterpret_cast<const T*>(a.k) + h * a.ks[1];
    const bool turned = 16 * u < a.rot, mine = t0 < a.per_pass;
    auto place = [&](int t) { return a.pos ? a.pos[row0 + t] : it.begin + t; };
    auto load = [&](int t, float (&v)[16]) {
        const T* x = src + (int64_t)(row0 + t) * a.ks[0];
        load8(x + at.a, v);
        load8(x + at.b, v + 8);
    };
    // Pair e of the unit in 64 bits, rounded to odd, and where its ends lie in the row.
    auto exact = [&](int t, int e, float (&w)[2], int (&d)[2]) {
        const T* x = src + (int64_t)(row0 + t) * a.ks[0];
        d[0] = at.a + (a.half ? e : 2 * e);
        d[1] = a.half ? at.b + e : d[0] + 1;
        w[0] = Io<T>::get(x + d[0]);
        w[1] = Io<T>::get(x + d[1]);
        const int n = at.pair(e);
        if (2 * n >= a.rot) return;
        double c, s;
        rotary::cos_sin(place(t), a.freq[n], (double)a.mul, &c, &s);
        const double p = w[0], q = w[1];
        w[0] = to_odd(p * c - q * s);
        w[1] = to_odd(q * c + p * s);
    };
    rotary::Angles<float, 8> w(a.freq, at, a.rot);
    float v[NP][16];
    Most most;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int t = first + i * a.per_pass + t0;
        if (mine && t < last) load(t, v[i]);
    }
    if ((uint32_t)page >= (uint32_t)a.s.pages) return;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int t = first + i * a.per_pass + t0;
        if (!mine || t >= last) continue;
        if (turned) {
            w.set(place(t), a.mul);
            w.turn(v[i], a.half, 1.f);
        }
        if constexpr (F8) most.take(v[i]);
    }

    uint8_t* const out = a.c.k + ((int64_t)page * a.c.kv_heads + h) * a.c.head_bytes;
    int scale = kBias, grown = 0;
    if constexpr (F8) {
        uint8_t* const held = a.c.k_scale + (int64_t)page * a.c.kv_heads + h;
        const int before = first ? (int)*held : 0;
        const bool tamed = __syncthreads_and(most.tame());
        float top = most_of_all(most.top, of);
        if (!tamed || scale_of(top * (1.f - 0x1p-19f)) != scale_of(top * (1.f + 0x1p-19f))) {
            Most again;
#pragma unroll 1
            for (int t = first + t0; mine && t < last; t += a.per_pass) {
#pragma unroll 1
                for (int e = 0; e < 8; ++e) {
                    float w[2];
                    int d[2];
                    exact(t, e, w, d);
                    again.take_finite(w);
                }
            }
            top = most_of_all(again.top, of);
#pragma unroll
            for (int i = 0; i < NP; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) v[i][e] = tame(v[i][e]);
        }
        scale = page_scale(top, before, first > 0, &grown);
        if (tid == 0) *held = (uint8_t)scale;  // read by all before the barriers
        if (grown)
            for (int i = tid; i < first * dim / 16; i += a.threads) {
                uint4 w = *reinterpret_cast<const uint4*>(out + 16 * i);
                w.x = again(w.x, grown);
                w.y = again(w.y, grown);
                w.z = again(w.z, grown);
                w.w = again(w.w, grown);
                *reinterpret_cast<uint4*>(out + 16 * i) = w;
            }
    }
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int t = first + i * a.per_pass + t0;
        if (!mine || t >= last) continue;
        // A rotation by mul keeps a pair's length l but for mul: mul (|x| + |y|) <= sqrt(2) mul l <= sqrt(2) (|x'| + |y'|).  Cosine
        // and sine are off by 2^-23 of mul, the products and their sum by two roundings of 2^-24 more: 4 2^-24 mul (|x| + |y|)
        // in all, 1.42 2^-22 (|x'| + |y'|) of the 2 2^-22 that are taken.
        float tol[8], all = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float x = a.half ? v[i][e] : v[i][2 * e], y = a.half ? v[i][8 + e] : v[i][2 * e + 1];
            tol[e] = 2 * (8 * u + e) < a.rot ? (fabsf(x) + fabsf(y)) * 0x1p-21f : 0.f;
            all += tol[e];
        }
        // A pair with an end that 32 bits could not hold (the 64 may, and its other end is held like any).
        uint32_t pairs = 0;
        if (!finite(all)) {
#pragma unroll
            for (int e = 0; e < 8; ++e) pairs |= finite(tol[e]) ? 0u : 1u << e;
        }
        uint4 differ[2];
#pragma unroll
        for (int run = 0; run < 2; ++run) {
            float lo[8], hi[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float d = tol[a.half ? e : 4 * run + e / 2];
                lo[e] = v[i][8 * run + e] - d;
                hi[e] = v[i][8 * run + e] + d;
            }
            const uint4 p = stored8<E>(lo, power(scale)), q = stored8<E>(hi, power(scale));
            store8<E>(out + ((int64_t)t * dim + (run ? at.b : at.a)) * sizeof(E), p);
            differ[run] = make_uint4(p.x ^ q.x, p.y ^ q.y, p.z ^ q.z, p.w ^ q.w);
        }
        if (!turned || !(pairs | differ[0].x | differ[0].y | differ[0].z | differ[0].w | differ[1].x | differ[1].y | differ[1].z | differ[1].w)) continue;
#pragma unroll
        for (int run = 0; run < 2; ++run)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int per = 4 / (int)sizeof(E);
                const uint32_t w[4] = {differ[run].x, differ[run].y, differ[run].z, differ[run].w};
                if (w[e / per] << (32 - 8 * (int)sizeof(E) * (e % per + 1)) >> (32 - 8 * (int)sizeof(E))) pairs |= 1u << (a.half ? e : 4 * run + e / 2);
            }
#pragma unroll 1
        for (; pairs; pairs &= pairs - 1) {
            float w[2];
            int d[2];
            exact(t, __builtin_ctz(pairs), w, d);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                uint8_t* y = out + ((int64_t)t * dim + d[k]) * sizeof(E);
                if constexpr (F8) *y = (uint8_t)to_e4m3x4(tame(w[k]), 0.f, 0.f, 0.f, power(scale));
                else Io<bf16>::put(reinterpret_cast<bf16*>(y), w[k]);
            }
        }
    }
}

// v of one page and head: a thread takes four tokens by four dims, so that a dim's four codes are a word of its
// row in LDS, from where whole 16-byte pieces of rows go out.
template <typename T, typename E, int NP>
__device__ __forceinline__ void append_v(const Args& a, const PageItem& it, int row0, int in_page, int h, float* of, uint32_t* turned) {
    constexpr bool F8 = sizeof(E) == 1;
    constexpr int WPT = sizeof(E);  // words of four tokens
    const int tid = threadIdx.x, dim = a.c.dim, page = 1 << a.c.page_log2, first = it.first, last = it.last;
    const int g0 = (int)fdiv((uint32_t)tid, a.quad_div), d0 = 4 * (tid - g0 * (dim / 4));
    const T* src = reinterpret_cast<const T*>(a.v) + h * a.vs[1] + d0;
    const bool mine = g0 < a.quads_per_pass;
    const int start = first & ~3;  // tokens in fours, as they lie in the page
    float v[NP][4][4];
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int t = start + 4 * (i * a.quads_per_pass + g0) + k;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[i][k][e] = 0.f;
            if (!mine || t < first || t >= last) continue;
            const T* x = src + (int64_t)(row0 + t) * a.vs[0];
            if constexpr (sizeof(T) == 4) {
                const float4 w = *reinterpret_cast<const float4*>(x);
                v[i][k][0] = w.x;
                v[i][k][1] = w.y;
                v[i][k][2] = w.z;
                v[i][k][3] = w.w;
            } else {
                const uint2 w = *reinterpret_cast<const uint2*>(x);
                v[i][k][0] = bf16_lo(w.x);
                v[i][k][1] = bf16_hi(w.x);
                v[i][k][2] = bf16_lo(w.y);
                v[i][k][3] = bf16_hi(w.y);
            }
        }
    if ((uint32_t)in_page >= (uint32_t)a.s.pages) return;
    uint8_t* const out = a.c.v + ((int64_t)in_page * a.c.kv_heads + h) * a.c.head_bytes;
    int scale = kBias, grown = 0;
    if constexpr (F8) {
        Most most;
#pragma unroll
        for (int i = 0; i < NP; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) most.take(v[i][k]);
        if (!__syncthreads_and(most.tame())) {
            most.top = 0.f;
#pragma unroll
            for (int i = 0; i < NP; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    most.take_finite(v[i][k]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[i][k][e] = tame(v[i][k][e]);
                }
        }
        uint8_t* const held = a.c.v_scale + (int64_t)in_page * a.c.kv_heads + h;
        const int before = first ? (int)*held : 0;
        scale = page_scale(most_of_all(most.top, of), before, first > 0, &grown);
        if (tid == 0) *held = (uint8_t)scale;  // read by all before the barriers
    }
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int t = start + 4 * (i * a.quads_per_pass + g0);
        if (!mine || t >= last) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            uint32_t* w = turned + (d0 + e) * a.lds_row + t / 4 * WPT;
            if constexpr (F8) {
                w[0] = to_e4m3x4(v[i][0][e], v[i][1][e], v[i][2][e], v[i][3][e], power(scale));
            } else {
                w[0] = pack_bf16x2(v[i][0][e], v[i][1][e]);
                w[1] = pack_bf16x2(v[i][2][e], v[i][3][e]);
            }
        }
    }
    __syncthreads();
    constexpr int PER = 16 / sizeof(E);  // tokens of a piece
    const int pieces = page / PER;       // of a row: a power of two
    for (int i = tid; i < dim * pieces; i += a.threads) {
        const int d = i / pieces, c = (i & (pieces - 1)) * PER;
        if (c >= last || (c + PER <= first && !grown)) continue;
        uint8_t* y = out + ((int64_t)d * page + c) * sizeof(E);
        const uint32_t* x = turned + d * a.lds_row + c * (int)sizeof(E) / 4;
        if (c >= first && c + PER <= last) {
            *reinterpret_cast<uint4*>(y) = make_uint4(x[0], x[1], x[2], x[3]);
            continue;
        }
        if constexpr (F8) {
            if (grown && c < first) {
                // Earlier tokens of the piece again; those that are not this call's stay.
                for (int n = 0; n < 4; ++n) {
                    if (c + 4 * n >= first) break;
                    const uint32_t w = reinterpret_cast<const uint32_t*>(y)[n], s = again(w, grown);
                    const int left = first - c - 4 * n;
                    const uint32_t m = left >= 4 ? ~0u : (1u << (8 * left)) - 1;
                    reinterpret_cast<uint32_t*>(y)[n] = (s & m) | (w & ~m);
                }
            }
        }
        for (int n = max(first - c, 0); n < min(last - c, PER); ++n) reinterpret_cast<E*>(y)[n] = reinterpret_cast<const E*>(x)[n];
    }
}

// NP passes hold a page.  Registers for five workgroups a CU where two passes do: 8750 tokens of 32 + 8 heads of 128
// 45 us, 46 with four, 51 with six.
template <typename T, typename E, int NP>
__global__ __launch_bounds__(256, NP <= 2 ? 5 : 2) void kv_append_kernel(const Args a) {
    extern __shared__ __attribute__((aligned(16))) uint32_t turned[];  // v: [dim][lds_row] words
    __shared__ float most_of[4];
    if ((int)blockIdx.x >= a.kv_blocks) {
        rotate_q<T>(a);
        return;
    }
    // Workgroup: (number of a page, head, k or v), heads innermost: they share rows.
    const int item = (int)fdiv(blockIdx.x >> 1, a.head_div), h = (int)(blockIdx.x >> 1) - item * a.c.kv_heads;
    const Found of = find_seq(a.s, item, [&a](int start, int i) { return first_item(a.s, start, i); });
    if (of.b < 0) return;
    const Seq q = of.seq(a.s);
    PageItem it;
    if (!page_item(a.s, q, of.b, item, &it)) return;
    const int row0 = q.row + it.begin - q.past;  // of the page's token 0 (there may be none)
    // The page's number is looked at when the tokens are on their way.
    const int page = a.s.table[of.b * a.s.table_stride + (it.begin >> a.s.page_log2)];
    if (blockIdx.x & 1) append_v<T, E, NP>(a, it, row0, page, h, most_of, turned);
    else append_k<T, E, NP>(a, it, row0, page, h, most_of);
}

template <typename T, typename E>
int launch(const Args& a, int passes, dim3 grid, hipStream_t st) {
    const size_t lds = (size_t)a.c.dim * a.lds_row * sizeof(uint32_t);
    if (passes <= 1) hipLaunchKernelGGL((kv_append_kernel<T, E, 1>), grid, dim3(a.threads), lds, st, a);
    else if (passes <= 2) hipLaunchKernelGGL((kv_append_kernel<T, E, 2>), grid, dim3(a.threads), lds, st, a);
    else if (passes <= 4) hipLaunchKernelGGL((kv_append_kernel<T, E, 4>), grid, dim3(a.threads), lds, st, a);
    else hipLaunchKernelGGL((kv_append_kernel<T, E, 8>), grid, dim3(a.threads), lds, st, a);
    return check_launch("dt_kv_append");
}

}  // namespace

int check_rows(const void* p, const int64_t* s, int64_t rows, int64_t heads, int64_t dim, int es, bool out, const char* name,
               const char* who) {
    if (rows == 0 || heads == 0) return DT_OK;
    DT_REQUIRE(p != nullptr && s != nullptr, "%s: null %s", who, name);
    DT_REQUIRE(aligned16(p), "%s: %s must be 16-byte aligned", who, name);
    const int64_t n[2] = {rows, heads};
    for (int i = 0; i < 2; ++i) {
        if (n[i] == 1) continue;
        DT_REQUIRE(s[i] * es % 16 == 0, "%s: %s strides must keep rows 16-byte aligned", who, name);
        DT_REQUIRE(s[i] >= 0 && s[i] < (1ll << 40), "%s: %s stride %lld unsupported", who, name, (long long)s[i]);
    }
    if (!out) return DT_OK;
    const int in = n[0] > 1 && (n[1] == 1 || s[0] < s[1]) ? 0 : 1;  // the closer dimension
    int64_t reach = dim;
    for (int i = 0; i < 2; ++i) {
        const int at = i ? 1 - in : in;
        if (n[at] == 1) continue;
        DT_REQUIRE(s[at] >= reach, "%s: elements of %s overlap", who, name);
        reach = s[at] * (n[at] - 1) + reach;
    }
    return DT_OK;
}

int prepare(const dt_kv_cache* x, const dt_kv_seqs* y, const char* who, Cache* c, Seqs* s) {
    DT_REQUIRE(x != nullptr && y != nullptr, "%s: null arguments", who);
    DT_REQUIRE(x->type == DT_TYPE_BF16 || x->type == DT_TYPE_F8_E4M3, "%s: cache type %d unsupported", who, x->type);
    DT_REQUIRE(x->head_dim > 0 && x->head_dim <= 128 && x->head_dim % 16 == 0,
               "%s: head_dim %lld unsupported (a multiple of 16 up to 128)", who, (long long)x->head_dim);
    DT_REQUIRE(x->page >= 16 && x->page <= 256 && (x->page & (x->page - 1)) == 0,
               "%s: pages of %lld tokens unsupported (16, 32, 64, 128 or 256)", who, (long long)x->page);
    DT_REQUIRE(x->pages > 0 && x->kv_heads > 0 && x->kv_heads < (1 << 16) && x->pages < (1ll << 31) / x->kv_heads,
               "%s: %lld pages of %lld heads unsupported", who, (long long)x->pages, (long long)x->kv_heads);
    DT_REQUIRE(x->k && x->v && aligned16(x->k) && aligned16(x->v), "%s: k and v must be given, 16-byte aligned", who);
    const bool f8 = x->type == DT_TYPE_F8_E4M3;
    DT_REQUIRE(!f8 || (x->k_scale && x->v_scale), "%s: an e4m3 cache needs k_scale and v_scale", who);
    DT_REQUIRE(y->seqs >= 0 && y->seqs < (1 << 20) && y->rows >= 0 && y->rows < (1 << 28), "%s: size out of range", who);
    DT_REQUIRE(y->table_pages >= 0 && y->table_pages <= (1ll << 30) / x->page, "%s: a table of %lld pages is too long", who,
               (long long)y->table_pages);
    if (y->seqs > 0 && y->rows > 0) {
        DT_REQUIRE(y->seq_start && y->past && ((uintptr_t)y->seq_start & 3) == 0 && ((uintptr_t)y->past & 3) == 0,
                   "%s: seq_start and past must be given, 4-byte aligned", who);
        DT_REQUIRE(y->table_pages == 0 || (y->table && ((uintptr_t)y->table & 3) == 0), "%s: table must be given, 4-byte aligned", who);
        DT_REQUIRE(y->seqs == 1 || (y->table_stride >= 0 && y->table_stride < (1ll << 40)), "%s: table_stride unsupported", who);
    }
    int lg = 0;
    while ((1 << lg) < x->page) ++lg;
    c->k = (uint8_t*)x->k;
    c->v = (uint8_t*)x->v;
    c->k_scale = f8 ? x->k_scale : nullptr;
    c->v_scale = f8 ? x->v_scale : nullptr;
    c->kv_heads = (int32_t)x->kv_heads;
    c->page_log2 = lg;
    c->dim = (int32_t)x->head_dim;
    c->head_bytes = x->page * x->head_dim * (f8 ? 1 : 2);
    s->table = y->table;
    s->table_stride = y->seqs == 1 ? 0 : y->table_stride;
    s->seq_start = y->seq_start;
    s->past = y->past;
    s->table_pages = (int32_t)y->table_pages;
    s->seqs = (int32_t)y->seqs;
    s->rows = (int32_t)y->rows;
    s->pages = (int32_t)x->pages;
    s->page_log2 = lg;
    return DT_OK;
}

}  // namespace kv
}  // namespace dit

extern "C" int dt_kv_append(const dt_kv_cache* cache, const dt_kv_seqs* seqs, const dt_kv_append_args* x, dt_stream_t stream) {
    using namespace dit;
    using namespace dit::kv;
    const char* who = "dt_kv_append";
    Args a{};
    int rc = prepare(cache, seqs, who, &a.c, &a.s);
    if (rc) return rc;
    DT_REQUIRE(x != nullptr, "%s: null arguments", who);
    DT_REQUIRE(is_io_type(x->io_type), "%s: io_type %d unsupported", who, x->io_type);
    const int es = elem_size(x->io_type);
    rc = check_rows(x->k, x->k_strides, a.s.rows, a.c.kv_heads, a.c.dim, es, false, "k", who);
    if (!rc) rc = check_rows(x->v, x->v_strides, a.s.rows, a.c.kv_heads, a.c.dim, es, false, "v", who);
    if (rc) return rc;
    DT_REQUIRE(x->heads >= 0 && x->heads < (1 << 16), "%s: size out of range", who);
    const bool turn_q = x->q && x->heads > 0;
    if (turn_q) {
        DT_REQUIRE(x->rotary, "%s: q needs a rotation", who);
        rc = check_rows(x->q, x->q_strides, a.s.rows, x->heads, a.c.dim, es, false, "q", who);
        if (!rc) rc = check_rows(x->q_out, x->q_out_strides, a.s.rows, x->heads, a.c.dim, es, true, "q_out", who);
        if (rc) return rc;
    }
    a.mul = 1.f;
    a.freq = reinterpret_cast<const float*>(a.s.seq_start);
    if (x->rotary) {
        rc = rotary::check_rotary(*x->rotary, a.c.dim, who);
        if (rc) return rc;
        DT_REQUIRE(!x->rotary->half || x->rotary->rot_dims % 16 == 0, "%s: halves of %lld dims unsupported (a multiple of 16)", who,
                   (long long)x->rotary->rot_dims);
        if (x->rotary->rot_dims) a.freq = x->rotary->freq;
        a.mul = x->rotary->attn_factor;
        a.rot = (int32_t)x->rotary->rot_dims;
        a.half = x->rotary->half != 0;
    }
    DT_REQUIRE(((uintptr_t)x->pos & 3) == 0, "%s: pos must be 4-byte aligned", who);
    if (a.s.rows == 0 || a.s.seqs == 0) return DT_OK;
    if (turn_q) {
        const int64_t q_sizes[2] = {a.s.rows, x->heads}, sizes[2] = {a.s.rows, a.c.kv_heads};
        const Strided q(x->q, es, 2, q_sizes, x->q_strides, a.c.dim), out(x->q_out, es, 2, q_sizes, x->q_out_strides, a.c.dim);
        DT_REQUIRE(out.same_as(q) || !share_memory(out, q), "%s: q_out is partly q", who);
        DT_REQUIRE(!share_memory(out, Strided(x->k, es, 2, sizes, x->k_strides, a.c.dim)), "%s: q_out is partly k", who);
        DT_REQUIRE(!share_memory(out, Strided(x->v, es, 2, sizes, x->v_strides, a.c.dim)), "%s: q_out is partly v", who);
    }
    a.k = x->k;
    a.v = x->v;
    a.q = x->q;
    a.q_out = x->q_out;
    for (int i = 0; i < 2; ++i) {
        a.ks[i] = x->k_strides[i];
        a.vs[i] = x->v_strides[i];
        a.qs[i] = x->q_strides[i];
        a.os[i] = x->q_out_strides[i];
    }
    a.heads = (int32_t)x->heads;
    a.pos = x->pos;
    a.units = a.c.dim / 16;
    a.q_units = a.c.dim * es / 32;
    a.slots = 64 / a.q_units;
    a.q_unit_div = make_fastdiv((uint32_t)a.q_units);
    a.unit_div = make_fastdiv((uint32_t)a.units);
    a.head_div = make_fastdiv((uint32_t)a.c.kv_heads);
    a.q_chunks = turn_q ? (a.heads + 4 * a.slots - 1) / (4 * a.slots) : 1;
    a.chunk_div = make_fastdiv((uint32_t)a.q_chunks);
    const int64_t page = 1ll << a.c.page_log2;
    const bool f8 = a.c.k_scale != nullptr;
    // An odd number of words: dims lie in other banks.
    a.lds_row = (int32_t)page * (f8 ? 1 : 2) / 4 + 1;
    // Threads for a pass over a page, which takes up to 256: pages of 16 tokens leave the rest without work (3003 tokens
    // of 12 heads of 80, bf16: 25.5 us with 256, 19.9 with 128).
    const int most = (int)page * a.units;
    a.threads = most >= 256 ? 256 : (most + 63) / 64 * 64;
    a.per_pass = a.threads / a.units;
    a.quads_per_pass = a.threads / (a.c.dim / 4);
    a.quad_div = make_fastdiv((uint32_t)(a.c.dim / 4));
    const int64_t kv_blocks = items(a.s) * a.c.kv_heads * 2;
    const int64_t waves = a.threads / 64;
    const int64_t q_blocks = turn_q ? ((int64_t)a.s.rows * a.q_chunks + waves - 1) / waves : 0;
    DT_REQUIRE(grid_fits(kv_blocks + q_blocks, a.threads) && (int64_t)a.s.rows * a.q_chunks < (1ll << 31), "%s: grid too large", who);
    a.kv_blocks = (int32_t)kv_blocks;
    const dim3 grid((unsigned)(kv_blocks + q_blocks));
    const int k_passes = ((int)page + a.per_pass - 1) / a.per_pass, v_passes = ((int)page / 4 + a.quads_per_pass - 1) / a.quads_per_pass;
    const int passes = k_passes > v_passes ? k_passes : v_passes;
    const hipStream_t st = (hipStream_t)stream;
    if (x->io_type == DT_TYPE_F32)
        return f8 ? launch<float, e4m3>(a, passes, grid, st) : launch<float, bf16>(a, passes, grid, st);
    return f8 ? launch<bf16, e4m3>(a, passes, grid, st) : launch<bf16, bf16>(a, passes, grid, st);
}
