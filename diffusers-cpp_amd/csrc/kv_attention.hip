// kv_attention.hip -- attention of new tokens to a paged cache (kv_cache.hpp):
//   o_i = sum_j softmax_j(scale <q_i, k_j>) v_j over the places j that row i sees.
//
// Few rows a sequence: the cache is a stream, and each wave takes an equal part of it.  The
// units of that stream, in order, are the steps of 4 KPL keys of every (sequence, block of 16
// rows); wave w of W takes units [total w / W, total (w + 1) / W), whatever sequences they
// belong to, so unequal lengths leave no wave idle and nothing is laid out for the longest.
// A block of rows that one wave takes whole is finished there; the others' partial results (at
// most two a wave) are joined by a second launch, in the waves' order.
//
// The products are taken transposed on v_mfma_f32_16x16x32_bf16, S^T = K Q^T and O^T += V^T
// P^T: lane l holds row l % 16 of the block in both, its accumulators rows 4 (l / 16) + i.  Which
// key an operand row stands for is free, so both operands come straight from memory, 16 bytes
// a lane, no LDS: lane group g = l / 16 takes 16 bytes = KPL keys of a value's row (keys KPL g +
// 8 m + e feed product m), and the row r of score tile (m, h) is key KPL (r / 4) + 8 m + 4 h + r % 4,
// which leaves every lane with the scores of exactly those keys.
#include <float.h>
#include <math.h>

#include <type_traits>

#include "kv_cache.hpp"

namespace dit {
namespace kv {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kRows = 16;      // rows of a block

struct Args {
    Cache c;
    Seqs s;
    const uint16_t* q;
    uint16_t* o;
    int64_t qs[2], os[2];  // row, head strides
    int32_t heads, group, causal;
    FastDiv group_div;
    float scale_log2;
    int32_t waves;        // a key head
    float* part_o;        // [kv_heads][waves][2][kRows][DP], unnormalised
    float* part_ml;       // [kv_heads][waves][2][kRows][2]: reference (log2), sum
};

// Units of sequence b, this lane's; 0 past the last sequence.
template <int STEP>
__device__ __forceinline__ int64_t units_of(const Args& a, int b, int* tiles = nullptr) {
    if (b >= a.s.seqs) return 0;
    const Seq q(a.s, b);
    if (q.n == 0) return 0;
    const int t = max((q.len + STEP - 1) / STEP, 1);
    if (tiles) *tiles = t;
    return (int64_t)((q.n * (int64_t)a.group + kRows - 1) / kRows) * t;
}

__device__ __forceinline__ int64_t scan64(int64_t v) {  // inclusive sum over the wave's lanes
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t x = __shfl_up(v, o, 64);
        if (lane >= o) v += x;
    }
    return v;
}

template <int STEP>
__device__ __forceinline__ int64_t total_units(const Args& a) {
    const int lane = threadIdx.x & 63;
    int64_t n = 0;
    for (int b0 = 0; b0 < a.s.seqs; b0 += 64) n += units_of<STEP>(a, b0 + lane);
    return __shfl(scan64(n), 63, 64);
}

// The sequence that unit x (below the total) belongs to, and the units before it.
template <int STEP>
__device__ __forceinline__ int find_unit(const Args& a, int64_t x, int64_t* before) {
    const int lane = threadIdx.x & 63;
    int64_t sum = 0;
    for (int b0 = 0; b0 < a.s.seqs; b0 += 64) {
        const int64_t u = units_of<STEP>(a, b0 + lane), end = sum + scan64(u);
        const uint64_t past = __builtin_amdgcn_ballot_w64(end > x);
        if (past) {
            const int at = __builtin_ctzll(past);
            *before = __shfl(end - u, at, 64);
            return b0 + at;
        }
        sum = __shfl(end, 63, 64);
    }
    *before = sum;
    return -1;
}

// How many of the W waves work: two steps each at least.
__device__ __forceinline__ int64_t working(const Args& a, int64_t total) {
    const int64_t most = (total + 1) / 2;
    return most < a.waves ? most : a.waves;
}

__device__ __forceinline__ float xor_max(float v) {  // over the lane groups
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float xor_sum(float v) {
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

// 16 bytes of the cache as bf16 operands of 8.
template <typename E> struct Held;
template <> struct Held<e4m3> {
    static constexpr int N = 2;
    // Codes times the power of two are exact in bf16.
    __device__ __forceinline__ static void get(const uint4& w, float scale, bf16x8_t (&f)[2]) {
        const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bf16x2_t lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[i], scale, false);
            const bf16x2_t hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[i], scale, true);
            f[i / 2][4 * (i & 1)] = lo[0];
            f[i / 2][4 * (i & 1) + 1] = lo[1];
            f[i / 2][4 * (i & 1) + 2] = hi[0];
            f[i / 2][4 * (i & 1) + 3] = hi[1];
        }
    }
    // Bits of the elements that are not finite.
    __device__ __forceinline__ static uint32_t wild(uint32_t w) { return ((((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7) * 0xffu; }
    __device__ __forceinline__ static float value(const uint8_t* p) { return (*p & 0x7f) == 0x7f ? __builtin_nanf("") : 0.f; }
};
template <> struct Held<bf16> {
    static constexpr int N = 1;
    __device__ __forceinline__ static void get(const uint4& w, float, bf16x8_t (&f)[1]) { f[0] = __builtin_bit_cast(bf16x8_t, w); }
    __device__ __forceinline__ static uint32_t wild(uint32_t w) {
        return ((w & 0x7f80u) == 0x7f80u ? 0xffffu : 0u) | ((w & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u);
    }
    // A value that is not finite; 0 for any other.
    __device__ __forceinline__ static float value(const uint8_t* p) {
        const uint32_t w = *reinterpret_cast<const uint16_t*>(p);
        return (w & 0x7f80u) == 0x7f80u ? __uint_as_float(w << 16) : 0.f;
    }
};

// Of a 16-byte piece of N-byte elements, the first n.
template <int N>
__device__ __forceinline__ uint4 leading(uint4 w, int n) {
    uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int bits = 8 * N * n - 32 * i;
        x[i] = bits >= 32 ? x[i] : bits <= 0 ? 0u : x[i] & ((1u << bits) - 1);
    }
    return make_uint4(x[0], x[1], x[2], x[3]);
}

template <typename E, int DP>
__global__ __launch_bounds__(256, 2) void kv_stream_kernel(const Args a) {
    constexpr int ES = sizeof(E), KPL = 16 / ES, STEP = 4 * KPL, M = Held<E>::N;
    constexpr int KC = DP * ES / 64;  // 16-byte pieces of a key's row a lane group takes
    constexpr int DB = DP / 16;
    const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
    const int id = (int)(blockIdx.x * 4) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = id / a.waves, w = id - h * a.waves;
    if (h >= a.c.kv_heads) return;
    const int64_t total = total_units<STEP>(a);
    if (total == 0) return;
    const int64_t W = working(a, total);
    if (w >= W) return;
    const int64_t x1 = total * (w + 1) / W;
    const int dim = a.c.dim, lg = a.c.page_log2, pmask = (1 << lg) - 1;
    const int krow = dim * ES, vrow = ES << lg;

    for (int64_t x = total * w / W; x < x1;) {
        int64_t before;
        const int b = find_unit<STEP>(a, x, &before);
        if (b < 0) return;
        const Seq sq(a.s, b);
        const int tiles = max((sq.len + STEP - 1) / STEP, 1);
        const int blk = (int)((x - before) / tiles);
        const int64_t s0 = before + (int64_t)blk * tiles;
        const int t0 = (int)(x - s0), t1 = (int)((x1 < s0 + tiles ? x1 : s0 + tiles) - s0);

        const int row = blk * kRows + col, rows = sq.n * a.group;
        const bool live = row < rows;
        const int tok = live ? (int)fdiv((uint32_t)row, a.group_div) : 0;
        const int head = h * a.group + (live ? row - tok * a.group : 0);
        // The row sees places below this; rows past the last one all that the first row of the block sees.
        const int tok0 = (int)fdiv((uint32_t)(blk * kRows), a.group_div);
        const int limit = a.causal ? min(sq.past + (live ? tok : tok0) + 1, sq.len) : sq.len;
        const int all = a.causal ? min(sq.past + tok0 + 1, sq.len) : sq.len;  // places that every row sees

        bf16x8_t qf[KC][M];
        {
            const uint16_t* qp = a.q + (int64_t)(sq.row + tok) * a.qs[0] + head * a.qs[1];
#pragma unroll
            for (int c = 0; c < KC; ++c)
#pragma unroll
                for (int m = 0; m < M; ++m) {
                    const int d = KPL * (g + 4 * c) + 8 * m;
                    uint4 z = make_uint4(0, 0, 0, 0);
                    if (live && d < dim) z = *reinterpret_cast<const uint4*>(qp + d);
                    qf[c][m] = __builtin_bit_cast(bf16x8_t, z);
                }
        }
        float m = -INFINITY, l = 0.f;
        f32x4_t o[DB];
#pragma unroll
        for (int d = 0; d < DB; ++d) o[d] = f32x4_t{0.f, 0.f, 0.f, 0.f};

        for (int t = t0; t < t1; ++t) {
            // This lane's keys' (scores, values) and its operand row's pages.
            const int kb = t * STEP + KPL * (col >> 2), vb = t * STEP + KPL * g;
            int kp = kb < sq.len ? page_of(a.s, b, kb) : -1, vp = vb < sq.len ? page_of(a.s, b, vb) : -1;
            const bool paged = vp >= 0;
            kp = max(kp, 0);
            vp = max(vp, 0);
            const int64_t kh = (int64_t)kp * a.c.kv_heads + h, vh = (int64_t)vp * a.c.kv_heads + h;
            const uint8_t* ka = a.c.k + kh * a.c.head_bytes + ((kb & pmask) + (col & 3)) * (int64_t)krow + 16 * g;
            const uint8_t* va = a.c.v + vh * a.c.head_bytes + (vb & pmask) * ES;
            float ks = 1.f, vs = 1.f;
            if constexpr (ES == 1) {
                ks = __uint_as_float((uint32_t)max((int)a.c.k_scale[kh], 1) << 23);
                if (paged) vs = __uint_as_float((uint32_t)max((int)a.c.v_scale[vh], 1) << 23);  // any other page's may be NaN
            }
            uint4 kr[M][2][KC], vr[DB];
#pragma unroll
            for (int mm = 0; mm < M; ++mm)
#pragma unroll
                for (int hh = 0; hh < 2; ++hh)
#pragma unroll
                    for (int c = 0; c < KC; ++c) {
                        kr[mm][hh][c] = make_uint4(0, 0, 0, 0);
                        if (16 * (g + 4 * c) < krow)
                            kr[mm][hh][c] = *reinterpret_cast<const uint4*>(ka + (8 * mm + 4 * hh) * krow + 64 * c);
                    }
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                vr[d] = make_uint4(0, 0, 0, 0);
                if (16 * d < dim) vr[d] = *reinterpret_cast<const uint4*>(va + (16 * d + col) * vrow);
            }

            f32x4_t s[M][2];
#pragma unroll
            for (int mm = 0; mm < M; ++mm)
#pragma unroll
                for (int hh = 0; hh < 2; ++hh) {
                    s[mm][hh] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int c = 0; c < KC; ++c) {
                        bf16x8_t kf[M];
                        Held<E>::get(kr[mm][hh][c], ks, kf);
#pragma unroll
                        for (int j = 0; j < M; ++j) s[mm][hh] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[j], qf[c][j], s[mm][hh], 0, 0, 0);
                    }
                }
            // Key 8 mm + 4 hh + i of this lane's is seen below `sees`.
            const int sees = paged ? limit - vb : 0, holds = paged ? min(max(sq.len - vb, 0), KPL) : 0;
            if (__builtin_amdgcn_ballot_w64(sees < KPL)) {
#pragma unroll
                for (int mm = 0; mm < M; ++mm)
#pragma unroll
                    for (int hh = 0; hh < 2; ++hh)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (8 * mm + 4 * hh + i >= sees) s[mm][hh][i] = -INFINITY;
            }
            // What lies behind the sequence, or in no page, is anything: values of weight 0 have to be numbers.
            if (__builtin_amdgcn_ballot_w64(holds < KPL)) {
#pragma unroll
                for (int d = 0; d < DB; ++d) vr[d] = leading<ES>(vr[d], holds);
            }
            // So have those that only later rows of the block see; what is none is added to these rows below.
            bool wild = false;
            if ((t + 1) * STEP > all) {
                uint32_t any = 0;
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    const uint32_t wx = Held<E>::wild(vr[d].x), wy = Held<E>::wild(vr[d].y), wz = Held<E>::wild(vr[d].z), ww = Held<E>::wild(vr[d].w);
                    any |= wx | wy | wz | ww;
                    vr[d] = make_uint4(vr[d].x & ~wx, vr[d].y & ~wy, vr[d].z & ~wz, vr[d].w & ~ww);
                }
                wild = __builtin_amdgcn_ballot_w64(any != 0) != 0;
            }

            float mx = -INFINITY;
#pragma unroll
            for (int mm = 0; mm < M; ++mm)
#pragma unroll
                for (int hh = 0; hh < 2; ++hh)
#pragma unroll
                    for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[mm][hh][i]);
            mx = xor_max(mx) * a.scale_log2;
            // The reference moves when a score exceeds it by more than 2^8: every weight stays <= 256.
            const bool move = mx > m + 8.0f;
            if (__builtin_amdgcn_ballot_w64(move)) {
                const float to = move ? mx : m, alpha = move ? __builtin_amdgcn_exp2f(m - to) : 1.0f;
                l *= alpha;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[d][i] *= alpha;
                m = to;
            }
            const float ref = m == -INFINITY ? 0.f : m;
            bf16x8_t pf[M];
#pragma unroll
            for (int mm = 0; mm < M; ++mm) {
                float p[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[mm][e / 4][e & 3], a.scale_log2, -ref));
                    l += p[e];
                }
                // Rounded to bf16 for the product, after the sum took them as they are.
                pf[mm] = __builtin_bit_cast(bf16x8_t, make_uint4(pack_bf16x2(p[0], p[1]), pack_bf16x2(p[2], p[3]),
                                                                 pack_bf16x2(p[4], p[5]), pack_bf16x2(p[6], p[7])));
            }
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                bf16x8_t vf[M];
                Held<E>::get(vr[d], vs, vf);
#pragma unroll
                for (int mm = 0; mm < M; ++mm) o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[mm], pf[mm], o[d], 0, 0, 0);
            }
            if (wild) {
                for (int key = t * STEP; key < min((t + 1) * STEP, sq.len); ++key) {
                    const int p = page_of(a.s, b, key);
                    if (p < 0 || key >= limit) continue;
                    const uint8_t* at = a.c.v + ((int64_t)p * a.c.kv_heads + h) * a.c.head_bytes + (key & pmask) * ES;
#pragma unroll
                    for (int d = 0; d < DB; ++d)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (16 * d < dim) o[d][i] += Held<E>::value(at + (16 * d + 4 * g + i) * vrow);
                }
            }
        }

        l = xor_sum(l);
        if (t0 == 0 && t1 == tiles) {
            const float inv = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);  // no place seen: 0; NaN stays
            if (live) {
                uint16_t* op = a.o + (int64_t)(sq.row + tok) * a.os[0] + head * a.os[1];
#pragma unroll
                for (int d = 0; d < DB; ++d)
                    if (16 * d < dim)
                        *reinterpret_cast<uint2*>(op + 16 * d + 4 * g) =
                            make_uint2(pack_bf16x2(o[d][0] * inv, o[d][1] * inv), pack_bf16x2(o[d][2] * inv, o[d][3] * inv));
            }
        } else if (live) {
            const int64_t at = (((int64_t)h * a.waves + w) * 2 + (t0 == 0 ? 1 : 0)) * kRows + col;
#pragma unroll
            for (int d = 0; d < DB; ++d)
                *reinterpret_cast<float4*>(a.part_o + at * DP + 16 * d + 4 * g) = make_float4(o[d][0], o[d][1], o[d][2], o[d][3]);
            if (g == 0) {
                a.part_ml[2 * at] = m;
                a.part_ml[2 * at + 1] = l;
            }
        }
        x = s0 + t1;
    }
}

// The partial results of a row (token, head): TPR threads, each every PL-th wave's share of four elements.
template <typename E, int DP, int TPR>
__global__ __launch_bounds__(256) void kv_join_kernel(const Args a) {
    constexpr int STEP = 4 * (16 / (int)sizeof(E)), LPD = DP / 4, PL = TPR / LPD;
    __shared__ float part[256][6];
    const int tid = threadIdx.x, sub = tid % TPR, pl = sub / LPD, d0 = (sub % LPD) * 4;
    const int64_t id = (int64_t)blockIdx.x * (256 / TPR) + __builtin_amdgcn_readfirstlane(tid / TPR);
    const int r = (int)(id / a.heads), head = (int)(id - (int64_t)r * a.heads);
    float m = -INFINITY, l = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
    bool join = false;
    if (r < a.s.rows) {
        const int b = find_seq(a.s, r, [](int start, int) { return start; });
        const int64_t total = total_units<STEP>(a);
        if (b >= 0 && total > 0) {
            const Seq sq(a.s, b);
            // The units before sequence b.
            const int lane = tid & 63;
            int64_t n = 0;
            for (int b0 = 0; b0 < b; b0 += 64) n += b0 + lane < b ? units_of<STEP>(a, b0 + lane) : 0;
            n = __shfl(scan64(n), 63, 64);
            if (r - sq.row < sq.n) {
                const int h = head / a.group, row = (r - sq.row) * a.group + head - h * a.group;
                const int tiles = max((sq.len + STEP - 1) / STEP, 1);
                const int64_t s0 = n + (int64_t)(row / kRows) * tiles, W = working(a, total);
                const int w0 = (int)(((s0 + 1) * W - 1) / total), w1 = (int)(((s0 + tiles) * W - 1) / total);
                join = w0 != w1;
                if (join) {
                    for (int w = w0 + pl; w <= w1; w += PL) {
                        const int64_t at = (((int64_t)h * a.waves + w) * 2 + (w == w0 ? 1 : 0)) * kRows + row % kRows;
                        const float m1 = a.part_ml[2 * at], l1 = a.part_ml[2 * at + 1];
                        const float4 x = *reinterpret_cast<const float4*>(a.part_o + at * DP + d0);
                        const float to = fmaxf(m, m1), ref = to == -INFINITY ? 0.f : to;
                        const float f0 = __builtin_amdgcn_exp2f(m - ref), f1 = __builtin_amdgcn_exp2f(m1 - ref);
                        m = to;
                        l = l * f0 + l1 * f1;
                        v[0] = v[0] * f0 + x.x * f1;
                        v[1] = v[1] * f0 + x.y * f1;
                        v[2] = v[2] * f0 + x.z * f1;
                        v[3] = v[3] * f0 + x.w * f1;
                    }
                }
            }
        }
    }
    part[tid][0] = m;
    part[tid][1] = l;
#pragma unroll
    for (int e = 0; e < 4; ++e) part[tid][2 + e] = v[e];
    __syncthreads();
    if (!join || pl != 0) return;
    for (int i = 1; i < PL; ++i) m = fmaxf(m, part[tid + i * LPD][0]);
    const float ref = m == -INFINITY ? 0.f : m;
    l = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = 0.f;
    for (int i = 0; i < PL; ++i) {
        const float* p = part[tid + i * LPD];
        const float f = __builtin_amdgcn_exp2f(p[0] - ref);
        l += p[1] * f;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += p[2 + e] * f;
    }
    if (d0 >= a.c.dim) return;
    const float inv = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);
    *reinterpret_cast<uint2*>(a.o + (int64_t)r * a.os[0] + head * a.os[1] + d0) =
        make_uint2(pack_bf16x2(v[0] * inv, v[1] * inv), pack_bf16x2(v[2] * inv, v[3] * inv));
}

// ---- choice and launch --------------------------------------------------------------
struct Plan {
    int waves, dp;
    int64_t floats;
};

Plan plan(const Cache& c, int cus) {
    Plan p{};
    // Two waves a SIMD in all, whole workgroups of four a key head.
    p.waves = (8 * cus / c.kv_heads + 3) / 4 * 4;
    if (p.waves < 4) p.waves = 4;
    p.dp = c.dim <= 64 ? 64 : 128;
    p.floats = (int64_t)c.kv_heads * p.waves * 2 * kRows * (p.dp + 2);
    return p;
}

template <typename E, int DP>
int launch(const Args& a, hipStream_t st) {
    hipLaunchKernelGGL((kv_stream_kernel<E, DP>), dim3((unsigned)(a.c.kv_heads * (a.waves / 4))), dim3(256), 0, st, a);
    int rc = check_launch("dt_kv_attn");
    if (rc) return rc;
    const int64_t n = (int64_t)a.s.rows * a.heads;
    if (n <= 1024) {
        hipLaunchKernelGGL((kv_join_kernel<E, DP, 256>), dim3((unsigned)n), dim3(256), 0, st, a);
    } else {
        hipLaunchKernelGGL((kv_join_kernel<E, DP, 64>), dim3((unsigned)((n + 3) / 4)), dim3(256), 0, st, a);
    }
    return check_launch("dt_kv_attn");
}

}  // namespace
}  // namespace kv
}  // namespace dit

extern "C" size_t dt_kv_attn_workspace_bytes(const dt_kv_cache* cache, const dt_kv_seqs* seqs, int64_t heads) {
    using namespace dit;
    using namespace dit::kv;
    Cache c;
    Seqs s;
    if (prepare(cache, seqs, "dt_kv_attn_workspace_bytes", &c, &s)) return 0;
    if (s.rows == 0 || s.seqs == 0 || heads <= 0) return 0;
    return (size_t)plan(c, cu_count()).floats * sizeof(float);
}

extern "C" int dt_kv_attn(const dt_kv_cache* cache, const dt_kv_seqs* seqs, const void* q, const int64_t* q_strides, int64_t heads,
                          int32_t causal, float scale, void* o, const int64_t* o_strides, void* workspace, size_t workspace_bytes,
                          dt_stream_t stream) {
    using namespace dit;
    using namespace dit::kv;
    const char* who = "dt_kv_attn";
    Args a{};
    int rc = prepare(cache, seqs, who, &a.c, &a.s);
    if (rc) return rc;
    DT_REQUIRE(heads >= 0 && heads < (1 << 16) && heads % a.c.kv_heads == 0, "%s: %lld query heads do not share %d key heads evenly",
               who, (long long)heads, a.c.kv_heads);
    DT_REQUIRE(scale >= 0.f && scale < INFINITY, "%s: scale must be >= 0 and finite (got %g)", who, (double)scale);
    rc = check_rows(q, q_strides, a.s.rows, heads, a.c.dim, 2, false, "q", who);
    if (!rc) rc = check_rows(o, o_strides, a.s.rows, heads, a.c.dim, 2, true, "o", who);
    if (rc) return rc;
    if (a.s.rows == 0 || a.s.seqs == 0 || heads == 0) return DT_OK;
    DT_REQUIRE((int64_t)a.s.rows * heads < (1ll << 30), "%s: grid too large", who);
    const Plan p = plan(a.c, cu_count());
    DT_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= (size_t)p.floats * sizeof(float),
               "%s: a 16-byte aligned workspace of %lld bytes is needed", who, (long long)(p.floats * sizeof(float)));
    a.q = (const uint16_t*)q;
    a.o = (uint16_t*)o;
    for (int i = 0; i < 2; ++i) {
        a.qs[i] = q_strides[i];
        a.os[i] = o_strides[i];
    }
    a.heads = (int32_t)heads;
    a.group = (int32_t)(heads / a.c.kv_heads);
    a.group_div = make_fastdiv((uint32_t)a.group);
    a.causal = causal != 0;
    // A scale of 0 as the least normal number: -inf times it is still -inf, every finite score next to 0.
    a.scale_log2 = scale * kLog2e > FLT_MIN ? scale * kLog2e : FLT_MIN;
    a.waves = p.waves;
    a.part_o = (float*)workspace;
    a.part_ml = a.part_o + (int64_t)a.c.kv_heads * p.waves * 2 * kRows * p.dp;
    const hipStream_t st = (hipStream_t)stream;
    if (a.c.k_scale) return p.dp == 64 ? launch<e4m3, 64>(a, st) : launch<e4m3, 128>(a, st);
    return p.dp == 64 ? launch<bf16, 64>(a, st) : launch<bf16, 128>(a, st);
}
