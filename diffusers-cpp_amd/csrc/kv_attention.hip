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

#include "attn_tiles.hpp"
#include "kv_cache.hpp"
#include "overlap.hpp"

namespace dit {
namespace kv {
namespace {

using attn::bf16x8_t;
using attn::f32x16_t;
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr int kRows = 16;      // rows of a block of the stream's
constexpr int kShort = 1 << 18;  // bytes of a key head's keys up to which the stream's blocks of rows are not shared out
// Beside the row blocks' kernel the stream takes sequences of up to so many rows (20 sequences of 48 rows behind 4000, 32 on
// 8 heads of 128: 56 us, with 64 88; 9 of 24 rows: 35, with 16 32, but of 48 rows 36).  Where all are such sequences there is
// nothing to run beside, and the stream's share of the CUs is too small (32 of 1, 2, 4 and 8 tokens behind 8000, e4m3: 66, 103,
// 104 and 191 us): what the sequences' rows are is known on the device only.
constexpr int kFew = 32;

struct Args {
    Cache c;
    Seqs s;
    const uint16_t* q;
    uint16_t* o;
    int64_t qs[2], os[2];  // row, head strides
    int32_t heads, group, causal;
    FastDiv group_div;
    float scale_log2;
    int32_t few;          // sequences of up to so many rows (new tokens times heads of a group) are the stream's
    int32_t splits;       // key ranges of the others' row blocks
    int32_t waves;        // the stream's, a key head
    int32_t stream_blocks;  // workgroups of the row blocks' kernel that are the stream's
    int32_t join_blocks;    // workgroups of the join that are the stream's
    float* part_o;        // [kv_heads][waves][2][kRows][DP], unnormalised
    float* part_ml;       // [kv_heads][waves][2][kRows][2]: reference (log2), sum
    float* rows_o;        // [splits][rows][heads][DP], as part_o
    float* rows_ml;       // [splits][rows][heads][2]
};

__device__ __forceinline__ int64_t scan64(int64_t v) {  // inclusive sum over the wave's lanes
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t x = __shfl_up(v, o, 64);
        if (lane >= o) v += x;
    }
    return v;
}

// Blocks of rows are numbered like the pages that are written (kv_index.hpp).
template <int BLOCK>
__device__ __forceinline__ int64_t first_block(const Args& a, int start, int b) { return (int64_t)start * a.group / BLOCK + b; }

// One sequence, the same in all lanes.
struct Mine {
    int b, row, n, past, len;
    int64_t before;  // units before it
};

__device__ __forceinline__ int64_t lane64(int64_t v, int l) {
    return (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), l) << 32) | (uint32_t)__builtin_amdgcn_readlane((int)v, l));
}

// The stream's sequences in order, 64 at a time, one a lane.
template <int STEP>
struct Walk {
    const Args& a;
    int from, row, n, past, len;
    int64_t units, end;  // of this lane's, and of all up to it
    __device__ __forceinline__ explicit Walk(const Args& args) : a(args) {}
    __device__ __forceinline__ static int tiles(int len) { return max((len + STEP - 1) / STEP, 1); }
    __device__ __forceinline__ void load(int b0, int64_t before) {
        from = b0;
        const int b = b0 + (threadIdx.x & 63);
        row = n = past = len = 0;
        units = 0;
        if (b < a.s.seqs) {
            const Seq q(a.s, b);
            row = q.row;
            n = q.n;
            past = q.past;
            len = q.len;
            if (n > 0 && n * (int64_t)a.group <= a.few) units = (n * (int64_t)a.group + kRows - 1) / kRows * tiles(len);
        }
        end = before + scan64(units);
    }
    // All units; and the sequence of the lane that picked it, if one did (b = -1: none).
    template <typename Pick>
    __device__ __forceinline__ int64_t total(Pick pick, Mine* picked) {
        int64_t sum = 0;
        picked->b = -1;
        for (int b0 = 0; b0 < a.s.seqs; b0 += 64) {
            load(b0, sum);
            const uint64_t it = __builtin_amdgcn_ballot_w64(pick());
            if (it) *picked = mine(__builtin_ctzll(it));
            sum = lane64(end, 63);
        }
        return sum;
    }
    __device__ __forceinline__ int64_t total() {
        Mine none;
        return total([] { return false; }, &none);
    }
    __device__ __forceinline__ Mine mine(int l) const {
        return {from + l, __builtin_amdgcn_readlane(row, l), __builtin_amdgcn_readlane(n, l), __builtin_amdgcn_readlane(past, l),
                __builtin_amdgcn_readlane(len, l), lane64(end - units, l)};
    }
    // The sequence that unit x (below the total) belongs to.  b = -1: none, which lengths that are written
    // under the call may make of it.
    __device__ __forceinline__ Mine find(int64_t x) {
        if (x < lane64(end - units, 0)) load(0, 0);
        while (x >= lane64(end, 63) && from + 64 < a.s.seqs) load(from + 64, lane64(end, 63));
        const uint64_t behind = __builtin_amdgcn_ballot_w64(end > x);
        Mine m = mine(behind ? __builtin_ctzll(behind) : 0);
        if (!behind) m.b = -1;
        return m;
    }
};

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
    // Codes times the power of two are exact in bf16 for scales from 3 (the least code is 2^-9, bf16's least value
    // 2^-133) to 246 (the largest is 448, bf16's range below 2^128); past that the largest are infinite.
    __device__ __forceinline__ static bf16x8_t part(const uint4& w, float scale, int m) {
        const uint32_t x[2] = {m ? w.z : w.x, m ? w.w : w.y};
        bf16x8_t f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const bf16x2_t lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[i], scale, false);
            const bf16x2_t hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[i], scale, true);
            f[4 * i] = lo[0];
            f[4 * i + 1] = lo[1];
            f[4 * i + 2] = hi[0];
            f[4 * i + 3] = hi[1];
        }
        return f;
    }
    // What takes the codes that are not finite to bit 7, in each byte: those from 2^(255 - scale) on, which is 8 (262 - scale), are
    // infinite; NaN is 0x7f.
    __device__ __forceinline__ static uint32_t past(uint32_t scale) { return 0x01010101u * (scale > 246 ? 128 - 8 * (262 - scale) : 1u); }
    // Bits of the elements that are not finite.
    __device__ __forceinline__ static uint32_t wild(uint32_t w, uint32_t past) { return ((((w & 0x7f7f7f7fu) + past) & 0x80808080u) >> 7) * 0xffu; }
    // A value that is not finite; 0 for any other.
    __device__ __forceinline__ static float value(const uint8_t* p, const uint8_t* scale) {
        const uint32_t w = *p;
        if (!wild(w, past(*scale))) return 0.f;
        return (w & 0x7fu) == 0x7fu ? __builtin_nanf("") : w & 0x80u ? -INFINITY : INFINITY;
    }
};
template <> struct Held<bf16> {
    static constexpr int N = 1;
    __device__ __forceinline__ static bf16x8_t part(const uint4& w, float, int) { return __builtin_bit_cast(bf16x8_t, w); }
    __device__ __forceinline__ static uint32_t past(uint32_t) { return 0; }
    __device__ __forceinline__ static uint32_t wild(uint32_t w, uint32_t) {
        return ((w & 0x7f80u) == 0x7f80u ? 0xffffu : 0u) | ((w & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u);
    }
    __device__ __forceinline__ static float value(const uint8_t* p, const uint8_t*) {
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

// Values that are not finite and were left out of the products are added to a row's stored result (or
// its share, where part is given): elements d .. d + 3, places [from, to).  The lane that stored them
// calls this.
template <typename E>
__device__ __forceinline__ void add_wild(const Args& a, int b, int h, int from, int to, int d, uint16_t* o, float* part) {
#pragma unroll 1
    for (int i = d; i < d + 4; ++i) {
        float x = part ? part[i] : __uint_as_float((uint32_t)o[i] << 16);
#pragma unroll 1
        for (int key = from; key < to; ++key) {
            const int p = page_of(a.s, b, key);
            if (p < 0) continue;
            const int64_t n = (int64_t)p * a.c.kv_heads + h;
            x += Held<E>::value(a.c.v + n * a.c.head_bytes + (((int64_t)i << a.c.page_log2) + (key & ((1 << a.c.page_log2) - 1))) * sizeof(E),
                                sizeof(E) == 1 ? a.c.v_scale + n : nullptr);
        }
        if (part) part[i] = x;
        else o[i] = (uint16_t)f32_to_bf16_bits(x);
    }
}

// 16 rows' part of the softmax over steps t0, t0 + by .. < t1 of a sequence.  A step's keys are loaded while the
// step before is in its second product, its values after that; nothing looks at what is on its way.
// Every byte is read once, past the caches (32 tokens to 8000, 332 MB: 76 -> 67 us).
// WIDE: a step's keys lie in one page, which is found and checked once for the wave.
template <typename E, int DP, bool WIDE>
struct Stream {
    static constexpr int ES = sizeof(E), KPL = 16 / ES, STEP = 4 * KPL, M = Held<E>::N;
    static constexpr int KC = DP * ES / 64;  // 16-byte pieces of a key's row a lane group takes
    static constexpr int DB = DP / 16;

    int tok, head;  // this lane's row
    bool live;
    int limit, all;  // places that it sees are those below; those that every row of the block sees
    bool wild;
    float m, l;
    f32x4_t o[DB];

    __device__ __forceinline__ void run(const Args& a, const Mine& sq, int h, int blk, int t0, int t1, int by) {
        const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
        const int dim = a.c.dim, lg = a.c.page_log2, pmask = (1 << lg) - 1, krow = dim * ES, vrow = ES << lg;
        const int row = blk * kRows + col, tok0 = (int)fdiv((uint32_t)(blk * kRows), a.group_div);
        live = row < sq.n * a.group;
        tok = live ? (int)fdiv((uint32_t)row, a.group_div) : 0;
        head = h * a.group + (live ? row - tok * a.group : 0);
        all = a.causal ? min(sq.past + tok0 + 1, sq.len) : sq.len;
        limit = !live ? all : a.causal ? min(sq.past + tok + 1, sq.len) : sq.len;
        wild = false;
        m = -INFINITY;
        l = 0.f;
#pragma unroll
        for (int d = 0; d < DB; ++d) o[d] = f32x4_t{0.f, 0.f, 0.f, 0.f};

        const int32_t* table = a.s.table + sq.b * a.s.table_stride;
        const int table_last = a.s.table_pages - 1;
        const int kin = KPL * (col >> 2), vin = KPL * g;  // first key of this lane's operand row's piece of four, of its scores and values
        int kpage, vpage = 0;
        auto find_pages = [&](int t) {
            kpage = table[max(min((t * STEP + (WIDE ? 0 : kin)) >> lg, table_last), 0)];
            if constexpr (!WIDE) vpage = table[max(min((t * STEP + vin) >> lg, table_last), 0)];
        };
        uint4 kr[M][2][KC], vr[DB];
        uint32_t kscale = 127, vscale = 127;
        bool paged;            // this lane's scores and values
        uint32_t vn = 0;       // page and head of the values
        auto slot = [&](int page, int key, bool& has) {
            has = key < sq.len && (uint32_t)page < (uint32_t)a.s.pages;
            return (uint32_t)((has ? page : 0) * a.c.kv_heads + h);
        };
        const uint32_t koff = (uint32_t)(((WIDE ? kin : 0) + (col & 3)) * krow + 16 * g), voff = (uint32_t)(col * vrow + (WIDE ? vin * ES : 0));
        auto load_k = [&](int t) {
            bool has;
            const uint32_t n = WIDE ? slot(__builtin_amdgcn_readfirstlane(kpage), t * STEP, has) : slot(kpage, t * STEP + kin, has);
            if constexpr (WIDE) vn = n;
            else vn = slot(vpage, t * STEP + vin, has);
            paged = has;
            const uint8_t* at = a.c.k + (uint64_t)n * (uint32_t)a.c.head_bytes + (uint32_t)((t * STEP + (WIDE ? 0 : kin)) & pmask) * (uint32_t)krow;
            if constexpr (ES == 1) {
                kscale = a.c.k_scale[n];
                vscale = a.c.v_scale[vn];
            }
#pragma unroll
            for (int mm = 0; mm < M; ++mm)
#pragma unroll
                for (int hh = 0; hh < 2; ++hh)
#pragma unroll
                    for (int c = 0; c < KC; ++c) {
                        // Pieces beyond the head's width are another's: their queries are 0, and they are cleared before use.
                        const bool in = DP * ES == krow || 16 * (g + 4 * c) < krow;
                        kr[mm][hh][c] = ld_stream(at + (in ? koff + (8 * mm + 4 * hh) * krow + 64 * c : 0));
                    }
        };
        auto load_v = [&](int t) {
            const uint8_t* at = a.c.v + (uint64_t)vn * (uint32_t)a.c.head_bytes + (uint32_t)((t * STEP + (WIDE ? 0 : vin)) & pmask) * ES;
#pragma unroll
            for (int d = 0; d < DB; ++d) vr[d] = ld_stream(at + (16 * d < dim ? 16 * d * vrow : 0) + voff);
        };
        if (t0 >= t1 || sq.len == 0) return;  // without a place there may be no table
        find_pages(t0);
        const int kpage0 = kpage, vpage0 = vpage;
        find_pages(t0 + by);
        const int kpage1 = kpage, vpage1 = vpage;
        kpage = kpage0;
        vpage = vpage0;
        // Queries first: the keys' loads wait for the pages anyway.
        bf16x8_t qf[KC][M];
        const uint16_t* qp = a.q + (int64_t)(sq.row + tok) * a.qs[0] + head * a.qs[1];
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
            for (int j = 0; j < M; ++j) {
                const int d = KPL * (g + 4 * c) + 8 * j;
                uint4 z = make_uint4(0, 0, 0, 0);
                if (live && d < dim) z = *reinterpret_cast<const uint4*>(qp + d);
                qf[c][j] = __builtin_bit_cast(bf16x8_t, z);
            }
        load_k(t0);
        load_v(t0);
        kpage = kpage1;
        vpage = vpage1;
        for (int t = t0; t < t1; t += by) {
            const bool here = paged;
            const float ks = ES == 1 ? __uint_as_float(max(kscale, 1u) << 23) : 1.f;
            // Of a place in no page the scale may be NaN.
            const float vs = ES == 1 && here ? __uint_as_float(max(vscale, 1u) << 23) : 1.f;
            f32x4_t s[M][2];
#pragma unroll
            for (int mm = 0; mm < M; ++mm)
#pragma unroll
                for (int hh = 0; hh < 2; ++hh) {
                    s[mm][hh] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int c = 0; c < KC; ++c) {
                        uint4 w = kr[mm][hh][c];
                        if (DP * ES != krow && 16 * (g + 4 * c) >= krow) w = make_uint4(0, 0, 0, 0);
#pragma unroll
                        for (int j = 0; j < M; ++j)
                            s[mm][hh] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(Held<E>::part(w, ks, j), qf[c][j], s[mm][hh], 0, 0, 0);
                    }
                }
            __builtin_amdgcn_sched_barrier(0);
            const bool more = t + by < t1;
            if (more) load_k(t + by);
            __builtin_amdgcn_sched_barrier(0);

            // Key 8 mm + 4 hh + i of this lane's is seen below `sees`.
            const int vb = t * STEP + vin, sees = here ? limit - vb : 0, holds = here ? min(max(sq.len - vb, 0), KPL) : 0;
            if (__builtin_amdgcn_ballot_w64(sees < KPL)) {
#pragma unroll
                for (int mm = 0; mm < M; ++mm)
#pragma unroll
                    for (int hh = 0; hh < 2; ++hh)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (8 * mm + 4 * hh + i >= sees) s[mm][hh][i] = -INFINITY;
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
            bf16x8_t pf[M], pl[M];
#pragma unroll
            for (int mm = 0; mm < M; ++mm) {
                float p[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[mm][e / 4][e & 3], a.scale_log2, -ref));
                    l += p[e];
                }
                // As two bf16, cut off and what that leaves: 2^-15 of a weight is lost, not 2^-8, for 0.1 to 0.4 us (32 tokens to
                // 8000 65.8 -> 66.2; against 64 bits 1.7e-3, the result's own rounding, instead of 2.2e-3).  The second
                // part is above 0 by 2^-23 of the weight, as 0 or less would make NaN of values that are infinite.
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t x = __float_as_uint(p[2 * e]), y = __float_as_uint(p[2 * e + 1]);
                    hi[e] = __builtin_amdgcn_perm(y, x, 0x07060302u);
                    lo[e] = pack_bf16x2(__builtin_fmaf(p[2 * e], 1.f + 0x1p-23f, -__uint_as_float(x & 0xffff0000u)),
                                        __builtin_fmaf(p[2 * e + 1], 1.f + 0x1p-23f, -__uint_as_float(y & 0xffff0000u)));
                }
                pf[mm] = __builtin_bit_cast(bf16x8_t, make_uint4(hi[0], hi[1], hi[2], hi[3]));
                pl[mm] = __builtin_bit_cast(bf16x8_t, make_uint4(lo[0], lo[1], lo[2], lo[3]));
            }
            // What lies behind the sequence, or in no page, is anything: values of weight 0 have to be numbers.
            if (__builtin_amdgcn_ballot_w64(holds < KPL)) {
#pragma unroll
                for (int d = 0; d < DB; ++d) vr[d] = leading<ES>(vr[d], holds);
            }
            // So have those that only some rows of the block see; what is none is added to these rows at the end.
            if ((t + 1) * STEP > all) {
                uint32_t any = 0;
                const uint32_t past = Held<E>::past(__float_as_uint(vs) >> 23);  // vscale is the next step's by now
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    const uint32_t wx = Held<E>::wild(vr[d].x, past), wy = Held<E>::wild(vr[d].y, past), wz = Held<E>::wild(vr[d].z, past),
                                   ww = Held<E>::wild(vr[d].w, past);
                    any |= wx | wy | wz | ww;
                    vr[d] = make_uint4(vr[d].x & ~wx, vr[d].y & ~wy, vr[d].z & ~wz, vr[d].w & ~ww);
                }
                wild |= __builtin_amdgcn_ballot_w64(any != 0) != 0;
            }
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int mm = 0; mm < M; ++mm) {
                    const bf16x8_t v = Held<E>::part(vr[d], vs, mm);
                    o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, pf[mm], o[d], 0, 0, 0);
                    o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, pl[mm], o[d], 0, 0, 0);
                }
            __builtin_amdgcn_sched_barrier(0);
            if (more) {
                // Pages first: results come in the order of the loads, and the next keys' loads wait for them.
                find_pages(t + 2 * by);
                __builtin_amdgcn_sched_barrier(0);
                load_v(t + by);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        l = xor_sum(l);
    }
    __device__ __forceinline__ uint16_t* out(const Args& a, const Mine& sq) const {
        return a.o + (int64_t)(sq.row + tok) * a.os[0] + head * a.os[1];
    }
};

// Wave id of all that share the stream out.
template <typename E, int DP, bool WIDE>
__device__ __forceinline__ void stream_part(const Args& a, int id) {
    typedef Stream<E, DP, WIDE> St;
    const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
    const int h = id / a.waves, w = id - h * a.waves;
    if (h >= a.c.kv_heads) return;
    Walk<St::STEP> walk(a);
    const int64_t total = walk.total();
    if (total == 0) return;
    const int64_t W = working(a, total);
    if (w >= W) return;
    const int64_t x1 = total * (w + 1) / W;
    for (int64_t x = total * w / W; x < x1;) {
        const Mine sq = walk.find(x);
        if (sq.b < 0) return;
        const int tiles = walk.tiles(sq.len), blk = (int)((x - sq.before) / tiles);
        const int64_t s0 = sq.before + (int64_t)blk * tiles;
        const int t0 = (int)(x - s0), t1 = (int)((x1 < s0 + tiles ? x1 : s0 + tiles) - s0);
        x = s0 + t1;
        St st;
        st.run(a, sq, h, blk, t0, t1, 1);
        if (!st.live) continue;
        const bool whole = t0 == 0 && t1 == tiles;
        const int64_t at = (((int64_t)h * a.waves + w) * 2 + (t0 == 0 ? 1 : 0)) * kRows + col;
        const float inv = !whole ? 1.f : st.l > 0.f ? 1.0f / st.l : (st.l == 0.f ? 0.f : st.l);  // no place seen: 0; NaN stays
        uint16_t* op = st.out(a, sq);
#pragma unroll
        for (int d = 0; d < St::DB; ++d) {
            const int e = 16 * d + 4 * g;
            const float v[4] = {st.o[d][0] * inv, st.o[d][1] * inv, st.o[d][2] * inv, st.o[d][3] * inv};
            if (!whole) attn::put4(a.part_o + at * DP + e, v);
            else if (16 * d < a.c.dim) attn::put4(reinterpret_cast<bf16*>(op) + e, v);
        }
        if (!whole && g == 0) {
            a.part_ml[2 * at] = st.m;
            a.part_ml[2 * at + 1] = st.l;
        }
        if (st.wild) {
#pragma unroll 1
            for (int d = 4 * g; d < a.c.dim; d += 16)
                add_wild<E>(a, sq.b, h, max(t0, st.all / St::STEP) * St::STEP, min(t1 * St::STEP, st.limit), d, op, whole ? nullptr : a.part_o + at * DP);
        }
    }
}

template <typename E, int DP, bool WIDE>
__global__ __launch_bounds__(256, 2) void kv_stream_kernel(const Args a) {
    stream_part<E, DP, WIDE>(a, (int)(blockIdx.x * 4) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6));
}

// Short tables: a workgroup takes a block of rows whole, its eight waves every eighth step, and joins them in LDS.
template <typename E, int DP, bool WIDE>
__global__ __launch_bounds__(512, 2) void kv_short_kernel(const Args a) {
    typedef Stream<E, DP, WIDE> St;
    constexpr int LD = DP + 4;  // a row's floats in LDS: rows in other banks
    extern __shared__ __attribute__((aligned(16))) float joined[];  // [8][kRows][LD]
    __shared__ float ml[8][kRows][2];
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = (int)(blockIdx.x % (uint32_t)a.c.kv_heads);
    const int64_t item = blockIdx.x / (uint32_t)a.c.kv_heads;
    const Found of = find_seq(a.s, item, [&a](int start, int i) { return first_block<kRows>(a, start, i); });
    const int b = of.b;
    if (b < 0) return;
    const Seq q = of.seq(a.s);
    const int64_t blk = item - first_block<kRows>(a, q.row, b), rows = q.n * (int64_t)a.group;
    if (blk < 0 || blk * kRows >= rows || rows > a.few) return;
    const Mine sq = {b, q.row, q.n, q.past, q.len, 0};
    const int tiles = max((sq.len + St::STEP - 1) / St::STEP, 1);
    St st;
    st.run(a, sq, h, (int)blk, wave, tiles, 8);
    float* mine = joined + (wave * kRows + col) * LD;
#pragma unroll
    for (int d = 0; d < St::DB; ++d) *reinterpret_cast<float4*>(mine + 16 * d + 4 * g) = make_float4(st.o[d][0], st.o[d][1], st.o[d][2], st.o[d][3]);
    if (g == 0) {
        ml[wave][col][0] = st.m;
        ml[wave][col][1] = st.l;
    }
    __syncthreads();
    const int n = min((int)(rows - blk * kRows), kRows);
    for (int i = tid; i < n * (DP / 4); i += 512) {
        const int r = i / (DP / 4), d = i % (DP / 4) * 4;
        if (d >= a.c.dim) continue;
        float m = ml[0][r][0];
#pragma unroll
        for (int w = 1; w < 8; ++w) m = fmaxf(m, ml[w][r][0]);
        const float ref = m == -INFINITY ? 0.f : m;
        float l = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 8; ++w) {
            const float f = __builtin_amdgcn_exp2f(ml[w][r][0] - ref);
            const float4 x = *reinterpret_cast<const float4*>(joined + (w * kRows + r) * LD + d);
            l += f * ml[w][r][1];
            v[0] += f * x.x;
            v[1] += f * x.y;
            v[2] += f * x.z;
            v[3] += f * x.w;
        }
        const float inv = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] *= inv;
        const int row = (int)blk * kRows + r, tok = (int)fdiv((uint32_t)row, a.group_div);
        attn::put4(reinterpret_cast<bf16*>(a.o) + (int64_t)(sq.row + tok) * a.os[0] + (h * a.group + row - tok * a.group) * a.os[1] + d, v);
    }
    if (!__syncthreads_or(st.wild)) return;
    __syncthreads();  // the results that other waves stored are read
    if (wave != 0 || !st.live) return;
#pragma unroll 1
    for (int d = 4 * g; d < a.c.dim; d += 16)
        add_wild<E>(a, b, h, st.all / St::STEP * St::STEP, min(tiles * St::STEP, st.limit), d, st.out(a, sq), nullptr);
}

// The key ranges of a row, joined in their order: a thread per four elements.
template <int DP>
__device__ __forceinline__ void join_ranges(const Args& a, int block) {
    constexpr int TPR = DP / 4;
    const int64_t n = (int64_t)a.s.rows * a.heads, id = ((int64_t)block * 256 + threadIdx.x) / TPR;
    const int d = (int)(threadIdx.x % TPR) * 4;
    // The sequences of the wave's rows, one after the other, by the whole wave.
    bool mine = false;
#pragma unroll
    for (int k = 0; k < 64 / TPR; ++k) {
        const int r = min(__shfl((int)(id / a.heads), k * TPR, 64), a.s.rows - 1);
        const Found of = find_seq(a.s, r, [](int start, int) { return start; });
        if (of.b < 0) continue;
        const Seq sq = of.seq(a.s);
        if ((int)(threadIdx.x & 63) / TPR == k) mine = r - sq.row < sq.n && sq.n * (int64_t)a.group > a.few;
    }
    if (!mine || id >= n || d >= a.c.dim) return;
    float m = -INFINITY, l = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < a.splits; s0 += 4) {
        float2 ml[4];
        float4 x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // all on their way before the first is used
            const int64_t at = (int64_t)min(s0 + i, a.splits - 1) * n + id;
            ml[i] = *reinterpret_cast<const float2*>(a.rows_ml + 2 * at);
            x[i] = *reinterpret_cast<const float4*>(a.rows_o + at * DP + d);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (s0 + i >= a.splits) break;
            const float to = fmaxf(m, ml[i].x), ref = to == -INFINITY ? 0.f : to;
            const float f0 = __builtin_amdgcn_exp2f(m - ref), f1 = __builtin_amdgcn_exp2f(ml[i].x - ref);
            m = to;
            l = l * f0 + ml[i].y * f1;
            v[0] = v[0] * f0 + x[i].x * f1;
            v[1] = v[1] * f0 + x[i].y * f1;
            v[2] = v[2] * f0 + x[i].z * f1;
            v[3] = v[3] * f0 + x[i].w * f1;
        }
    }
    const float inv = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] *= inv;
    const int r = (int)(id / a.heads), head = (int)(id - (int64_t)r * a.heads);
    attn::put4(reinterpret_cast<bf16*>(a.o) + (int64_t)r * a.os[0] + head * a.os[1] + d, v);
}

// The partial results of a row: TPR threads, each every PL-th wave's share of four elements.  Rows are
// numbered as (token, head), or, beside the row blocks' kernel, as (sequence, key head, row of up to kFew).
template <typename E, int DP, int TPR>
__global__ __launch_bounds__(256) void kv_join_kernel(const Args a) {
    constexpr int STEP = 4 * (16 / (int)sizeof(E)), LPD = DP / 4, PL = TPR / LPD;
    if ((int)blockIdx.x >= a.join_blocks) {
        join_ranges<DP>(a, (int)blockIdx.x - a.join_blocks);
        return;
    }
    __shared__ float part[256][6];
    const int tid = threadIdx.x, sub = tid % TPR, pl = sub / LPD, d0 = (sub % LPD) * 4;
    const int64_t id = (int64_t)blockIdx.x * (256 / TPR) + __builtin_amdgcn_readfirstlane(tid / TPR);
    const bool by_seq = a.few == kFew;
    const int b = (int)(id / (a.c.kv_heads * kFew)), r0 = (int)(id / a.heads);
    float m = -INFINITY, l = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
    bool join = false;
    Walk<STEP> walk(a);
    Mine sq;
    const int64_t total = walk.total([&] { return by_seq ? walk.from + (tid & 63) == b : r0 >= walk.row && r0 - walk.row < walk.n; }, &sq);
    int r = 0, head = 0;
    if (sq.b >= 0 && total > 0) {
        const int h = by_seq ? (int)(id / kFew % a.c.kv_heads) : (int)(id % a.heads) / a.group;
        const int row = by_seq ? (int)(id % kFew) : (r0 - sq.row) * a.group + (int)(id % a.heads) % a.group;
        r = sq.row + row / a.group;
        head = h * a.group + row % a.group;
        if (row < sq.n * (int64_t)a.group && sq.n * (int64_t)a.group <= a.few) {
            const int tiles = walk.tiles(sq.len);
            const int64_t s0 = sq.before + (int64_t)(row / kRows) * tiles, W = working(a, total);
            const int w0 = (int)(((s0 + 1) * W - 1) / total), w1 = (int)(((s0 + tiles) * W - 1) / total);
            join = w0 != w1;
            for (int w = w0 + pl; join && w <= w1; w += 4 * PL) {
                float2 ml[4];
                float4 x[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {  // all on their way before the first is used
                    const int from = min(w + i * PL, w1);
                    const int64_t at = (((int64_t)h * a.waves + from) * 2 + (from == w0 ? 1 : 0)) * kRows + row % kRows;
                    ml[i] = *reinterpret_cast<const float2*>(a.part_ml + 2 * at);
                    x[i] = *reinterpret_cast<const float4*>(a.part_o + at * DP + d0);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (w + i * PL > w1) break;
                    const float to = fmaxf(m, ml[i].x), ref = to == -INFINITY ? 0.f : to;
                    const float f0 = __builtin_amdgcn_exp2f(m - ref), f1 = __builtin_amdgcn_exp2f(ml[i].x - ref);
                    m = to;
                    l = l * f0 + ml[i].y * f1;
                    v[0] = v[0] * f0 + x[i].x * f1;
                    v[1] = v[1] * f0 + x[i].y * f1;
                    v[2] = v[2] * f0 + x[i].z * f1;
                    v[3] = v[3] * f0 + x[i].w * f1;
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

// ---- many rows: 256 or 128 rows per workgroup, 32 per wave, tiles of 64 keys --------------
// Codes are turned into bf16 once for the workgroup, on their way through registers into LDS; bf16
// comes there by direct DMA.  Every wave multiplies from there on v_mfma_f32_32x32x16_bf16, again transposed: a lane
// holds one row.  LDS row 8 a + 4 g + c of a tile's 16 holds key 8 g + 4 a + c, so that a lane's
// scores are those of 8 keys in order, and a value's operand one 16-byte piece.
//
// The barrier of every tile keeps the waves in step, so each wave's matrix and vector
// instructions have to overlap by themselves: a step takes 32 keys through three stages at once, the scores of the next 32, the softmax of
// these, and the product with the values of the 32 before, none of which waits for another.
// Keys therefore run a tile ahead of values in LDS (two buffers each).
constexpr int kTile = 64;
constexpr uint32_t kOne = 127;  // a page's scale of 1

// The softmax of 32 keys for one row: reference m (log2), this lane's half of the sum.
template <int BLOCKS>
struct Softmax {
    float m, l, sum;
    f32x16_t o[BLOCKS];
    __device__ __forceinline__ float ref() const { return m == -INFINITY ? 0.f : m; }
    // Whether the weights by the reference as it is may stay: nearly always, and then their sizes are never
    // looked at.  Weights whose sum in a lane is at most 2^12 are small enough; without a reference yet
    // (ref() is then 0) they may all be too small.
    __device__ __forceinline__ bool stays() const { return __builtin_amdgcn_ballot_w64(sum > 4096.0f || m == -INFINITY) == 0; }
    // A reference for scores s: it moves when one exceeds it by more than 2^8, and the sums before follow.
    __device__ __forceinline__ void refer(const f32x16_t& s, float sc) {
        float top = s[0];
#pragma unroll
        for (int e = 1; e < 16; ++e) top = fmaxf(top, s[e]);
        top = fmaxf(top, attn::swap32(top)) * sc;
        const bool move = top > m + 8.0f;
        const float alpha = move ? __builtin_amdgcn_exp2f(m - top) : 1.0f;
        m = move ? top : m;
        l *= alpha;
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[b][e] *= alpha;
    }
    // Elements 2 i and 2 i + 1 as weights, and those rounded to bf16 for the product, where a second part of each would be half
    // as many products again.  The sum takes them as the product does: what rounding adds to all of them it takes off again.
    __device__ __forceinline__ static void weigh(const f32x16_t& s, float sc, float minus_ref, int i, float (&x)[2]) {
#pragma unroll
        for (int e = 0; e < 2; ++e) x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * i + e], sc, minus_ref));
    }
    __device__ __forceinline__ void pack(const float (&x)[2], uint32_t& w) {
        w = pack_bf16x2(x[0], x[1]);
        const bf16x2_t ones = {(__bf16)1.0f, (__bf16)1.0f};
        sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, w), ones, sum, false);
        asm volatile("" : "+v"(w), "+v"(sum));  // made here, not where they are first used
    }
};

// 16 bytes a lane from `at` to lds + 16 lane (lds uniform) by direct DMA.
__device__ __forceinline__ void dma16(const uint8_t* at, uint8_t* lds) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)at, (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
}

// Its first workgroups share out the stream of the sequences of few rows, which waits for memory while
// the others multiply.
template <typename E, int DP, bool WIDE, int NW>
__global__ __launch_bounds__(64 * NW, 2) void kv_rows_kernel(const Args a) {
    if ((int)blockIdx.x < a.stream_blocks) {
        stream_part<E, DP, WIDE>(a, (int)(blockIdx.x * NW) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6));
        return;
    }
    constexpr int kThreads = 64 * NW, kBlock = 32 * NW;
    typedef attn::Tile<bf16, DP> KT;
    typedef attn::Tile<bf16, kTile> VT;
    typedef typename KT::Frag Frag;
    constexpr int ES = sizeof(E), KPL = 16 / ES, M = Held<E>::N;
    constexpr int KCH = DP / KPL, VCH = kTile / KPL;                           // 16-byte pieces of a row
    constexpr int PIECES = kTile * KCH, J = (PIECES + kThreads - 1) / kThreads;               // of a tile, a thread's
    constexpr int KBYTES = kTile * KT::RB, VBYTES = DP * VT::RB;
    static_assert(PIECES == DP * VCH && (PIECES % kThreads == 0 || J == 1), "pieces");
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];             // [2][K], [2][V]
    __shared__ uint32_t paged[2];                                              // a byte per 16 keys: whether they have a page
    __shared__ int wild_seen;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 31, g = lane >> 5;

    // Heads innermost: an XCD's workgroups share them.  The longest rows first.
    const uint32_t bid = blockIdx.x - a.stream_blocks, n_items = (gridDim.x - a.stream_blocks) / (uint32_t)(a.c.kv_heads * a.splits);
    const int h = (int)(bid % (uint32_t)a.c.kv_heads);
    const uint32_t rest = bid / (uint32_t)a.c.kv_heads;
    const int split = (int)(rest % (uint32_t)a.splits);
    const int64_t item = (int64_t)n_items - 1 - rest / (uint32_t)a.splits;
    const Found of = find_seq(a.s, item, [&a](int start, int i) { return first_block<kBlock>(a, start, i); });
    const int b = of.b;
    if (b < 0) return;
    const Seq sq = of.seq(a.s);
    const int64_t all_rows = sq.n * (int64_t)a.group, row0 = (item - first_block<kBlock>(a, sq.row, b)) * kBlock;
    if (all_rows <= a.few || row0 < 0 || row0 >= all_rows) return;
    const int rows = (int)all_rows, first = (int)row0, last = min(first + kBlock, rows) - 1;
    // The places that a row sees are those below:
    auto limit_of = [&](int row) { return a.causal ? min(sq.past + (int)fdiv((uint32_t)row, a.group_div) + 1, sq.len) : sq.len; };
    const int most = limit_of(last), all = limit_of(first);  // some row sees, every row sees
    const int tiles = (most + kTile - 1) / kTile;
    const int t0 = (int)((int64_t)tiles * split / a.splits), t1 = (int)((int64_t)tiles * (split + 1) / a.splits);

    const int row = first + wave * 32 + r;
    const bool live = row < rows;
    const int tok = live ? (int)fdiv((uint32_t)row, a.group_div) : 0, head = h * a.group + (live ? row - tok * a.group : 0);
    const int limit = live ? limit_of(row) : all;
    // This wave's tiles end where its last row sees no more.
    const int wave_last = min(first + wave * 32 + 31, rows - 1);
    const int w1 = wave_last < first + wave * 32 ? t0 : max(t0, min(t1, (limit_of(wave_last) + kTile - 1) / kTile));

    const int dim = a.c.dim, lg = a.c.page_log2, pmask = (1 << lg) - 1, krow = dim * ES, vrow = ES << lg;
    // This thread's pieces of a tile.  Codes come through registers: piece tid + kThreads j in the pool's
    // order.  bf16 goes to LDS by direct DMA: the piece that belongs at place 64 (J wave + j) + lane there.
    constexpr bool DMA = ES == 2;
    static_assert(!DMA || PIECES % kThreads == 0, "pieces");
    auto piece = [&](int j) { return DMA ? (wave * J + j) * 64 + lane : min(tid + kThreads * j, PIECES - 1); };
    auto swapped = [](int key) { return (key & 0x33) | ((key & 4) << 1) | ((key & 8) >> 1); };
    auto k_key = [&](int j) { return DMA ? swapped(piece(j) / KCH) : piece(j) / KCH; };
    auto k_col = [&](int j) { return DMA ? (piece(j) % KCH) ^ KT::swz(piece(j) / KCH) : piece(j) % KCH; };
    auto v_dim = [&](int j) { return piece(j) / VCH; };
    auto v_col = [&](int j) { return DMA ? (piece(j) % VCH) ^ VT::swz(v_dim(j)) : piece(j) % VCH; };

    // What is on its way stays as it is loaded: whatever looks at it would wait for it.  Threads
    // without a piece, and places without a page, load another's.
    uint4 kst[DMA ? 1 : J], vst[DMA ? 1 : J];
    uint32_t kscale[J], vscale[J];
    bool khas[J], vhas[J];     // whether they lie in a page
    int kpage[J], vpage[J];    // the table's entries for the tiles that are loaded next
    uint32_t koff[J], voff[J];  // this thread's pieces in a page, from the tile's first place in it on
    int kin[J], vin[J];         // and their first places in the tile
#pragma unroll
    for (int j = 0; j < J; ++j) {
        kin[j] = k_key(j);
        vin[j] = v_col(j) * KPL;
        koff[j] = (kin[j] & pmask) * krow + (16 * k_col(j) < krow ? 16 * k_col(j) : 0);
        voff[j] = (v_dim(j) < dim ? v_dim(j) : 0) * vrow + (vin[j] & pmask) * ES;
    }
    const int32_t* table = a.s.table + b * a.s.table_stride;
    const int table_last = a.s.table_pages - 1;
    // WIDE: a tile lies in one page, which is found and checked once for the wave.
    constexpr int PJ = WIDE ? 1 : J;
    auto find_pages = [&](int kt, int vt) {
#pragma unroll
        for (int j = 0; j < PJ; ++j) {
            kpage[j] = table[min((kt * kTile + (WIDE ? 0 : kin[j])) >> lg, table_last)];
            vpage[j] = table[min((vt * kTile + (WIDE ? 0 : vin[j])) >> lg, table_last)];
        }
    };
    auto load = [&](const uint8_t* pool, const uint8_t* scales, int t, const int (&in_tile)[J], const int (&page)[J], const uint32_t (&off)[J],
                    uint4* w, uint8_t* lds, uint32_t (&scale)[J], bool (&has)[J], int tile_bytes) {
        const uint8_t* from[PJ];
#pragma unroll
        for (int j = 0; j < PJ; ++j) {
            const int pg = WIDE ? __builtin_amdgcn_readfirstlane(page[j]) : page[j];
            has[j] = t * kTile + (WIDE ? 0 : in_tile[j]) < sq.len && (uint32_t)pg < (uint32_t)a.s.pages;
            const uint32_t n = (uint32_t)((has[j] ? pg : 0) * a.c.kv_heads + h);
            from[j] = pool + (uint64_t)n * (uint32_t)a.c.head_bytes + (uint32_t)((t * kTile & pmask) * tile_bytes);
            if constexpr (ES == 1) scale[j] = scales[n];
        }
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const uint8_t* at = from[WIDE ? 0 : j] + off[j];
            if constexpr (DMA) dma16(at, lds + (wave * J + j) * 1024);
            else w[j] = *reinterpret_cast<const uint4*>(at);
        }
    };
    auto k_buf = [&](int t) { return smem + (t & 1) * KBYTES; };
    auto v_buf = [&](int t) { return smem + 2 * KBYTES + (t & 1) * VBYTES; };
    auto load_k = [&](int t) { load(a.c.k, a.c.k_scale, t, kin, kpage, koff, kst, k_buf(t), kscale, khas, krow); };
    auto load_v = [&](int t) { load(a.c.v, a.c.v_scale, t, vin, vpage, voff, vst, v_buf(t), vscale, vhas, ES); };
    auto factor = [](uint32_t scale) { return ES == 1 ? __uint_as_float(max(scale, 1u) << 23) : 1.f; };
    // Part `part` of this thread's pieces into LDS: half a piece of codes.
    constexpr int PARTS = DMA ? 0 : J * M;
    auto put_k = [&](int t, int part) {
        const int j = part / M, m = part % M, lr = swapped(k_key(j));
        if (PIECES % kThreads && tid + kThreads * j >= PIECES) return;
        *reinterpret_cast<bf16x8_t*>(k_buf(t) + lr * KT::RB + (((M * k_col(j) + m) ^ KT::swz(lr)) << 4)) =
            Held<E>::part(kst[j], factor(kscale[WIDE ? 0 : j]), m);
    };
    auto put_v = [&](int t, int part) {
        const int j = part / M, m = part % M, d = v_dim(j);
        if (PIECES % kThreads && tid + kThreads * j >= PIECES) return;
        *reinterpret_cast<bf16x8_t*>(v_buf(t) + d * VT::RB + (((M * v_col(j) + m) ^ VT::swz(d)) << 4)) =
            Held<E>::part(vst[j], factor(vscale[WIDE ? 0 : j]), m);
    };
    // Before codes are put, after bf16 is there: whether keys have pages, and what may not enter a product.
    auto mend_k = [&](int t) {
        if (DP * ES > krow) {  // beyond the head's width
#pragma unroll
            for (int j = 0; j < J; ++j)
                if (16 * k_col(j) >= krow) {
                    if constexpr (DMA) *reinterpret_cast<uint4*>(k_buf(t) + 16 * piece(j)) = make_uint4(0, 0, 0, 0);
                    else kst[j] = make_uint4(0, 0, 0, 0);
                }
        }
        if constexpr (WIDE) {
            if (tid == 0) paged[t & 1] = khas[0] ? 0x01010101u : 0;
        } else {
#pragma unroll
            for (int j = 0; j < J; ++j)
                if ((PIECES % kThreads == 0 || tid + kThreads * j < PIECES) && k_col(j) == 0 && kin[j] % 16 == 0)
                    reinterpret_cast<uint8_t*>(&paged[t & 1])[kin[j] / 16] = khas[j] ? 1 : 0;
        }
    };
    auto mend_v = [&](int t) {
        bool there = true;
#pragma unroll
        for (int j = 0; j < PJ; ++j) there &= vhas[j];
        // What lies behind the sequence, or in no page, is anything: values of weight 0 have to be numbers.
        const bool tail = (t + 1) * kTile > sq.len || !(WIDE ? there : __builtin_amdgcn_ballot_w64(!there) == 0);
        // So have those that only some rows see; what is none is added to those rows at the end.
        const bool some = (t + 1) * kTile > all;
        if (__builtin_expect(tail || some, 0)) {
#pragma unroll
            for (int j = 0; j < J; ++j) {
                uint4* const at = reinterpret_cast<uint4*>(v_buf(t) + 16 * piece(j));
                uint4 v;
                if constexpr (DMA) v = *at;
                else v = vst[j];
                const bool has = vhas[WIDE ? 0 : j];
                v = leading<ES>(v, has ? max(sq.len - (t * kTile + vin[j]), 0) : 0);
                if (some) {
                    uint32_t scale = ES == 1 ? vscale[WIDE ? 0 : j] : kOne;
                    asm("" : "+v"(scale));  // a scalar would be made of it, and waited for, where it is loaded
                    const uint32_t past = Held<E>::past(scale);
                    const uint32_t wx = Held<E>::wild(v.x, past), wy = Held<E>::wild(v.y, past), wz = Held<E>::wild(v.z, past), ww = Held<E>::wild(v.w, past);
                    if (wx | wy | wz | ww) wild_seen = 1;
                    v = make_uint4(v.x & ~wx, v.y & ~wy, v.z & ~wz, v.w & ~ww);
                }
                if constexpr (DMA) *at = v;
                else vst[j] = v;
                if (!has) vscale[WIDE ? 0 : j] = kOne;
            }
        }
    };

    Frag qf[KT::STEPS];
    {
        const bf16* qp = reinterpret_cast<const bf16*>(a.q) + (int64_t)(sq.row + tok) * a.qs[0] + head * a.qs[1];
#pragma unroll
        for (int c = 0; c < KT::STEPS; ++c) qf[c] = live ? attn::frag_global<bf16>(qp, c, g, dim) : attn::frag_zero<bf16>();
    }
    Softmax<KT::BLOCKS> run;
    run.m = -INFINITY;
    run.l = 0.f;
#pragma unroll
    for (int d = 0; d < KT::BLOCKS; ++d) run.o[d] = attn::zero16();
    const float sc = a.scale_log2;
    // Scores and weights of the even and of the odd 32 keys.
    f32x16_t s[2];
    attn::FragParts<bf16> p[2][2];
#pragma unroll
    for (int e = 0; e < 16; ++e) s[1][e] = -INFINITY;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) p[0][j].w[e] = 0;

    // One step: the softmax of scores s[1 - hh], the product of weights p[hh] with half hh of the values at
    // V, and the scores s[hh] of half hh of the keys at K, tile t.  Its products alternate, scores
    // and values; beside each goes the read of the operand four products on (the first ones' are in
    // f already) and a piece of the vector work, in this order.  (In larger pieces the compiler
    // gathers the products, and each waits for the one before with the vector work behind it.)
    constexpr int NS = KT::STEPS, N = 2 * NS, AHEAD = NW == 8 ? 4 : 3, RING = AHEAD + 1;  // three: what registers are left for
    static_assert(NS == 2 * KT::BLOCKS, "as many products of either kind");
    Frag f[RING];
    auto read = [&](int hh, const uint8_t* K, const uint8_t* V, int i) {
        const int n = i / 2;
        f[(hh * N + i) % RING] = i & 1 ? VT::row_frag(V, 32 * (n % KT::BLOCKS) + r, 2 * hh + n / KT::BLOCKS, g) : KT::row_frag(K, 32 * hh + r, n, g);
    };
    auto step = [&](auto hc, const uint8_t* K, const uint8_t* V, int t, uint32_t has, auto put) {
        constexpr int hh = decltype(hc)::value;
        const f32x16_t& now = s[1 - hh];
        f32x16_t next = attn::zero16();
        float x[8][2];
        const float minus_ref = -run.ref();
        run.sum = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (i + AHEAD < N) read(hh, K, V, i + AHEAD);
            else if (hh == 0) read(1, K, V, i + AHEAD - N);
            if (i & 1) run.o[i / 2 % KT::BLOCKS] = attn::mma(f[(hh * N + i) % RING], p[hh][i / 2 / KT::BLOCKS].frag(), run.o[i / 2 % KT::BLOCKS]);
            else next = attn::mma(f[(hh * N + i) % RING], qf[i / 2], next);
            // Two weights' exponentials, those of two products before into their operand, then what goes to LDS.
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if (1 + k * N / 16 == i) run.weigh(now, sc, minus_ref, k, x[k]);
                if (1 + N / 8 + k * N / 16 == i) run.pack(x[k], p[1 - hh][k / 4].w[k % 4]);
            }
#pragma unroll
            for (int k = 0; k < PARTS; ++k)
                if (N / 2 + 3 + k * (N / 2 - 3) / (PARTS ? PARTS : 1) == i) put(k);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (__builtin_expect(!run.stays(), 0)) {
            run.refer(now, sc);
            run.sum = 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                run.weigh(now, sc, -run.ref(), k, x[k]);
                run.pack(x[k], p[1 - hh][k / 4].w[k % 4]);
            }
        }
        // Element 8 j + e is key 16 j + 8 g + e of the half.
        if (__builtin_expect((t + 1) * kTile > all || t >= w1, 0)) {
            const int sees = t >= w1 ? 0 : limit - (t * kTile + 32 * hh + 8 * g);
#pragma unroll
            for (int i = 0; i < 16; ++i) next[i] = 16 * (i >> 3) + (i & 7) < sees ? next[i] : -INFINITY;
        }
        if (__builtin_expect(has != 0x01010101u, 0)) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const bool there = has >> (8 * (2 * hh + j)) & 1;
#pragma unroll
                for (int e = 0; e < 8; ++e) next[8 * j + e] = there ? next[8 * j + e] : -INFINITY;
            }
        }
        run.l += run.sum;
        s[hh] = next;
    };

    // Before the first tile the weights are 0, and so have to be the values.
    for (int i = tid; i < VBYTES / 16; i += kThreads)
        *reinterpret_cast<uint4*>(smem + 2 * KBYTES + ((t0 + 1) & 1) * VBYTES + 16 * i) = make_uint4(0, 0, 0, 0);
    if (tid == 0) wild_seen = 0;
    if (t0 < t1) {
        find_pages(t0, t0);
        load_k(t0);
        if constexpr (DMA) attn::wait_vmem<0>();
        mend_k(t0);
#pragma unroll
        for (int part = 0; part < PARTS; ++part) put_k(t0, part);
        find_pages(t0 + 1, t0);
        if constexpr (!DMA) {
            load_k(t0 + 1);
            load_v(t0);
            find_pages(t0 + 2, t0 + 1);
        }
    }
    attn::wait_vmem<0>();  // the queries: their first use would wait for the loop's first loads too
    // Keys a tile ahead: at hand are those of tile t + 1 and the values of tile t.  Meanwhile those of tiles
    // t + 2 and t + 1 come to LDS (codes by way of registers, a tile earlier), where nobody reads any more.
#pragma unroll 1
    for (int t = t0 - 1; t < t1; ++t) {
        __syncthreads();
        const uint8_t* K = k_buf(t + 1);
        const uint8_t* V = v_buf(t + 2);
        const uint32_t has = __builtin_amdgcn_readfirstlane(paged[(t + 1) & 1]);
        if (t + 1 < t1) {
            if constexpr (DMA) {
                load_k(t + 2);
                load_v(t + 1);
                find_pages(t + 3, t + 2);
            } else {
                mend_k(t + 2);
                mend_v(t + 1);
            }
        }
        if (t < w1) {
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) read(0, K, V, i);
            step(std::integral_constant<int, 0>{}, K, V, t + 1, has, [&](int part) { put_k(t + 2, part); });
            if (!DMA && t + 2 < t1) load_k(t + 3);
            step(std::integral_constant<int, 1>{}, K, V, t + 1, has, [&](int part) { put_v(t + 1, part); });
        } else if (t + 1 < t1) {
#pragma unroll
            for (int part = 0; part < PARTS; ++part) {
                put_k(t + 2, part);
                put_v(t + 1, part);
            }
            if (!DMA && t + 2 < t1) load_k(t + 3);
        }
        if constexpr (DMA) {
            if (t + 1 < t1) {
                attn::wait_vmem<0>();
                mend_k(t + 2);
                mend_v(t + 1);
            }
        } else if (t + 2 < t1) {
            load_v(t + 2);
            find_pages(t + 4, t + 3);
        }
    }
    __syncthreads();
    const float l = run.l + attn::swap32(run.l);
    if (!live) return;
    const bool whole = a.splits == 1;
    const float inv = !whole ? 1.f : l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);  // no place seen: 0; NaN stays
    bf16* op = reinterpret_cast<bf16*>(a.o) + (int64_t)(sq.row + tok) * a.os[0] + head * a.os[1];
    const int64_t at = ((int64_t)split * a.s.rows + sq.row + tok) * a.heads + head;
#pragma unroll
    for (int d = 0; d < KT::BLOCKS; ++d)
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) {
            const int e0 = 32 * d + 8 * i4 + 4 * g;
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = run.o[d][4 * i4 + e] * inv;
            if (!whole) attn::put4(a.rows_o + at * DP + e0, v);
            else if (e0 < dim) attn::put4(op + e0, v);
        }
    if (!whole && g == 0) {
        a.rows_ml[2 * at] = run.m;
        a.rows_ml[2 * at + 1] = l;
    }
    if (wild_seen) {
#pragma unroll 1
        for (int e = 4 * g; e < dim; e += 8)
            add_wild<E>(a, b, h, max(t0, all / kTile) * kTile, min(t1 * kTile, limit), e, reinterpret_cast<uint16_t*>(op),
                        whole ? nullptr : a.rows_o + at * DP);
    }
}

// ---- choice and launch --------------------------------------------------------------
struct Plan {
    bool stream, rows, whole;    // whole: the stream's blocks of rows are not shared out
    int few, waves, dp, block, splits;
    int64_t blocks;             // of rows, at most
    int64_t floats, row_floats;  // workspace: the stream's partial results, the row blocks'
};

// What a sequence's rows are is known on the device: with more rows than sequences both kernels
// are launched, and each takes its own.
Plan plan(const Cache& c, const Seqs& s, int64_t heads, int cus) {
    Plan p{};
    const int64_t group = heads / c.kv_heads, rows = s.rows * group;
    p.dp = c.dim <= 64 ? 64 : 128;
    p.rows = s.rows > s.seqs && rows > kFew;
    p.stream = !p.rows || s.seqs > 1;
    p.few = !p.rows ? INT32_MAX : p.stream ? kFew : 0;
    p.splits = 1;
    // By the table, as wide as it is: what is held is known on the device only (one token to 1001 10.9 us, with a table of 64
    // pages of 64 16.6).  A workgroup's time goes by its own bytes, the stream's by all of them, with 5 to 8 us for its second launch
    // (32 on 8 heads of 128, whole and shared out: bf16, one token to 800 14 and 17.5 us, 8 to 1500 27 and 20; e4m3, 16
    // to 1500 17 and 21).  Blocks enough for every CU may be twice as long (e4m3, 32 tokens to 2300 23 and 30, 64
    // to 3700 54 and 64; but 24 to 3900 of 16 heads of 64 in bf16 53 and 48).
    const int64_t bytes = ((int64_t)s.table_pages << s.page_log2) * p.dp * (c.k_scale ? 1 : 2), blocks = (rows / kRows + s.seqs) * c.kv_heads;
    p.whole = !p.rows && bytes <= (blocks >= cus ? 2 : 1) * (int64_t)kShort;
    if (p.stream && !p.whole) {
        // Two waves a SIMD in all.  Beside blocks of rows a quarter of that, and so of the CUs at most: where there are
        // prompts the stream is over before the products are (with all of its waves first the step of 17 requests below
        // took 128 us).
        p.waves = ((p.rows ? 2 : 8) * cus / c.kv_heads + 7) / 8 * 8;
        if (p.waves < 8) p.waves = 8;
        p.floats = (int64_t)c.kv_heads * p.waves * 2 * kRows * (p.dp + 2);
    }
    if (p.rows) {
        // Blocks of 256 rows, one workgroup a CU, where keys are many and so are blocks, or a single
        // sequence's keys are shared out anyway (32 heads on 8 x 128: 4096 tokens 149 us against 159 in blocks
        // of 128; 512 behind 30000 245 and 262).  Else 128 rows and two workgroups a CU, of which one starts
        // while the other works, and fewer rows are filled up (2048 tokens 62 us against 70; 8 x 1024 78 and 87;
        // 4 x 300 behind 5000 101 and 127), but for codes in pages of less than a tile, whose 128 rows lack the
        // registers (17 requests, two of them with 512 new tokens, behind 3500, pages of 16: 112 us against 99;
        // in bf16 116 against 125, two requests alone 94 against 89).
        const int64_t keys = (int64_t)s.table_pages << s.page_log2;  // that the table has places for (see above)
        const bool many = keys >= 4096 && (rows * c.kv_heads >= 512 * (int64_t)cus || s.seqs == 1);
        p.block = many || (c.k_scale && 1 << c.page_log2 < kTile) ? 256 : 128;
        p.blocks = rows / p.block + s.seqs;
        const int64_t full = ((rows + p.block - 1) / p.block) * c.kv_heads;
        // Twice as many beside a stream, whose workgroups end at their own time (17 requests, two of them with
        // 512 new tokens, behind 3500: 143 -> 124 us).
        int64_t n = (p.block == 128 ? 2 : 1) * (p.stream ? 2 : 1) * cus / (full > 0 ? full : 1);
        // Eight tiles a range (64 tokens behind 1000: 25.5 us, 22 with four, 32 with sixteen; 200: 30, 31, 34).
        const int64_t longest = keys / (8 * kTile);
        if (n > longest) n = longest;
        if (n > 32) n = 32;
        p.splits = n < 2 ? 1 : (int)n;
        if (p.splits > 1) p.row_floats = (int64_t)p.splits * s.rows * heads * (p.dp + 2);
    }
    return p;
}

template <typename E, int DP>
int launch(Args& a, const Plan& p, hipStream_t st) {
    const int64_t n = (int64_t)a.s.rows * a.heads;
    const bool wide = 1 << a.c.page_log2 >= (p.rows ? kTile : Stream<E, DP, true>::STEP);
    if (p.whole) {
        const int64_t blocks = (n / a.c.kv_heads / kRows + a.s.seqs) * a.c.kv_heads;
        DT_REQUIRE(grid_fits(blocks, 512), "dt_kv_attn: grid too large");
        const dim3 grid((unsigned)blocks);
        const size_t lds = 8 * kRows * (DP + 4) * sizeof(float);
        if (wide) hipLaunchKernelGGL((kv_short_kernel<E, DP, true>), grid, dim3(512), lds, st, a);
        else hipLaunchKernelGGL((kv_short_kernel<E, DP, false>), grid, dim3(512), lds, st, a);
        return check_launch("dt_kv_attn");
    }
    // Shares of the stream: few rows may each have many, then a workgroup a row (24 tokens to 4000, 768 rows: 34 us, in
    // fours 36; 4096 rows 129 and 122).  Key ranges: four elements a thread.
    const int64_t joined = !p.stream ? 0 : p.rows ? (int64_t)a.s.seqs * a.c.kv_heads * kFew : n;
    const int64_t ranges = p.splits > 1 ? (n * (DP / 4) + 255) / 256 : 0;
    const int64_t join_blocks = joined <= 1024 ? joined : (joined + 3) / 4;
    DT_REQUIRE(grid_fits(join_blocks + ranges, 256), "dt_kv_attn: grid too large");
    if (p.rows) {
        a.stream_blocks = p.stream ? a.c.kv_heads * a.waves / (p.block / 32) : 0;
        const int64_t blocks = a.stream_blocks + p.blocks * p.splits * a.c.kv_heads;
        DT_REQUIRE(grid_fits(blocks, 2 * p.block), "dt_kv_attn: grid too large");
        const dim3 grid((unsigned)blocks), block(2 * p.block);
        const size_t lds = 2 * (size_t)(kTile * DP + DP * kTile) * 2;
        if (p.block == 256) {
            if (wide) hipLaunchKernelGGL((kv_rows_kernel<E, DP, true, 8>), grid, block, lds, st, a);
            else hipLaunchKernelGGL((kv_rows_kernel<E, DP, false, 8>), grid, block, lds, st, a);
        } else if (wide) {
            hipLaunchKernelGGL((kv_rows_kernel<E, DP, true, 4>), grid, block, lds, st, a);
        } else if constexpr (sizeof(E) == 2) {
            hipLaunchKernelGGL((kv_rows_kernel<E, DP, false, 4>), grid, block, lds, st, a);
        }
    } else {
        const dim3 grid((unsigned)(a.c.kv_heads * (a.waves / 4)));
        if (wide) hipLaunchKernelGGL((kv_stream_kernel<E, DP, true>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((kv_stream_kernel<E, DP, false>), grid, dim3(256), 0, st, a);
    }
    const int rc = check_launch("dt_kv_attn");
    if (rc || join_blocks + ranges == 0) return rc;
    a.join_blocks = (int32_t)join_blocks;
    const dim3 grid((unsigned)(join_blocks + ranges));
    if (joined <= 1024) hipLaunchKernelGGL((kv_join_kernel<E, DP, 256>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((kv_join_kernel<E, DP, 64>), grid, dim3(256), 0, st, a);
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
    const Plan p = plan(c, s, heads, cu_count());
    return (size_t)(p.floats + p.row_floats) * sizeof(float);
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
    const Plan p = plan(a.c, a.s, heads, cu_count());
    const size_t need = (size_t)(p.floats + p.row_floats) * sizeof(float);
    DT_REQUIRE(need == 0 || (workspace && aligned16(workspace) && workspace_bytes >= need),
               "%s: a 16-byte aligned workspace of %lld bytes is needed", who, (long long)need);
    DT_REQUIRE((p.blocks + 1) * p.splits * a.c.kv_heads < (1ll << 30) &&
                   ((int64_t)a.s.rows * (heads / a.c.kv_heads) / kRows + a.s.seqs) * a.c.kv_heads < (1ll << 31) && (int64_t)a.s.seqs * a.c.kv_heads * kFew < (1ll << 31),
               "%s: grid too large", who);
    // A row's q is read by the waves of its block alone, and o is stored where they all have it: o may be q.
    const int64_t sizes[2] = {a.s.rows, heads};
    const Strided q_rows(q, 2, 2, sizes, q_strides, a.c.dim), o_rows(o, 2, 2, sizes, o_strides, a.c.dim);
    DT_REQUIRE(o_rows.same_as(q_rows) || !share_memory(o_rows, q_rows), "%s: o is partly q", who);
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
    a.scale_log2 = scale * attn::kLog2e > FLT_MIN ? scale * attn::kLog2e : FLT_MIN;
    a.few = p.few;
    a.splits = p.splits;
    a.waves = p.waves;
    a.part_o = (float*)workspace;
    a.part_ml = a.part_o + (int64_t)a.c.kv_heads * p.waves * 2 * kRows * p.dp;
    a.rows_o = a.part_o + p.floats;
    a.rows_ml = a.rows_o + (int64_t)p.splits * a.s.rows * heads * p.dp;
    const hipStream_t st = (hipStream_t)stream;
    if (a.c.k_scale) return p.dp == 64 ? launch<e4m3, 64>(a, p, st) : launch<e4m3, 128>(a, p, st);
    return p.dp == 64 ? launch<bf16, 64>(a, p, st) : launch<bf16, 128>(a, p, st);
}
