// attn_tiles.hpp -- the pieces shared by the masked attention kernels
// (cross_attention.hip, cross_attention_bwd.hip): arguments, LDS tiles of rows
// filled by direct DMA, the two ways an MFMA operand is read from a tile, the
// words that say which keys of a tile are kept, and the bias line of a head.
//
// Everything is written for one 32 x 32 block of a product with 16 terms of the
// reduction per step: lane l supplies 8 of them (8 (l / 32) + e) of operand row
// l % 32, and holds rows 8 (i / 4) + 4 (l / 32) + i % 4 of column l % 32 in
// accumulator element i.  bf16: one v_mfma_f32_32x32x16_bf16.  fp32: eight
// v_mfma_f32_32x32x2_f32 of the same 8 elements (term e of both lane halves
// per instruction), so operands are exact and sums are fp32 in both types.
#pragma once

#include "capi_util.hpp"
#include "common.hpp"

namespace dit {
namespace attn {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kMaxSide = 64;          // buckets of one side of the bias
constexpr int kMaxDistance = 1024;    // offset from which one bucket takes all

// Relative position bias: bucket thresholds of one side, start[t] = the least
// distance of bucket t.
struct RelArgs {
    const float* table;   // [buckets][heads]; null: no bias
    int64_t table_stride;
    const int32_t* q_pos;  // position of query 0 per batch entry, or null (0)
    int32_t side, two_sided, reach;  // buckets a side; reach = start[side - 1], offsets are clamped to it
    int32_t start[kMaxSide];
};

struct AttnIn {
    const void* q;
    const void* k;
    const void* v;
    int64_t qs[3], ks[3], vs[3];  // batch, token, head strides (elements)
    int32_t batch, heads, kv_heads, shared, seq_q, seq_kv, dim;
    const int32_t* kv_len;        // kept keys are those below kv_len[b] ...
    const uint8_t* kv_mask;       // ... with kv_mask[b * mask_stride + j] != 0 (either may be null)
    int64_t mask_stride;
    float scale, scale_log2;
    RelArgs rel;
};

template <typename T> struct Elem;
template <> struct Elem<bf16> {
    typedef bf16x8_t Frag;
    static constexpr int EPC = 8;  // elements of a 16-byte chunk
};
template <> struct Elem<float> {
    struct Frag {
        float v[8];
    };
    static constexpr int EPC = 4;
};

__device__ __forceinline__ f32x16_t zero16() {
    f32x16_t z;
#pragma unroll
    for (int e = 0; e < 16; ++e) z[e] = 0.f;
    return z;
}

__device__ __forceinline__ f32x16_t mma(const bf16x8_t& a, const bf16x8_t& b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16_t mma(const Elem<float>::Frag& a, const Elem<float>::Frag& b, f32x16_t c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[e], b.v[e], c, 0, 0, 0);
    return c;
}

// Accumulator elements 8 j .. 8 j + 7 as the second operand of a product whose
// terms are the accumulator's rows.  bf16 rounds them (the products' inputs are
// bf16 anyway: each term is off by half a step, 2^-9 of itself, as the stored
// result is; sums over them stay fp32).
__device__ __forceinline__ void to_frag(const float (&p)[8], bf16x8_t& f) {
    f = __builtin_bit_cast(bf16x8_t, make_uint4(pack_bf16x2(p[0], p[1]), pack_bf16x2(p[2], p[3]),
                                                pack_bf16x2(p[4], p[5]), pack_bf16x2(p[6], p[7])));
}
__device__ __forceinline__ void to_frag(const float (&p)[8], Elem<float>::Frag& f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f.v[e] = p[e];
}

__device__ __forceinline__ float frag_dot(const bf16x8_t& a, const bf16x8_t& b) {
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) s = __builtin_fmaf((float)a[e], (float)b[e], s);
    return s;
}
__device__ __forceinline__ float frag_dot(const Elem<float>::Frag& a, const Elem<float>::Frag& b) {
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) s = __builtin_fmaf(a.v[e], b.v[e], s);
    return s;
}

// Four consecutive elements of a row.
__device__ __forceinline__ void put4(float* p, const float (&v)[4]) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void put4(bf16* p, const float (&v)[4]) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
}

// Elements 16 c + 8 g .. + 7 of a row in global memory; zeros past the head width.
template <typename T>
__device__ __forceinline__ typename Elem<T>::Frag frag_global(const T* row, int c, int g, int dim) {
    uint4 u[Elem<T>::EPC == 8 ? 1 : 2];
    const int d = 16 * c + 8 * g;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(u) / 16); ++i)
        u[i] = d < dim ? *reinterpret_cast<const uint4*>(row + d + 4 * i) : make_uint4(0, 0, 0, 0);
    typename Elem<T>::Frag f;
    __builtin_memcpy(&f, u, sizeof(f));
    return f;
}

template <typename T>
__device__ __forceinline__ typename Elem<T>::Frag frag_zero() {
    uint4 u[Elem<T>::EPC == 8 ? 1 : 2];
#pragma unroll
    for (int i = 0; i < (int)(sizeof(u) / 16); ++i) u[i] = make_uint4(0, 0, 0, 0);
    typename Elem<T>::Frag f;
    __builtin_memcpy(&f, u, sizeof(f));
    return f;
}

template <int N_OUT>
__device__ __forceinline__ void wait_vmem() {
    __builtin_amdgcn_s_waitcnt((N_OUT & 15) | ((N_OUT >> 4) << 14) | 0x0F70);
}
__device__ __forceinline__ void wait_lds() { __builtin_amdgcn_s_waitcnt(0xC07F); }

typedef short short4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) short4_t* lds_short4_p;
__device__ __forceinline__ uint2 read_tr16(const uint8_t* p) {
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4_p)(p)));
}

// Rows of DP elements in LDS.  Chunk c (16 bytes) of row r lies at chunk c ^
// swz(r): row operands (32 rows, one chunk each) and column operands (4 rows x
// 64 bytes per transposed read) both spread over all banks.
template <typename T, int DP>
struct Tile {
    typedef typename Elem<T>::Frag Frag;
    static constexpr int RB = DP * (int)sizeof(T), CPR = RB / 16, STEPS = DP / 16, BLOCKS = DP / 32;
    static_assert(CPR >= 8, "row");

    __device__ __forceinline__ static int swz(int r) {
        return CPR == 8 ? (((r >> 1) & 1) << 2) | ((r >> 2) & 3) : ((r & 3) << 2) | ((r >> 2) & 3);
    }

    // ROWS rows by NW waves (this one is `wave`): row(r) gives the source row.
    // Chunks past the head width are not written: the tile is cleared once
    // before its first use (clear()).
    template <int ROWS, int NW, typename Row>
    __device__ __forceinline__ static void load(const T* src, int64_t stride, int dim, uint8_t* lds, int wave, int lane,
                                                Row row) {
        constexpr int J = ROWS * CPR / 64 / NW;
        static_assert(J >= 1 && ROWS * CPR % (64 * NW) == 0, "tile");
        const int chunks = dim / Elem<T>::EPC;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int at = (wave * J + j) * 64, r = (at + lane) / CPR, c = ((at + lane) % CPR) ^ swz(r);
            const T* p = src + (int64_t)row(r) * stride + c * Elem<T>::EPC;
            if (chunks == CPR || c < chunks) __builtin_amdgcn_global_load_lds(p, lds + at * 16, 16, 0, 0);
        }
    }

    __device__ __forceinline__ static void clear(uint8_t* lds, int bytes, int tid, int threads) {
        for (int i = tid * 16; i < bytes; i += threads * 16) *reinterpret_cast<uint4*>(lds + i) = make_uint4(0, 0, 0, 0);
    }

    // Row operand: elements 16 c + 8 g .. + 7 of row r.
    __device__ __forceinline__ static Frag row_frag(const uint8_t* t, int r, int c, int g) {
        Frag f;
        if constexpr (sizeof(T) == 2) {
            f = *reinterpret_cast<const bf16x8_t*>(t + r * RB + (((2 * c + g) ^ swz(r)) << 4));
        } else {
            const int c0 = 4 * c + 2 * g, s = swz(r);
            const uint4 a = *reinterpret_cast<const uint4*>(t + r * RB + ((c0 ^ s) << 4));
            const uint4 b = *reinterpret_cast<const uint4*>(t + r * RB + (((c0 + 1) ^ s) << 4));
            const uint4 u[2] = {a, b};
            __builtin_memcpy(&f, u, sizeof(f));
        }
        return f;
    }

    // Per-lane offsets of the column operand (see col_frag): [block][half].
    struct Cols {
        int at[sizeof(T) == 2 ? BLOCKS : 1][2];
    };
    __device__ __forceinline__ static Cols cols(int lane) {
        Cols o;
        const int g = lane >> 5;
        if constexpr (sizeof(T) == 2) {
            const int s16 = lane & 15, dsub = (lane >> 4) & 1, trow = s16 >> 2, tcol = 16 * dsub + 4 * (s16 & 3);
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int r = 8 * h + 4 * g + trow;
                    o.at[b][h] = r * RB + (((4 * b + (tcol >> 3)) ^ swz(r)) << 4) + 8 * ((tcol >> 2) & 1);
                }
        } else {
            o.at[0][0] = lane & 31;
            o.at[0][1] = g;
        }
        return o;
    }
    // Column operand: rows {r0 + 4 g + e, r0 + 8 + 4 g + e} (e < 4; r0 a multiple
    // of 16) of element 32 b + lane % 32 -- the rows an accumulator of 16 rows
    // holds in this lane.
    __device__ __forceinline__ static Frag col_frag(const uint8_t* t, int r0, int b, const Cols& o) {
        Frag f;
        if constexpr (sizeof(T) == 2) {
            const uint2 lo = read_tr16(t + r0 * RB + o.at[b][0]);
            const uint2 hi = read_tr16(t + r0 * RB + o.at[b][1]);
            f = __builtin_bit_cast(bf16x8_t, make_uint4(lo.x, lo.y, hi.x, hi.y));
        } else {
            const int l = o.at[0][0], g = o.at[0][1], c = 8 * b + (l >> 2);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = 8 * h + 4 * g + e;
                    f.v[4 * h + e] = *reinterpret_cast<const float*>(t + (r0 + r) * RB + ((c ^ swz(r)) << 4) + 4 * (l & 3));
                }
        }
        return f;
    }
};

// ---- kept keys --------------------------------------------------------------------
__device__ __forceinline__ int kept_len(const AttnIn& a, int b) {
    int n = a.seq_kv;
    if (a.kv_len) n = min(max(a.kv_len[b], 0), n);
    return n;
}

// Walks the tiles of N keys (32 or 64) that hold a kept key, from `t` on by
// `step` to `end`, the mask bytes of the tile after read ahead.  Uniform in the wave.
template <int N>
struct Kept {
    const uint8_t* mask;
    int len, t, end, step;
    uint32_t ahead;  // mask byte of key N t + lane
    uint64_t word;   // kept keys of the tile next() returned

    __device__ __forceinline__ void fetch(int lane) {
        const int key = t * N + lane;
        ahead = t < end && lane < N && key < len ? (mask ? mask[key] : 1u) : 0u;
    }
    __device__ __forceinline__ void start(const AttnIn& a, int b, int n, int first, int last, int by, int lane) {
        mask = a.kv_mask ? a.kv_mask + b * a.mask_stride : nullptr;
        len = n;
        t = first;
        end = min(last, (n + N - 1) / N);
        step = by;
        fetch(lane);
    }
    // The next tile with a kept key, or -1.
    __device__ __forceinline__ int next(int lane) {
        while (t < end) {
            word = __builtin_amdgcn_ballot_w64(ahead != 0);
            const int at = t;
            t += step;
            fetch(lane);
            if (word) return at;
        }
        return -1;
    }
};
template <int N>
__device__ __forceinline__ bool all_kept(uint64_t word) {
    return N == 64 ? word == ~0ull : (uint32_t)word == 0xFFFFFFFFu;
}
// Source row of tile row r: itself, or the tile's first kept row where it is not
// kept, whose values (a mask may hide NaN, a tail lies outside the tensor)
// then never reach a product.
__device__ __forceinline__ int kept_row(uint64_t word, int r) {
    return (word >> r) & 1 ? r : (int)__builtin_ctzll(word);
}

// ---- bias -------------------------------------------------------------------------
// Offset key - query, clamped to +-reach, to its bucket.
__device__ __forceinline__ int rel_bucket(const RelArgs& r, int off) {
    const int dist = off > 0 ? (r.two_sided ? off : 0) : -off;
    int t = 0;
    for (int i = 1; i < r.side; ++i) t += dist >= r.start[i];
    return t + (r.two_sided && off > 0 ? r.side : 0);
}
// line[reach + off] = the bias of that offset in units of log2, for one head.
__device__ __forceinline__ void rel_line(const RelArgs& r, int head, float* line, int tid, int threads) {
    for (int i = tid; i < 2 * r.reach + 1; i += threads)
        line[i] = r.table[rel_bucket(r, i - r.reach) * r.table_stride + head] * kLog2e;
}
inline int rel_line_floats(const RelArgs& r) { return r.table ? 2 * r.reach + 1 : 0; }
// Position of query 0 of batch entry b.  Positions far from every key differ only in
// being far: the bound keeps offsets in 32 bits.
__device__ __forceinline__ int rel_position(const RelArgs& r, int b) {
    return r.table && r.q_pos ? min(max(r.q_pos[b], -(1 << 29)), 1 << 29) : 0;
}

// ---- host ---------------------------------------------------------------------------
constexpr int64_t kMaxSeq = 1 << 28;
// Checks the shared arguments and fills `in` (cross_attention.hip).
int prepare_in(const dt_attn_args* args, const char* who, AttnIn* in);
// Checks one strided operand [batch][seq][heads][head_dim]; `out`: no element twice.
int check_rows(const dt_attn_args* args, const void* p, const int64_t* strides, int64_t heads, int64_t seq, bool out,
               const char* name, const char* who);

// XCD-contiguous block numbers: consecutive numbers run on one XCD (one L2).
__device__ __forceinline__ uint32_t xcd_block() {
    const uint32_t b = blockIdx.x, n = gridDim.x;
    return (n & 7u) == 0 ? (b & 7u) * (n >> 3) + (b >> 3) : b;
}

}  // namespace attn
}  // namespace dit
