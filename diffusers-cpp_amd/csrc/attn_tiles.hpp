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
    int32_t side, two_sided, reach;  // buckets a side; reach = start[side - 1]: one bucket from there on
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
// bf16 anyway: each term is off by half a step at most, 2^-8 of itself, as the stored
// result is; sums over them stay fp32).
__device__ __forceinline__ void to_frag(const float (&p)[8], bf16x8_t& f) {
    f = __builtin_bit_cast(bf16x8_t, make_uint4(pack_bf16x2(p[0], p[1]), pack_bf16x2(p[2], p[3]),
                                                pack_bf16x2(p[4], p[5]), pack_bf16x2(p[6], p[7])));
}
__device__ __forceinline__ void to_frag(const float (&p)[8], Elem<float>::Frag& f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f.v[e] = p[e];
}

template <typename T>
__device__ __forceinline__ void acc_frag(const f32x16_t& p, int j, typename Elem<T>::Frag& f) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = p[8 * j + e];
    to_frag(v, f);
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

    // ROWS rows by NW waves (this one is `wave`) as buffer loads to LDS: a scalar base
    // per tile, the lane's rows and chunks as 32-bit offsets for all tiles.  An offset out of
    // the buffer's range gives zeros: chunks past the head width, and rows that are not
    // kept (keep), whose values then reach no product (a mask may hide NaN, a tail
    // lies outside the tensor).
    template <int ROWS, int NW>
    struct Loads {
        static constexpr int J = ROWS * CPR / 64 / NW;
        static_assert(J >= 1 && ROWS * CPR % (64 * NW) == 0, "tile");
        uint32_t at[J];

        __device__ __forceinline__ void init(int64_t stride, int dim, int wave, int lane) {
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const int i = (wave * J + j) * 64 + lane, r = i / CPR, c = (i % CPR) ^ swz(r);
                at[j] = c * Elem<T>::EPC < dim ? (uint32_t)((r * stride + c * Elem<T>::EPC) * (int64_t)sizeof(T)) : kOutOfBuffer;
            }
        }
        __device__ __forceinline__ static int row(int wave, int lane, int j) { return ((wave * J + j) * 64 + lane) / CPR; }

        // base: the tile's first row.
        __device__ __forceinline__ void issue_all(const T* base, uint8_t* lds, int wave) const {
#pragma unroll
            for (int j = 0; j < J; ++j) lds_dma16(base, at[j], lds + (wave * J + j) * 1024);
        }
        template <typename Keep>
        __device__ __forceinline__ void issue(const T* base, uint8_t* lds, int wave, int lane, Keep keep) const {
#pragma unroll
            for (int j = 0; j < J; ++j) lds_dma16(base, keep(row(wave, lane, j)) ? at[j] : kOutOfBuffer, lds + (wave * J + j) * 1024);
        }
    };
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

// N products whose first operands come from LDS: read(i) gives one, mul(i, f) uses it, and
// side(n, of) is other work for the n-th of `of` parts, of V vector instructions for each
// product (0: none).  bf16 reads four operands ahead, R LDS instructions each, while the
// four before are multiplied, and spreads the other work between the products: left alone
// the compiler reads each operand right before its product, into the same registers, and
// every product waits for LDS.  An fp32 operand lasts eight instructions of 64 cycles: it is
// read when it is needed.
struct NoSide {
    __device__ __forceinline__ void operator()(int, int) const {}
};
template <typename T, int N, int R, int V = 0, typename Read, typename Mul, typename Side = NoSide>
__device__ __forceinline__ void products(Read read, Mul mul, Side side = Side{}) {
    constexpr int G = 4;
    static_assert(N % G == 0, "groups");
    if constexpr (sizeof(T) == 2) {
        typename Elem<T>::Frag f[2][G];
#pragma unroll
        for (int i = 0; i < G; ++i) f[0][i] = read(i);
#pragma unroll
        for (int n = 0; n < N / G; ++n) {
            if (n + 1 < N / G) {
#pragma unroll
                for (int i = 0; i < G; ++i) f[(n + 1) & 1][i] = read((n + 1) * G + i);
            }
#pragma unroll
            for (int i = 0; i < G; ++i) mul(n * G + i, f[n & 1][i]);
            side(n, N / G);
            if (n == 0) __builtin_amdgcn_sched_group_barrier(0x100, R * G, 0);
            if constexpr (V == 0) {
                __builtin_amdgcn_sched_group_barrier(0x100, R * G, 0);  // LDS reads
                __builtin_amdgcn_sched_group_barrier(0x008, G, 0);      // MFMA
            } else {
#pragma unroll
                for (int i = 0; i < G; ++i) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x100, R, 0);
                    __builtin_amdgcn_sched_group_barrier(0x402, V, 0);  // vector and transcendental ALU
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            mul(i, read(i));
            if (i % G == G - 1) side(i / G, N / G);
        }
    }
}

// An operand put together from four accumulator elements at a time (see to_frag).
template <typename T> struct FragParts;
template <> struct FragParts<bf16> {
    uint32_t w[4];
    __device__ __forceinline__ void set(int half, const float (&v)[4]) {
        w[2 * half] = pack_bf16x2(v[0], v[1]);
        w[2 * half + 1] = pack_bf16x2(v[2], v[3]);
    }
    __device__ __forceinline__ bf16x8_t frag() const { return __builtin_bit_cast(bf16x8_t, make_uint4(w[0], w[1], w[2], w[3])); }
};
template <> struct FragParts<float> {
    Elem<float>::Frag f;
    __device__ __forceinline__ void set(int half, const float (&v)[4]) {
#pragma unroll
        for (int e = 0; e < 4; ++e) f.v[4 * half + e] = v[e];
    }
    __device__ __forceinline__ const Elem<float>::Frag& frag() const { return f; }
};

// The other lane half's value (lane ^ 32).
__device__ __forceinline__ float swap32(float v) {
    const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float((threadIdx.x & 32) ? p[0] : p[1]);
}

// ---- kept keys --------------------------------------------------------------------
__device__ __forceinline__ int kept_len(const AttnIn& a, int b) {
    int n = a.seq_kv;
    if (a.kv_len) n = min(max(a.kv_len[b], 0), n);
    return n;
}

// Walks the tiles of N keys (32, 64 or 128) that hold a kept key, from `t` on by
// `step` to `end`, the mask bytes of the tile after read ahead.  Uniform in the wave.
template <int N>
struct Kept {
    static constexpr int W = (N + 63) / 64;
    const uint8_t* mask;
    int len, t, end, step;
    uint32_t ahead[W];  // mask byte of key N t + 64 w + lane
    uint64_t word[W];   // kept keys of the tile next() returned

    __device__ __forceinline__ void fetch(int lane) {
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const int key = t * N + 64 * w + lane;
            ahead[w] = t < end && (N >= 64 || lane < N) && key < len ? (mask ? mask[key] : 1u) : 0u;
        }
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
            uint64_t any = 0;
#pragma unroll
            for (int w = 0; w < W; ++w) any |= word[w] = __builtin_amdgcn_ballot_w64(ahead[w] != 0);
            const int at = t;
            t += step;
            fetch(lane);
            if (any) return at;
        }
        return -1;
    }
};
template <int N>
__device__ __forceinline__ bool all_kept(const uint64_t (&word)[(N + 63) / 64]) {
    if constexpr (N == 32) return (uint32_t)word[0] == 0xFFFFFFFFu;
    if constexpr (N == 64) return word[0] == ~0ull;
    return (word[0] & word[N / 64 - 1]) == ~0ull;
}
template <int W>
__device__ __forceinline__ bool kept_row(const uint64_t (&word)[W], int r) {
    return ((W == 1 || r < 64 ? word[0] : word[W - 1]) >> (r & 63)) & 1;
}

// ---- bias -------------------------------------------------------------------------
// Offset key - query to its bucket.
__device__ __forceinline__ int rel_bucket(const RelArgs& r, int off) {
    const int dist = off > 0 ? (r.two_sided ? off : 0) : -off;
    int t = 0;
    for (int i = 1; i < r.side; ++i) t += dist >= r.start[i];
    return t + (r.two_sided && off > 0 ? r.side : 0);
}
// line[reach + kMargin + off] = the bias of that offset in units of log2, for one head.  The
// margins are what a 32 x 32 block with some |offset| < reach can have beyond it: no offset
// is clamped.
constexpr int kMargin = 62;
__host__ __device__ inline int rel_line_len(int reach) { return 2 * (reach + kMargin) + 1; }
__device__ __forceinline__ void rel_line(const RelArgs& r, int head, float* line, int tid, int threads) {
    const int mid = r.reach + kMargin;
    for (int i = tid; i < 2 * mid + 1; i += threads)
        line[i] = r.table[rel_bucket(r, i - mid) * r.table_stride + head] * kLog2e;
}
inline int rel_line_floats(const RelArgs& r) { return r.table ? rel_line_len(r.reach) : 0; }
// Where a lane reads the bias of offsets lo + {0 .. 27}: in a block out of reach the end of the
// line on its side, which holds one value.
__device__ __forceinline__ const float* rel_at(const float* line, int reach, int lo) {
    const int mid = reach + kMargin;
    return line + mid + min(max(lo, -mid), mid - 27);
}
// Position of query 0 of batch entry b.  Positions far from every key differ only in
// being far: the bound keeps offsets in 32 bits.
__device__ __forceinline__ int rel_position(const RelArgs& r, int b) {
    return r.table && r.q_pos ? min(max(r.q_pos[b], -(1 << 29)), 1 << 29) : 0;
}

// ---- host ---------------------------------------------------------------------------
constexpr int64_t kMaxSeq = 1 << 28;
constexpr int64_t kMaxRowBytes = (1 << 24) - 256;  // a tile's 128 rows stay below kOutOfBuffer bytes
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
