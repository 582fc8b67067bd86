// kv_cache.hpp -- the paged key/value cache as its kernels see it (kv_cache.hip,
// kv_attention.hip), e4m3 conversions, and the search for a row's sequence.
#pragma once

#include "capi_util.hpp"
#include "common.hpp"
#include "kv_index.hpp"

namespace dit {
namespace kv {

struct e4m3 {
    uint8_t bits;
};

struct Cache {
    uint8_t* k;
    uint8_t* v;
    uint8_t* k_scale;  // null: bf16
    uint8_t* v_scale;
    int32_t kv_heads, page_log2, dim;
    int64_t head_bytes;  // one page of one head: page * dim elements
};

// The last of the sequences b with key(seq_start[b], b) <= x, or -1: with ascending keys, the one
// that x belongs to.  Its description as well, from lanes that read all of it at once: a load's wait
// less than to look the sequence up after it is known.  By a whole wave.
struct Found {
    int b = -1, start = 0, end = 0, past = 0;
    __device__ __forceinline__ Seq seq(const Seqs& s) const { return Seq(s, start, end, past); }
};
template <typename Key>
__device__ __forceinline__ Found find_seq(const Seqs& s, int64_t x, Key key) {
    const int lane = threadIdx.x & 63;
    Found f;
    for (int b0 = 0; b0 < s.seqs; b0 += 64) {
        const int b = min(b0 + lane, s.seqs - 1);
        const int start = s.seq_start[b], end = s.seq_start[b + 1], past = s.past[b];
        const int n = __popcll(__builtin_amdgcn_ballot_w64(b0 + lane < s.seqs && key(clamped(start, 0, s.rows), b) <= x));
        if (n == 0) break;
        f.b = b0 + n - 1;
        f.start = __builtin_amdgcn_readlane(start, n - 1);
        f.end = __builtin_amdgcn_readlane(end, n - 1);
        f.past = __builtin_amdgcn_readlane(past, n - 1);
    }
    return f;
}

// ---- e4m3: four bits of significand, 2^-9 to 448, NaN but no infinity --------------------
typedef float f32x2_t __attribute__((ext_vector_type(2)));

// Four values over `scale` (a power of two; at most 448 then, or NaN) to codes, to nearest even.
typedef short s16x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t to_e4m3x4(float a, float b, float c, float d, float scale) {
    s16x2_t w = {0, 0};
    w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, a, b, scale, false);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, c, d, scale, true);
    return __builtin_bit_cast(uint32_t, w);
}
__device__ __forceinline__ void from_e4m3x4(uint32_t w, float (&v)[4]) {
    const f32x2_t a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    v[0] = a[0];
    v[1] = a[1];
    v[2] = b[0];
    v[3] = b[1];
}

// ---- host -------------------------------------------------------------------------------
// Checks the descriptions and fills the kernels' own (kv_cache.hip).
int prepare(const dt_kv_cache* cache, const dt_kv_seqs* seqs, const char* who, Cache* c, Seqs* s);
// Rows of heads * dim elements of `es` bytes, strides {row, head}: `out`: no element twice.
int check_rows(const void* p, const int64_t* strides, int64_t rows, int64_t heads, int64_t dim, int es, bool out,
               const char* name, const char* who);

}  // namespace kv

namespace rotary {
int check_rotary(const dt_rotary& r, int64_t head_dim, const char* who);  // rotary.hip
}

}  // namespace dit
