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
    int32_t units, per_pass, slots;  // 16-element units a row; tokens a pass of 256 threads; heads side by side in a wave
    FastDiv unit_div;
    int32_t kv_blocks;               // workgroups before q's
    int32_t q_chunks;                // waves a row of q
    FastDiv head_div, chunk_div;
    int32_t lds_row;                 // elements a dim's row of v takes in LDS
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

// A value times 2^shift as an e4m3 code's input: NaN unless finite.
__device__ __forceinline__ float scaled(float x, int shift) {
    return finite(x) ? __builtin_amdgcn_ldexpf(x, shift) : __builtin_nanf("");
}

// Codes times 2^shift, rounded again.
__device__ __forceinline__ uint32_t again(uint32_t w, int shift) {
    float v[4];
    from_e4m3x4(w, v);
    return to_e4m3x4(__builtin_amdgcn_ldexpf(v[0], shift), __builtin_amdgcn_ldexpf(v[1], shift),
                     __builtin_amdgcn_ldexpf(v[2], shift), __builtin_amdgcn_ldexpf(v[3], shift));
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, float* v) {
#pragma unroll
    for (int n = 0; n < 8 / Io<T>::EPV; ++n) Io<T>::load(p + n * Io<T>::EPV, v + n * Io<T>::EPV);
}

template <typename T>
__device__ void rotate_q(const Args& a) {
    const uint32_t wave = (blockIdx.x - a.kv_blocks) * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int row = (int)fdiv(wave, a.chunk_div), chunk = (int)(wave - (uint32_t)row * a.q_chunks);
    if (row >= a.s.rows) return;
    const int b = find_seq(a.s, row, [](int start, int) { return start; });
    if (b < 0) return;
    const Seq q(a.s, b);
    if (row - q.row >= q.n) return;
    const int slot = (int)fdiv(lane, a.unit_div), u = (int)lane - slot * a.units;
    if (slot >= a.slots) return;
    const int p = a.pos ? a.pos[row] : q.past + row - q.row;
    const rotary::Unit at(u, a.rot, a.half);
    constexpr int ITER = 4;
    const int first = chunk * ITER * a.slots + slot;
    float v[ITER][16];
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        const int h = first + i * a.slots;
        if (h >= a.heads) continue;
        const T* x = reinterpret_cast<const T*>(a.q) + row * a.qs[0] + h * a.qs[1];
        load8(x + at.a, v[i]);
        load8(x + at.b, v[i] + 8);
    }
    rotary::Angles<float> w;
    w.set(p, a.freq, u, a.rot, a.mul);
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
        const int h = first + i * a.slots;
        if (h >= a.heads) continue;
        w.turn(v[i], u, a.rot, a.half, 1.f);
        T* y = reinterpret_cast<T*>(a.q_out) + row * a.os[0] + h * a.os[1];
#pragma unroll
        for (int n = 0; n < 8 / Io<T>::EPV; ++n) {
            Io<T>::store(y + at.a + n * Io<T>::EPV, v[i] + n * Io<T>::EPV);
            Io<T>::store(y + at.b + n * Io<T>::EPV, v[i] + 8 + n * Io<T>::EPV);
        }
    }
}

// NP passes hold a page.
template <typename T, typename E, int NP>
__global__ __launch_bounds__(256) void kv_append_kernel(const Args a) {
    constexpr bool F8 = sizeof(E) == 1;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];  // v: [dim][lds_row] elements
    __shared__ float most_of[4];
    if ((int)blockIdx.x >= a.kv_blocks) {
        rotate_q<T>(a);
        return;
    }
    // Workgroup: (number of a page, head, k or v), heads innermost: they share rows.
    const int tid = threadIdx.x, wave = tid >> 6;
    const bool is_v = blockIdx.x & 1;
    const int item = (int)fdiv(blockIdx.x >> 1, a.head_div), h = (int)(blockIdx.x >> 1) - item * a.c.kv_heads;
    const int page = 1 << a.c.page_log2, dim = a.c.dim;
    const int b = find_seq(a.s, item, [&a](int start, int i) { return first_item(a.s, start, i); });
    if (b < 0) return;
    const Seq q(a.s, b);
    PageItem it;
    if (!page_item(a.s, q, b, item, &it)) return;
    const int first = it.first, last = it.last;

    const int t0 = (int)fdiv((uint32_t)tid, a.unit_div), u = tid - t0 * a.units;
    const rotary::Unit at(u, is_v ? 0 : a.rot, a.half);
    const T* src = reinterpret_cast<const T*>(is_v ? a.v : a.k) + h * (is_v ? a.vs[1] : a.ks[1]);
    const int64_t stride = is_v ? a.vs[0] : a.ks[0];
    const int row0 = q.row + it.begin - q.past;  // of the page's token 0 (there may be none)
    float v[NP][16];
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int t = first + i * a.per_pass + t0;
        if (t0 >= a.per_pass || t >= last) continue;
        const T* x = src + (int64_t)(row0 + t) * stride;
        load8(x + at.a, v[i]);
        load8(x + at.b, v[i] + 8);
    }
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int t = first + i * a.per_pass + t0;
        if (t0 >= a.per_pass || t >= last) continue;
        if (!is_v && 16 * u < a.rot) {
            rotary::Angles<double> w;
            w.set(a.pos ? a.pos[row0 + t] : it.begin + t, a.freq, u, a.rot, (double)a.mul);
            double d[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) d[e] = (double)v[i][e];
            w.turn(d, u, a.rot, a.half, 1.0);
#pragma unroll
            for (int e = 0; e < 16; ++e) v[i][e] = to_odd(d[e]);
        }
        if constexpr (F8) {
#pragma unroll
            for (int e = 0; e < 16; ++e) most = fmaxf(most, finite(v[i][e]) ? fabsf(v[i][e]) : 0.f);
        }
    }

    uint8_t* const out = (is_v ? a.c.v : a.c.k) + ((int64_t)it.page * a.c.kv_heads + h) * a.c.head_bytes;
    int scale = kBias, grown = 0;  // grown: by how much the page's earlier codes shrink
    if constexpr (F8) {
        uint8_t* const held = (is_v ? a.c.v_scale : a.c.k_scale) + (int64_t)it.page * a.c.kv_heads + h;
#pragma unroll
        for (int o = 32; o; o >>= 1) most = fmaxf(most, __shfl_xor(most, o, 64));
        if ((tid & 63) == 0) most_of[wave] = most;
        const int before = first ? (int)*held : 0;
        __syncthreads();
        scale = scale_of(fmaxf(fmaxf(most_of[0], most_of[1]), fmaxf(most_of[2], most_of[3])));
        if (first) {
            if (scale > before) grown = scale - before;
            scale = max(scale, before);
        }
        if (tid == 0) *held = (uint8_t)scale;  // read by all before the barrier
    }

    if (!is_v) {
        if (grown)
            for (int i = tid; i < first * dim / 16; i += 256) {
                uint4 w = *reinterpret_cast<const uint4*>(out + 16 * i);
                w.x = again(w.x, -grown);
                w.y = again(w.y, -grown);
                w.z = again(w.z, -grown);
                w.w = again(w.w, -grown);
                *reinterpret_cast<uint4*>(out + 16 * i) = w;
            }
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int t = first + i * a.per_pass + t0;
            if (t0 >= a.per_pass || t >= last) continue;
#pragma unroll
            for (int run = 0; run < 2; ++run) {
                const float* x = v[i] + 8 * run;
                uint8_t* y = out + ((int64_t)t * dim + (run ? at.b : at.a)) * sizeof(E);
                if constexpr (F8) {
                    float c[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) c[e] = scaled(x[e], kBias - scale);
                    *reinterpret_cast<uint2*>(y) = make_uint2(to_e4m3x4(c[0], c[1], c[2], c[3]), to_e4m3x4(c[4], c[5], c[6], c[7]));
                } else {
                    *reinterpret_cast<uint4*>(y) = Io<bf16>::pack(x);
                }
            }
        }
        return;
    }

    // v: codes to LDS by (dim, token), then whole 16-byte pieces of a dim's row.
    E* const turned = reinterpret_cast<E*>(lds);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int t = first + i * a.per_pass + t0;
        if (t0 >= a.per_pass || t >= last) continue;
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            if constexpr (F8) {
                const uint32_t w = to_e4m3x4(scaled(v[i][e], kBias - scale), scaled(v[i][e + 1], kBias - scale),
                                             scaled(v[i][e + 2], kBias - scale), scaled(v[i][e + 3], kBias - scale));
#pragma unroll
                for (int n = 0; n < 4; ++n) turned[(16 * u + e + n) * a.lds_row + t].bits = (uint8_t)(w >> (8 * n));
            } else {
#pragma unroll
                for (int n = 0; n < 4; ++n) Io<bf16>::put((bf16*)turned + (16 * u + e + n) * a.lds_row + t, v[i][e + n]);
            }
        }
    }
    __syncthreads();
    constexpr int PER = 16 / sizeof(E);  // tokens of a piece
    const int pieces = page / PER;       // of a row: a power of two
    for (int i = tid; i < dim * pieces; i += 256) {
        const int d = i / pieces, c = (i & (pieces - 1)) * PER;
        if (c >= last || (c + PER <= first && !grown)) continue;
        uint8_t* y = out + ((int64_t)d * page + c) * sizeof(E);
        const E* x = turned + d * a.lds_row + c;
        if (c >= first && c + PER <= last) {
            *reinterpret_cast<uint4*>(y) = *reinterpret_cast<const uint4*>(x);
            continue;
        }
        if constexpr (F8) {
            if (grown && c < first) {
                // Earlier tokens of the piece again; those that are not this call's stay.
                for (int n = 0; n < 4; ++n) {
                    if (c + 4 * n >= first) break;
                    const uint32_t w = reinterpret_cast<const uint32_t*>(y)[n], s = again(w, -grown);
                    const int left = first - c - 4 * n;
                    const uint32_t m = left >= 4 ? ~0u : (1u << (8 * left)) - 1;
                    reinterpret_cast<uint32_t*>(y)[n] = (s & m) | (w & ~m);
                }
            }
        }
        for (int n = max(first - c, 0); n < min(last - c, PER); ++n) reinterpret_cast<E*>(y)[n] = x[n];
    }
}

template <typename T, typename E>
int launch(const Args& a, int passes, dim3 grid, hipStream_t st) {
    const size_t lds = (size_t)a.c.dim * a.lds_row * sizeof(E);
    if (passes <= 1) hipLaunchKernelGGL((kv_append_kernel<T, E, 1>), grid, dim3(256), lds, st, a);
    else if (passes <= 2) hipLaunchKernelGGL((kv_append_kernel<T, E, 2>), grid, dim3(256), lds, st, a);
    else if (passes <= 4) hipLaunchKernelGGL((kv_append_kernel<T, E, 4>), grid, dim3(256), lds, st, a);
    else hipLaunchKernelGGL((kv_append_kernel<T, E, 8>), grid, dim3(256), lds, st, a);
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
    DT_REQUIRE(y->table_pages >= 0 && y->table_pages * x->page <= (1ll << 30), "%s: a table of %lld pages is too long", who,
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
    if (x->rotary) {
        rc = rotary::check_rotary(*x->rotary, a.c.dim, who);
        if (rc) return rc;
        DT_REQUIRE(!x->rotary->half || x->rotary->rot_dims % 16 == 0, "%s: halves of %lld dims unsupported (a multiple of 16)", who,
                   (long long)x->rotary->rot_dims);
        a.freq = x->rotary->freq;
        a.mul = x->rotary->attn_factor;
        a.rot = (int32_t)x->rotary->rot_dims;
        a.half = x->rotary->half != 0;
    }
    DT_REQUIRE(((uintptr_t)x->pos & 3) == 0, "%s: pos must be 4-byte aligned", who);
    if (a.s.rows == 0 || a.s.seqs == 0) return DT_OK;
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
    a.per_pass = 256 / a.units;
    a.slots = 64 / a.units;
    a.unit_div = make_fastdiv((uint32_t)a.units);
    a.head_div = make_fastdiv((uint32_t)a.c.kv_heads);
    a.q_chunks = turn_q ? (a.heads + 4 * a.slots - 1) / (4 * a.slots) : 1;
    a.chunk_div = make_fastdiv((uint32_t)a.q_chunks);
    const int64_t page = 1ll << a.c.page_log2;
    const bool f8 = a.c.k_scale != nullptr;
    a.lds_row = (int32_t)page + 16 / (f8 ? 1 : 2);
    const int64_t kv_blocks = items(a.s) * a.c.kv_heads * 2;
    const int64_t q_blocks = turn_q ? ((int64_t)a.s.rows * a.q_chunks + 3) / 4 : 0;
    DT_REQUIRE(kv_blocks + q_blocks < (1ll << 31) && (int64_t)a.s.rows * a.q_chunks < (1ll << 31), "%s: grid too large", who);
    a.kv_blocks = (int32_t)kv_blocks;
    const dim3 grid((unsigned)(kv_blocks + q_blocks));
    const int passes = ((int)page + a.per_pass - 1) / a.per_pass;
    const hipStream_t st = (hipStream_t)stream;
    if (x->io_type == DT_TYPE_F32)
        return f8 ? launch<float, e4m3>(a, passes, grid, st) : launch<float, bf16>(a, passes, grid, st);
    return f8 ? launch<bf16, e4m3>(a, passes, grid, st) : launch<bf16, bf16>(a, passes, grid, st);
}
