// rotary.hip -- rotary positions of q and k in one launch, and their gradient (the
// rotation back): pair (x, y) -> (x c - y s, y c + x s), c = f cos(p w), s = f sin(p w).
//
// One pass: 16 bytes a lane and load.  A wave takes one token and up to ITER heads a lane;
// lane l holds two vectors of 16 bytes of every (64 / units)-th head, so the angles, which cost
// more than the rotation, are worked out once for ITER heads.
#include <math.h>

#include "capi_util.hpp"
#include "common.hpp"
#include "overlap.hpp"
#include "rotary.hpp"

namespace dit {
namespace rotary {
namespace {

struct Tensor {
    const void* x;
    void* y;
    int64_t xs[3], ys[3];  // batch, token, head strides
};

struct Args {
    Tensor t[2];
    int32_t heads[2];
    int32_t seq, dim, rot, half;
    FastDiv seq_div;
    int64_t rows;  // batch * seq
    const int32_t* pos;
    int64_t pos_stride;
    const float* freq;
    float mul, sign;
    int32_t units, slots, chunks;  // units of two vectors a head; heads side by side in a wave; waves a token
    FastDiv unit_div, chunk_div;
    uint32_t grid_x;
};

// Workgroups in lines of grid_x: one dimension of a launch holds less than 2^32 threads, and is cut short past that.
__device__ __forceinline__ uint32_t block_id(const Args& a) { return blockIdx.y * a.grid_x + blockIdx.x; }

template <typename T, int ITER>
__global__ __launch_bounds__(256) void rotary_kernel(const Args a) {
    const uint32_t wave = block_id(a) * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    const uint32_t row = fdiv(wave, a.chunk_div), chunk = wave - row * a.chunks;
    if (row >= (uint64_t)a.rows) return;
    const uint32_t slot = fdiv(lane, a.unit_div);
    const int u = lane - slot * a.units;
    if (slot >= (uint32_t)a.slots) return;
    const uint32_t b = fdiv(row, a.seq_div), tok = row - b * a.seq;
    const int p = a.pos[(int64_t)b * a.pos_stride + tok];
    const int first = (int)(chunk * ITER * a.slots + slot);

    // By value: a stride picked by its address would be a load.
    const Tensor q = a.t[0], k = a.t[1];
    auto at = [&](int i, int64_t qb, int64_t qt, int64_t qh, int64_t kb, int64_t kt, int64_t kh) {
        const int h = first + i * a.slots;
        const int64_t in_q = b * qb + tok * qt + h * qh, in_k = b * kb + tok * kt + (h - a.heads[0]) * kh;
        return h < a.heads[0] ? in_q : in_k;
    };
    auto is_q = [&](int i) { return first + i * a.slots < a.heads[0]; };
    turn_heads<T, ITER>(
        p, a.freq, u, a.units, a.rot, a.half, a.mul, a.sign, [&](int i) { return first + i * a.slots < a.heads[0] + a.heads[1]; },
        [&](int i) {
            return reinterpret_cast<const T*>(is_q(i) ? q.x : k.x) + at(i, q.xs[0], q.xs[1], q.xs[2], k.xs[0], k.xs[1], k.xs[2]);
        },
        [&](int i) {
            return reinterpret_cast<T*>(is_q(i) ? q.y : k.y) + at(i, q.ys[0], q.ys[1], q.ys[2], k.ys[0], k.ys[1], k.ys[2]);
        });
}

// Any width, part and alignment: a thread per pair, or per element behind the rotated part, each with the angle worked out anew
// and elements one by one (4096 tokens of 40 heads of 80, 20 turned, in halves, bf16: 62.9 us; 32 turned, by whole vectors, 14.1).
template <typename T>
__global__ __launch_bounds__(256) void rotary_any_kernel(const Args a) {
    const int items = a.rot / 2 + a.dim - a.rot, heads = a.heads[0] + a.heads[1];
    const int64_t id = (int64_t)block_id(a) * 256 + threadIdx.x;
    const int64_t row = id / ((int64_t)items * heads);
    if (row >= a.rows) return;
    const int rest = (int)(id - row * items * heads);
    int h = rest / items;
    const int i = rest - h * items;
    const int64_t b = row / a.seq, tok = row - b * a.seq;
    const bool k = h >= a.heads[0];
    if (k) h -= a.heads[0];
    const Tensor& t = a.t[k ? 1 : 0];
    const T* x = reinterpret_cast<const T*>(t.x) + b * t.xs[0] + tok * t.xs[1] + h * t.xs[2];
    T* y = reinterpret_cast<T*>(t.y) + b * t.ys[0] + tok * t.ys[1] + h * t.ys[2];
    if (i >= a.rot / 2) {
        const int d = i + a.rot / 2;
        y[d] = x[d];
        return;
    }
    float c, s;
    cos_sin(a.pos[b * a.pos_stride + tok], a.freq[i], a.mul, &c, &s);
    s *= a.sign;
    const int d0 = a.half ? i : 2 * i, d1 = a.half ? i + a.rot / 2 : 2 * i + 1;
    const float u = Io<T>::get(x + d0), v = Io<T>::get(x + d1);
    Io<T>::put(y + d0, u * c - v * s);
    Io<T>::put(y + d1, v * c + u * s);
}

// `blocks` workgroups of 256 threads in lines of equal length.
dim3 lines_of(int64_t blocks, Args* a) {
    const int64_t lines = (blocks + (1 << 23) - 1) >> 23;
    a->grid_x = (uint32_t)((blocks + lines - 1) / lines);
    return dim3(a->grid_x, (unsigned)lines);
}

template <typename T>
int launch(Args& a, bool wide, hipStream_t st) {
    const int heads = a.heads[0] + a.heads[1];
    if (!wide) {
        const int64_t n = a.rows * heads * (a.rot / 2 + a.dim - a.rot);
        DT_REQUIRE((n + 255) / 256 < (1ll << 31), "dt_rotary_apply: grid too large");
        const dim3 grid = lines_of((n + 255) / 256, &a);
        hipLaunchKernelGGL((rotary_any_kernel<T>), grid, dim3(256), 0, st, a);
        return check_launch("dt_rotary_apply");
    }
    // Four heads a lane where that leaves every SIMD a wave; else one, whose loads are the shorter wait (40 heads of
    // 128, bf16: 64 tokens 3.6 us with one, 4.5 with four; 512 5.6 and 5.0; 4096 22 and 17.6).
    const int four = (heads + 4 * a.slots - 1) / (4 * a.slots);
    const bool many = a.rows * four >= 4 * cu_count();
    a.chunks = many ? four : (heads + a.slots - 1) / a.slots;
    a.chunk_div = make_fastdiv((uint32_t)a.chunks);
    const int64_t waves = a.rows * a.chunks;
    DT_REQUIRE(waves < (1ll << 30), "dt_rotary_apply: grid too large");
    const dim3 grid = lines_of((waves + 3) / 4, &a);
    if (many) hipLaunchKernelGGL((rotary_kernel<T, 4>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((rotary_kernel<T, 1>), grid, dim3(256), 0, st, a);
    return check_launch("dt_rotary_apply");
}

// One strided operand [batch][seq][heads][dim]: refused where it cannot be, *wide cleared where
// its rows are not whole 16-byte vectors.
int check_tensor(const dt_rotary_args* x, const void* p, const int64_t* s, int64_t heads, bool out, const char* name, bool* wide) {
    const char* who = "dt_rotary_apply";
    DT_REQUIRE(p != nullptr, "%s: null %s", who, name);
    const int es = elem_size(x->io_type);
    DT_REQUIRE((uintptr_t)p % es == 0, "%s: %s must be aligned to its elements", who, name);
    if (!aligned16(p)) *wide = false;
    const int64_t n[3] = {x->batch, x->seq, heads};
    int64_t reach = x->head_dim;
    bool done[3] = {false, false, false};
    for (int pass = 0; pass < 3; ++pass) {
        int at = -1;
        for (int i = 0; i < 3; ++i)
            if (!done[i] && (at < 0 || s[i] < s[at])) at = i;
        done[at] = true;
        if (n[at] == 1) continue;
        DT_REQUIRE(s[at] >= 0 && s[at] < (1ll << 40), "%s: %s stride %lld unsupported", who, name, (long long)s[at]);
        if (s[at] * es % 16) *wide = false;
        if (!out) continue;
        DT_REQUIRE(s[at] >= reach, "%s: elements of %s overlap", who, name);
        reach = s[at] * (n[at] - 1) + reach;
    }
    return DT_OK;
}

}  // namespace

int check_rotary(const dt_rotary& r, int64_t head_dim, const char* who) {
    DT_REQUIRE(r.rot_dims >= 0 && r.rot_dims % 2 == 0 && r.rot_dims <= head_dim,
               "%s: %lld rotated dims of %lld unsupported (an even number, at most the head's)", who, (long long)r.rot_dims,
               (long long)head_dim);
    DT_REQUIRE(r.rot_dims == 0 || r.freq, "%s: null freq", who);
    DT_REQUIRE(((uintptr_t)r.freq & 3) == 0, "%s: freq must be 4-byte aligned", who);
    DT_REQUIRE(isfinite(r.attn_factor), "%s: attn_factor must be finite", who);
    return DT_OK;
}

}  // namespace rotary
}  // namespace dit

extern "C" int dt_rotary_freq_fill(float* freq, int64_t rot_dims, double base, double factor, int64_t context, double turns_low,
                                   double turns_high) {
    using namespace dit;
    const char* who = "dt_rotary_freq_fill";
    DT_REQUIRE(rot_dims >= 0 && rot_dims % 2 == 0 && (freq || rot_dims == 0), "%s: an even number of dims and a list are needed", who);
    DT_REQUIRE(base > 0 && isfinite(base) && factor > 0 && isfinite(factor), "%s: base and factor must be positive and finite", who);
    DT_REQUIRE(context >= 0, "%s: negative context", who);
    DT_REQUIRE(context == 0 || (turns_low >= 0 && turns_high > turns_low && isfinite(turns_high)),
               "%s: turns_high must be above turns_low, turns_low not negative", who);
    for (int64_t i = 0; i < rot_dims / 2; ++i) {
        const double f = pow(base, -2.0 * (double)i / (double)rot_dims);
        double keep = 0.0;
        if (context > 0) {
            const double turns = (double)context * f / 6.283185307179586;
            keep = (turns - turns_low) / (turns_high - turns_low);
            keep = keep < 0.0 ? 0.0 : keep > 1.0 ? 1.0 : keep;
        }
        freq[i] = (float)(f * (keep + (1.0 - keep) / factor));
    }
    return DT_OK;
}

extern "C" int dt_rotary_apply(const dt_rotary_args* x, dt_stream_t stream) {
    using namespace dit;
    using namespace dit::rotary;
    const char* who = "dt_rotary_apply";
    DT_REQUIRE(x != nullptr, "%s: null arguments", who);
    DT_REQUIRE(is_io_type(x->io_type), "%s: io_type %d unsupported", who, x->io_type);
    DT_REQUIRE(x->batch >= 0 && x->seq >= 0 && x->heads >= 0 && x->kv_heads >= 0, "%s: negative size", who);
    DT_REQUIRE(x->head_dim > 0 && x->head_dim <= 4096, "%s: head_dim %lld unsupported (1 to 4096)", who, (long long)x->head_dim);
    DT_REQUIRE(x->batch < (1ll << 30) && x->seq < (1ll << 30) && x->batch * x->seq < (1ll << 30) && x->heads < (1 << 16) &&
                   x->kv_heads < (1 << 16), "%s: size too large", who);
    int rc = check_rotary(x->rotary, x->head_dim, who);
    if (rc) return rc;
    Args a{};
    a.heads[0] = x->q ? (int32_t)x->heads : 0;
    a.heads[1] = x->k ? (int32_t)x->kv_heads : 0;
    a.rows = x->batch * x->seq;
    if (a.rows == 0 || a.heads[0] + a.heads[1] == 0) return DT_OK;
    a.dim = (int32_t)x->head_dim;
    a.rot = (int32_t)x->rotary.rot_dims;
    a.half = x->rotary.half != 0;
    // Whole units, whose runs are whole vectors.
    const int unit = 32 / elem_size(x->io_type);
    bool wide = a.dim % unit == 0 && a.dim <= 64 * unit && (!a.half || a.rot % unit == 0);
    if (a.heads[0]) {
        rc = check_tensor(x, x->q, x->q_strides, x->heads, false, "q", &wide);
        if (!rc) rc = check_tensor(x, x->q_out, x->q_out_strides, x->heads, true, "q_out", &wide);
        if (rc) return rc;
        a.t[0] = {x->q, x->q_out, {}, {}};
    }
    if (a.heads[1]) {
        rc = check_tensor(x, x->k, x->k_strides, x->kv_heads, false, "k", &wide);
        if (!rc) rc = check_tensor(x, x->k_out, x->k_out_strides, x->kv_heads, true, "k_out", &wide);
        if (rc) return rc;
        a.t[1] = {x->k, x->k_out, {}, {}};
    }
    for (int i = 0; i < 3; ++i) {
        a.t[0].xs[i] = x->q_strides[i];
        a.t[0].ys[i] = x->q_out_strides[i];
        a.t[1].xs[i] = x->k_strides[i];
        a.t[1].ys[i] = x->k_out_strides[i];
    }
    DT_REQUIRE(x->pos && ((uintptr_t)x->pos & 3) == 0, "%s: pos must be given, 4-byte aligned", who);
    DT_REQUIRE(x->batch <= 1 || (x->pos_stride >= 0 && x->pos_stride < (1ll << 40)), "%s: pos_stride unsupported", who);
    const int64_t q_sizes[3] = {x->batch, x->seq, x->heads}, k_sizes[3] = {x->batch, x->seq, x->kv_heads};
    const int es = elem_size(x->io_type);
    const Strided q(x->q, es, 3, q_sizes, x->q_strides, x->head_dim), q_out(x->q_out, es, 3, q_sizes, x->q_out_strides, x->head_dim);
    const Strided k(x->k, es, 3, k_sizes, x->k_strides, x->head_dim), k_out(x->k_out, es, 3, k_sizes, x->k_out_strides, x->head_dim);
    if (a.heads[0]) DT_REQUIRE(q_out.same_as(q) || !share_memory(q_out, q), "%s: q_out is partly q", who);
    if (a.heads[1]) DT_REQUIRE(k_out.same_as(k) || !share_memory(k_out, k), "%s: k_out is partly k", who);
    if (a.heads[0] && a.heads[1]) {
        DT_REQUIRE(!share_memory(q_out, k), "%s: q_out is partly k", who);
        DT_REQUIRE(!share_memory(k_out, q), "%s: k_out is partly q", who);
        DT_REQUIRE(!share_memory(q_out, k_out), "%s: q_out is partly k_out", who);
    }
    a.seq = (int32_t)x->seq;
    a.seq_div = make_fastdiv((uint32_t)x->seq);
    a.pos = x->pos;
    a.pos_stride = x->pos_stride;
    a.freq = a.rot ? x->rotary.freq : reinterpret_cast<const float*>(x->pos);
    a.mul = x->rotary.attn_factor;
    a.sign = x->backward ? -1.f : 1.f;
    a.units = a.dim / unit;
    a.slots = a.units ? 64 / a.units : 0;
    if (wide) a.unit_div = make_fastdiv((uint32_t)a.units);
    const hipStream_t st = (hipStream_t)stream;
    return x->io_type == DT_TYPE_F32 ? launch<float>(a, wide, st) : launch<bf16>(a, wide, st);
}
