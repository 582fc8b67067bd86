// cross_attention.hip -- attention of queries to kept keys of their own number per
// batch entry, with shared key heads and an optional relative position bias:
//   s_ij = scale <q_i, k_j> + table[bucket(j - i - q_pos)][h],  j kept,
//   o_i = sum_j softmax_j(s_ij) v_j,  lse_i = log sum_j exp(s_ij);
// a query without kept keys has o = 0 and lse = -inf.
//
// The products are taken transposed, S^T = K Q^T and O^T += V^T P^T, so a lane
// holds one query in both: the running maximum and sum of the softmax are
// per-lane scalars, and P^T goes from the accumulator straight into the second
// product.  One pass over the keys, no score is stored.  The bias is a line of
// 2 (reach + kMargin) + 1 values per head in LDS (one value from the last bucket's
// start on), read by offset for each score of a 32 x 32 block that the band
// |offset| < reach meets and once for any other.
#include <float.h>
#include <math.h>

#include <type_traits>

#include "attn_tiles.hpp"

namespace dit {
namespace attn {
namespace {

struct FwdArgs {
    AttnIn in;
    void* o;
    int64_t os[3];
    float* lse;      // [batch][heads][seq_q], or null
    int32_t pack;    // query heads of one key head side by side as rows: row = token * pack + head
    FastDiv pack_div;
    int32_t rows, row_blocks, groups;  // rows = seq_q * pack; groups = heads / pack per batch entry
    int32_t splits;  // key ranges of a row block (few-rows kernel)
    float* part_o;   // [splits][batch * groups][rows][DP]: partial results, unnormalised
    float* part_ml;  // [splits][batch * groups][rows][2]: their reference (log2) and sum
};

// With a bias: scores in units of log2, the bias added.  Without: as they are (the scale
// is folded into the exponent).  -inf for a key that is not kept.  Element i of s is key
// 8 (i / 4) + 4 g + i % 4 of the 32 whose kept ones `word` says.
template <bool BIAS>
__device__ __forceinline__ void finish_scores(f32x16_t& s, float sc, uint32_t word, const float* line, int reach, int off0,
                                              int g) {
    if constexpr (BIAS) {
        // off0 + r: offset of key r to this lane's query.
        const int lo = off0 + 4 * g;
        const float* at = line + reach + kMargin + lo;
        if (__builtin_amdgcn_ballot_w64(lo < reach && lo + 28 > -reach) == 0) {
            const float far = line[lo > 0 ? 2 * (reach + kMargin) : 0];
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = __builtin_fmaf(s[i], sc, far);
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = __builtin_fmaf(s[i], sc, at[8 * (i >> 2) + (i & 3)]);
        }
    }
    if (word != 0xFFFFFFFFu) {
        const uint32_t w = word >> (4 * g);
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (!(w & (1u << (8 * (i >> 2) + (i & 3))))) s[i] = -INFINITY;
    }
}

// The running softmax of one query: reference m (log2), this lane's half of the sum.
// Scores are in units of 1 / sc of log2 (sc > 0; 1 with a bias).
template <typename T, int BLOCKS>
struct Running {
    float m, l;
    f32x16_t o[BLOCKS];

    __device__ __forceinline__ void clear() {
        m = -INFINITY;
        l = 0.f;
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b) o[b] = zero16();
    }
    // Whether the reference moved.  It does only when a score exceeds it by more than 2^8, so
    // most tiles skip the rescale, and every weight stays <= 256.
    __device__ __forceinline__ bool look(const f32x16_t& s, float sc) {
        float mx = s[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
        mx = fmaxf(mx, swap32(mx)) * sc;
        const bool move = mx > m + 8.0f;
        if (__builtin_amdgcn_ballot_w64(move) == 0) return false;
        const float to = move ? mx : m;
        const float alpha = move ? __builtin_amdgcn_exp2f(m - to) : 1.0f;
        l *= alpha;
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[b][e] *= alpha;
        m = to;
        return true;
    }
    // The weights of elements 4 i4 .. + 3 into their operand, and added to `sum` before that
    // rounds them: lse, from which the gradients' weights come, stays fp32.
    __device__ __forceinline__ void weigh(const f32x16_t& s, float sc, int i4, FragParts<T> (&p)[2], float& sum) const {
        const float ref = m == -INFINITY ? 0.f : m;  // scores of -inf only, so far: weight 0
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * i4 + e], sc, -ref));
        p[i4 / 2].set(i4 & 1, v);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum += v[e];
    }
};

// The lane's row of a row block.
struct Row {
    int tok, h;
    bool live;
    __device__ __forceinline__ Row(const FwdArgs& a, int row, int h0) {
        live = row < a.rows;
        tok = live ? (int)fdiv((uint32_t)row, a.pack_div) : 0;
        h = h0 + (live ? row - tok * a.pack : 0);
    }
};

// ---- many rows: 128 rows per workgroup, 32 per wave, tiles of 64 KG keys shared --------
// A tile's two 32-key halves are staggered, so that one half's weights (vector and
// exponential instructions) run between the other half's products.
// KG = 1: four waves, two workgroups per CU; head widths up to 64 four, for whose 16 waves the
// registers are held to 128 (4 x 64 heads x 512 tokens with a bias: 33.5 -> 30.4 us).
// KG = 2: for at most one block per CU eight waves, two per SIMD; each half of them
// takes half of a 128-key tile, and the halves' results are joined through LDS (2048
// queries x 16 heads x 128 to 1500 keys: 52 -> 40 us).
template <typename T, int DP, bool BIAS, int KG>
__global__ __launch_bounds__(256 * KG, sizeof(T) == 4 ? 1 : DP == 64 && KG == 1 ? 4 : 2) void attn_rows_kernel(const FwdArgs a) {
    typedef Tile<T, DP> Tl;
    constexpr int KB = 64 * KG, TILE = KB * Tl::RB, NW = 4 * KG;
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];  // [buffer][K | V], then the bias line
    float* const line = reinterpret_cast<float*>(smem + 4 * TILE);
    const AttnIn& in = a.in;

    // Batch entries innermost: their lengths differ, and every XCD gets some of each.
    const uint32_t bid = xcd_block();
    const int blk = (int)(bid % (uint32_t)a.row_blocks), bg = (int)(bid / (uint32_t)a.row_blocks);
    const int b = bg % in.batch, h0 = bg / in.batch * a.pack, kvh = h0 / in.shared;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 31, g = lane >> 5, kg = wave >> 2;
    const int row = blk * 128 + (wave & 3) * 32 + r;
    const Row w(a, row, h0);

    const T* Kp = reinterpret_cast<const T*>(in.k) + b * in.ks[0] + kvh * in.ks[2];
    const T* Vp = reinterpret_cast<const T*>(in.v) + b * in.vs[0] + kvh * in.vs[2];
    Kept<KB> kept;
    kept.start(in, b, kept_len(in, b), 0, in.seq_kv, 1, lane);
    typename Tl::template Loads<KB, NW> kl, vl;
    kl.init(in.ks[1], in.dim, wave, lane);
    vl.init(in.vs[1], in.dim, wave, lane);
    auto issue = [&](int t, int buf) {
        uint8_t* kb = smem + buf * 2 * TILE;
        const T* ks = Kp + (int64_t)t * KB * in.ks[1];
        const T* vs = Vp + (int64_t)t * KB * in.vs[1];
        if (all_kept<KB>(kept.word)) {
            kl.issue_all(ks, kb, wave);
            vl.issue_all(vs, kb + TILE, wave);
        } else {
            const auto keep = [&](int i) { return kept_row(kept.word, i); };
            kl.issue(ks, kb, wave, lane, keep);
            vl.issue(vs, kb + TILE, wave, lane, keep);
        }
    };
    int t = kept.next(lane);
    uint64_t word = kg ? kept.word[KG - 1] : kept.word[0];
    if (t >= 0) issue(t, 0);

    typename Tl::Frag qf[Tl::STEPS];
    {
        const T* qp = reinterpret_cast<const T*>(in.q) + b * in.qs[0] + (int64_t)w.tok * in.qs[1] + w.h * in.qs[2];
#pragma unroll
        for (int c = 0; c < Tl::STEPS; ++c) qf[c] = w.live ? frag_global<T>(qp, c, g, in.dim) : frag_zero<T>();
    }
    if constexpr (BIAS) rel_line(in.rel, h0, line, tid, 64 * NW);  // read after the first tile's barrier
    const typename Tl::Cols cols = Tl::cols(lane);
    Running<T, Tl::BLOCKS> run;
    run.clear();
    const float sc = BIAS ? 1.0f : in.scale_log2;
    // With a bias a row is a token; rows past the last one too, so the block's offsets stay together.
    const int at = BIAS ? row + rel_position(in.rel, b) : 0;

    int buf = 0;
    while (t >= 0) {
        wait_vmem<0>();
        wait_lds();
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        const int t_next = kept.next(lane);
        if (t_next >= 0) issue(t_next, buf ^ 1);
        const uint8_t* Kt = smem + buf * 2 * TILE + kg * 64 * Tl::RB;
        const uint8_t* Vt = Kt + TILE;
        if (KG == 1 || word) {
            f32x16_t s[2] = {zero16(), zero16()};
            FragParts<T> p[2][2];
            float sum[2] = {0.f, 0.f};
            auto scores = [&](auto hc, auto vc, auto side) {
                constexpr int hh = decltype(hc)::value;
                products<T, Tl::STEPS, 1, decltype(vc)::value>(
                    [&](int i) { return Tl::row_frag(Kt, 32 * hh + r, i, g); },
                    [&](int i, const typename Tl::Frag& f) { s[hh] = mma(f, qf[i], s[hh]); }, side);
            };
            auto finish = [&](int hh) {
                finish_scores<BIAS>(s[hh], in.scale_log2, (uint32_t)(word >> (32 * hh)), line, in.rel.reach,
                                    t * KB + kg * 64 + 32 * hh - at, g);
            };
            auto weights = [&](auto hc) {
                return [&, hc](int part, int of) {
#pragma unroll
                    for (int i4 = 0; i4 < 4; ++i4)
                        if (i4 * of / 4 == part) run.weigh(s[hc], sc, i4, p[hc], sum[hc]);
                };
            };
            auto values = [&](auto hc, auto vc, auto side) {
                constexpr int hh = decltype(hc)::value;
                products<T, 2 * Tl::BLOCKS, 2, decltype(vc)::value>(
                    [&](int i) { return Tl::col_frag(Vt, 32 * hh + 16 * (i / Tl::BLOCKS), i % Tl::BLOCKS, cols); },
                    [&](int i, const typename Tl::Frag& f) {
                        run.o[i % Tl::BLOCKS] = mma(f, p[hh][i / Tl::BLOCKS].frag(), run.o[i % Tl::BLOCKS]);
                    },
                    side);
            };
            using H0 = std::integral_constant<int, 0>;
            using H1 = std::integral_constant<int, 1>;
            using V = std::integral_constant<int, DP == 64 ? 12 : 6>;  // vector instructions per product
            scores(H0{}, H0{}, NoSide{});
            finish(0);
            run.look(s[0], sc);
            scores(H1{}, V{}, weights(H0{}));
            finish(1);
            if (run.look(s[1], sc)) {  // the first half's weights again, by the new reference
                sum[0] = 0.f;
                weights(H0{})(0, 1);
            }
            values(H0{}, V{}, weights(H1{}));
            values(H1{}, H0{}, NoSide{});
            run.l += sum[0] + sum[1];
        }
        t = t_next;
        word = kg ? kept.word[KG - 1] : kept.word[0];
        buf ^= 1;
    }
    if constexpr (KG == 2) {
        // The second half's waves hand theirs over in the tiles' place, lane for lane.
        __syncthreads();
        float* part = reinterpret_cast<float*>(smem) + (wave & 3) * (Tl::BLOCKS * 16 + 2) * 64 + lane;
        if (kg == 1) {
            part[0] = run.m;
            part[64] = run.l;
#pragma unroll
            for (int d = 0; d < Tl::BLOCKS; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) part[(2 + 16 * d + e) * 64] = run.o[d][e];
        }
        __syncthreads();
        if (kg == 1) return;
        const float m1 = part[0], m = fmaxf(run.m, m1), ref = m == -INFINITY ? 0.f : m;
        const float w0 = __builtin_amdgcn_exp2f(run.m - ref), w1 = __builtin_amdgcn_exp2f(m1 - ref);
        run.m = m;
        run.l = run.l * w0 + part[64] * w1;
#pragma unroll
        for (int d = 0; d < Tl::BLOCKS; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) run.o[d][e] = run.o[d][e] * w0 + part[(2 + 16 * d + e) * 64] * w1;
    }
    const float l = run.l + swap32(run.l);
    const float inv = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);  // no kept key: 0; NaN stays
    if (!w.live) return;
    T* op = reinterpret_cast<T*>(a.o) + b * a.os[0] + (int64_t)w.tok * a.os[1] + w.h * a.os[2];
#pragma unroll
    for (int d = 0; d < Tl::BLOCKS; ++d)
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) {
            const int e0 = 32 * d + 8 * i4 + 4 * g;
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = run.o[d][4 * i4 + e] * inv;
            if (e0 < in.dim) put4(op + e0, v);
        }
    if (a.lse && g == 0)
        a.lse[((int64_t)b * in.heads + w.h) * in.seq_q + w.tok] =
            l == 0.f ? -INFINITY : (run.m + __builtin_amdgcn_logf(l)) * kLn2;
}

// ---- few rows: 32 rows per workgroup, keys over its waves and over workgroups --------
// One new token, or few rows in all: the keys are a stream.  Each wave takes every
// fourth 32-key tile of the workgroup's key range from buffers of its own and waits
// for its own DMA only; the waves' results meet in LDS.  With more than one range
// per row block the partial results go through the workspace (attn_join_kernel).
template <typename T, int DP, bool BIAS>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void attn_few_kernel(const FwdArgs a) {
    typedef Tile<T, DP> Tl;
    constexpr int KB = 32, TILE = KB * Tl::RB, NW = 4;
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];  // [wave][K | V], then the bias line
    __shared__ float ml[2][NW][32];
    static_assert(NW * 2 * TILE >= NW * DP * 32 * 2, "the partial results take the tiles' place");
    float* const line = reinterpret_cast<float*>(smem + NW * 2 * TILE);
    const AttnIn& in = a.in;

    const uint32_t bid = xcd_block();
    const int blk = (int)(bid % (uint32_t)a.row_blocks), rest = (int)(bid / (uint32_t)a.row_blocks);
    const int split = rest % a.splits, bg = rest / a.splits;
    const int b = bg % in.batch, h0 = bg / in.batch * a.pack, kvh = h0 / in.shared;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 31, g = lane >> 5;
    const int row = blk * 32 + r;
    const Row w(a, row, h0);
    const int tok = w.tok, h = w.h;
    const bool live = w.live;

    const T* Kp = reinterpret_cast<const T*>(in.k) + b * in.ks[0] + kvh * in.ks[2];
    const T* Vp = reinterpret_cast<const T*>(in.v) + b * in.vs[0] + kvh * in.vs[2];
    uint8_t* const Kt = smem + wave * 2 * TILE;
    uint8_t* const Vt = Kt + TILE;
    // This range's tiles of the entry's own kept length: ranges stay even however
    // the lengths differ.
    const int len = kept_len(in, b), tiles = (len + KB - 1) / KB;
    const int first = (int)((int64_t)tiles * split / a.splits), last = (int)((int64_t)tiles * (split + 1) / a.splits);
    Kept<KB> kept;
    kept.start(in, b, len, first + wave, last, NW, lane);
    typename Tl::template Loads<KB, 1> kl, vl;
    kl.init(in.ks[1], in.dim, 0, lane);
    vl.init(in.vs[1], in.dim, 0, lane);
    auto issue = [&](const auto& loads, const T* src, int64_t stride, int t, uint32_t word, uint8_t* lds) {
        const T* p = src + (int64_t)t * KB * stride;
        if (word == 0xFFFFFFFFu) loads.issue_all(p, lds, 0);
        else loads.issue(p, lds, 0, lane, [&](int i) { return (word >> i) & 1; });
    };
    constexpr int VL = KB * Tl::CPR / 64;  // loads of one tile
    int t = kept.next(lane);
    uint32_t word = (uint32_t)kept.word[0];
    if (t >= 0) issue(kl, Kp, in.ks[1], t, word, Kt);

    typename Tl::Frag qf[Tl::STEPS];
    {
        const T* qp = reinterpret_cast<const T*>(in.q) + b * in.qs[0] + (int64_t)tok * in.qs[1] + h * in.qs[2];
#pragma unroll
        for (int c = 0; c < Tl::STEPS; ++c) qf[c] = live ? frag_global<T>(qp, c, g, in.dim) : frag_zero<T>();
    }
    if (t >= 0) issue(vl, Vp, in.vs[1], t, word, Vt);
    if constexpr (BIAS) {  // its loads behind the first tile's
        rel_line(in.rel, h0, line, tid, 256);
        __syncthreads();
    }
    const typename Tl::Cols cols = Tl::cols(lane);
    Running<T, Tl::BLOCKS> run;
    run.clear();
    // With a bias a row is a token; rows past the last one too, so the block's offsets stay together.
    const int at = BIAS ? row + rel_position(in.rel, b) : 0;

    while (t >= 0) {
        wait_vmem<VL>();  // K (V's loads are younger)
        __builtin_amdgcn_sched_barrier(0);
        f32x16_t s[1] = {zero16()}, s2 = zero16();
        products<T, Tl::STEPS, 1>([&](int i) { return Tl::row_frag(Kt, r, i, g); },
                                  [&](int i, const typename Tl::Frag& f) {
                                      if (i & 1) s2 = mma(f, qf[i], s2);
                                      else s[0] = mma(f, qf[i], s[0]);
                                  });
#pragma unroll
        for (int i = 0; i < 16; ++i) s[0][i] += s2[i];
        wait_lds();  // K is read: its buffer is free
        __builtin_amdgcn_sched_barrier(0);
        const int t_next = kept.next(lane);
        const uint32_t word_next = (uint32_t)kept.word[0];
        if (t_next >= 0) issue(kl, Kp, in.ks[1], t_next, word_next, Kt);
        finish_scores<BIAS>(s[0], in.scale_log2, word, line, in.rel.reach, t * KB - at, g);
        run.look(s[0], BIAS ? 1.0f : in.scale_log2);
        FragParts<T> p[2];
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) run.weigh(s[0], BIAS ? 1.0f : in.scale_log2, i4, p, run.l);
        // V (the next K's loads, and the mask byte read ahead, are younger).
        if (t_next >= 0) wait_vmem<VL>();
        else wait_vmem<0>();
        __builtin_amdgcn_sched_barrier(0);
        products<T, 2 * Tl::BLOCKS, 2>(
            [&](int i) { return Tl::col_frag(Vt, 16 * (i / Tl::BLOCKS), i % Tl::BLOCKS, cols); },
            [&](int i, const typename Tl::Frag& f) {
                run.o[i % Tl::BLOCKS] = mma(f, p[i / Tl::BLOCKS].frag(), run.o[i % Tl::BLOCKS]);
            });
        wait_lds();
        __builtin_amdgcn_sched_barrier(0);
        if (t_next >= 0) issue(vl, Vp, in.vs[1], t_next, word_next, Vt);
        t = t_next;
        word = word_next;
    }

    // The waves' results under the largest reference.
    const float l = run.l + swap32(run.l);
    if (g == 0) {
        ml[0][wave][r] = run.m;
        ml[1][wave][r] = l;
    }
    __syncthreads();
    float m = ml[0][0][r];
#pragma unroll
    for (int w = 1; w < NW; ++w) m = fmaxf(m, ml[0][w][r]);
    const float ref = m == -INFINITY ? 0.f : m;
    const float mine = __builtin_amdgcn_exp2f(run.m - ref);
    float total = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) total += __builtin_amdgcn_exp2f(ml[0][w][r] - ref) * ml[1][w][r];
    float* part = reinterpret_cast<float*>(smem);  // half of the width at a time: [wave][DP / 2][32]
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        if (half) __syncthreads();
#pragma unroll
        for (int d = 0; d < Tl::BLOCKS / 2; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e)
                part[(wave * (DP / 2) + 32 * d + 8 * (e >> 2) + 4 * g + (e & 3)) * 32 + r] =
                    run.o[half * (Tl::BLOCKS / 2) + d][e] * mine;
        __syncthreads();
        constexpr int PER = DP / 2 / 8;  // elements a thread (32 rows x 8 threads)
        if (live) {
            const int d0 = (tid >> 5) * PER;
            float* po = a.splits > 1 ? a.part_o + (((int64_t)split * in.batch * a.groups + bg) * a.rows + row) * DP : nullptr;
            T* op = reinterpret_cast<T*>(a.o) + b * a.os[0] + (int64_t)tok * a.os[1] + h * a.os[2];
            const float inv = total > 0.f ? 1.0f / total : (total == 0.f ? 0.f : total);
#pragma unroll
            for (int d = 0; d < PER; d += 4) {
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float x = 0.f;
#pragma unroll
                    for (int w = 0; w < NW; ++w) x += part[(w * (DP / 2) + d0 + d + e) * 32 + r];
                    v[e] = po ? x : x * inv;
                }
                const int e0 = half * (DP / 2) + d0 + d;
                if (e0 >= in.dim) continue;
                if (po) put4(po + e0, v);
                else put4(op + e0, v);
            }
        }
    }
    if (!live || tid >= 32) return;
    if (a.splits > 1) {
        float* p = a.part_ml + (((int64_t)split * in.batch * a.groups + bg) * a.rows + row) * 2;
        p[0] = m;
        p[1] = total;
    } else if (a.lse) {
        a.lse[((int64_t)b * in.heads + h) * in.seq_q + tok] =
            total == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(total)) * kLn2;
    }
}

// The key ranges' results of one row, joined in range order: a thread per four elements.
template <typename T, int DP>
__global__ __launch_bounds__(256) void attn_join_kernel(const FwdArgs a) {
    const AttnIn& in = a.in;
    constexpr int TPR = DP / 4;
    const int64_t id = ((int64_t)blockIdx.x * 256 + threadIdx.x) / TPR;
    const int d = (int)(threadIdx.x % TPR) * 4;
    const int64_t n = (int64_t)in.batch * a.groups * a.rows;
    if (id >= n) return;
    const int row = (int)(id % a.rows), bg = (int)(id / a.rows);
    const Row r(a, row, bg / in.batch * a.pack);
    const int tok = r.tok, h = r.h, b = bg % in.batch;
    float m = -INFINITY;
    for (int s = 0; s < a.splits; ++s) m = fmaxf(m, a.part_ml[((int64_t)s * n + id) * 2]);
    const float ref = m == -INFINITY ? 0.f : m;
    float l = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
    if (d < in.dim) {
        for (int s = 0; s < a.splits; ++s) {
            const float* p = a.part_ml + ((int64_t)s * n + id) * 2;
            const float w = __builtin_amdgcn_exp2f(p[0] - ref);
            l += w * p[1];
            const float4 x = *reinterpret_cast<const float4*>(a.part_o + ((int64_t)s * n + id) * DP + d);
            v[0] += w * x.x;
            v[1] += w * x.y;
            v[2] += w * x.z;
            v[3] += w * x.w;
        }
        const float inv = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] *= inv;
        put4(reinterpret_cast<T*>(a.o) + b * a.os[0] + (int64_t)tok * a.os[1] + h * a.os[2] + d, v);
    }
    if (a.lse && d == 0)
        a.lse[((int64_t)b * in.heads + h) * in.seq_q + tok] = l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn2;
}

// ---- choice and launch --------------------------------------------------------------
struct Plan {
    bool few;
    int kg, pack, groups, rows, row_blocks, splits;
    int64_t part_floats;  // workspace
};

int padded_dim(int64_t dim) { return dim <= 64 ? 64 : 128; }

// Query heads that share a key head lie side by side as rows (their keys are then
// read once), but with a bias, whose line belongs to one head.
Plan plan(const AttnIn& in, bool bf16_io, int cus) {
    Plan p{};
    const int64_t batch = in.batch;
    p.pack = in.rel.table ? 1 : in.shared;
    p.groups = in.heads / p.pack;
    p.rows = in.seq_q * p.pack;
    const int64_t wide = (int64_t)((p.rows + 127) / 128) * p.groups * batch;
    const int64_t narrow = (int64_t)((p.rows + 31) / 32) * p.groups * batch;
    // Blocks of 128 rows while they give three quarters of the CUs one, and are not three quarters
    // empty (16 heads x 128, 512 keys: 192 blocks 16.4 us, in 32 rows 19.9; 128 blocks 15.8
    // and 13.2; 8192 keys: 131 and 167; 144 and 98).  Workgroups of 32 rows come in rounds of
    // their own, by which the line is off in places, in either direction: width 128, 160 blocks
    // 15.4 and 18.5 at 512 keys, 131 and 162 at 8192; 192 blocks at width 64 and 2048 keys 27.7
    // and 24.5, in fp32 165 and 121.
    p.few = wide * 4 < 3 * cus || p.rows <= 32;
    p.splits = p.kg = 1;
    if (!p.few) {
        p.row_blocks = (p.rows + 127) / 128;
        // bf16 leaves room for a second workgroup, or twice the waves, on a CU.
        if (wide <= cus && in.seq_kv > 64 && bf16_io) p.kg = 2;
        return p;
    }
    p.row_blocks = (p.rows + 31) / 32;
    int64_t s = 2 * cus / (narrow > 0 ? narrow : 1);
    // Eight tiles of 32 keys a range, two a wave; sixteen where every CU has a workgroup anyway.
    const int64_t most = in.seq_kv / (narrow < cus ? 256 : 512);
    if (s > most) s = most;
    if (s > 64) s = 64;
    p.splits = s < 2 ? 1 : (int)s;
    if (p.splits > 1) p.part_floats = (int64_t)p.splits * batch * p.groups * p.rows * (padded_dim(in.dim) + 2);
    return p;
}

template <typename T, int DP, bool BIAS>
int launch(const FwdArgs& a, const Plan& p, hipStream_t st) {
    const size_t tiles = p.few ? 4 * 2 * 32 * Tile<T, DP>::RB : p.kg * 4 * 64 * Tile<T, DP>::RB;
    const size_t lds = tiles + rel_line_floats(a.in.rel) * sizeof(float);
    const int64_t bg = (int64_t)p.groups * a.in.batch;
    const int64_t wide = p.row_blocks * bg;
    if (p.few) {
        hipLaunchKernelGGL((attn_few_kernel<T, DP, BIAS>), dim3((unsigned)(p.row_blocks * p.splits * bg)), dim3(256), lds, st, a);
    } else {
        if constexpr (sizeof(T) == 2)
            if (p.kg == 2) hipLaunchKernelGGL((attn_rows_kernel<T, DP, BIAS, 2>), dim3((unsigned)wide), dim3(512), lds, st, a);
        if (p.kg == 1) hipLaunchKernelGGL((attn_rows_kernel<T, DP, BIAS, 1>), dim3((unsigned)wide), dim3(256), lds, st, a);
    }
    int rc = check_launch("dt_attn_fwd");
    if (rc || p.splits == 1) return rc;
    const int64_t n = bg * p.rows * (DP / 4);
    hipLaunchKernelGGL((attn_join_kernel<T, DP>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, a);
    return check_launch("dt_attn_fwd");
}

template <typename T, int DP>
int launch_bias(const FwdArgs& a, const Plan& p, hipStream_t st) {
    return a.in.rel.table ? launch<T, DP, true>(a, p, st) : launch<T, DP, false>(a, p, st);
}

// n^far >= near^(far - j) * max^j in whole numbers of up to 512 bits (1024^32 has 321).
struct Wide {
    uint32_t w[16] = {1};
    void times(uint32_t f) {
        uint64_t c = 0;
        for (uint32_t& x : w) {
            c += (uint64_t)x * f;
            x = (uint32_t)c;
            c >>= 32;
        }
    }
    bool at_least(const Wide& o) const {
        for (int i = 15; i >= 0; --i)
            if (w[i] != o.w[i]) return w[i] > o.w[i];
        return true;
    }
};
bool reaches(int n, int near, int max, int far, int j) {
    // By logarithms where they are not next to each other (they are off by 1e-13 at most).
    const double d = far * log((double)n) - (far - j) * log((double)near) - j * log((double)max);
    if (fabs(d) > 1e-9) return d > 0;
    Wide a, b;
    for (int i = 0; i < far; ++i) {
        a.times((uint32_t)n);
        b.times((uint32_t)(i < j ? max : near));
    }
    return a.at_least(b);
}

// start[t]: the least distance of bucket t of a side: t up to half of them, then the least n
// with near + floor(log(n / near) / log(max / near) * far) >= t.
void bucket_starts(int side, int max, int32_t* start) {
    const int near = side / 2, far = side - near;
    for (int t = 0; t <= near; ++t) start[t] = t;
    for (int t = near + 1; t < side; ++t) {
        const int j = t - near;
        int n = (int)ceil(near * pow((double)max / near, (double)j / far));
        while (n > near && reaches(n - 1, near, max, far, j)) --n;
        while (!reaches(n, near, max, far, j)) ++n;
        start[t] = n;
    }
}

int check_rel(int64_t buckets, int64_t distance, int32_t two_sided, const char* who) {
    const int64_t side = two_sided ? buckets / 2 : buckets;
    DT_REQUIRE((!two_sided || buckets % 2 == 0) && side >= 2 && side <= kMaxSide,
               "%s: %lld relative position buckets unsupported (2 to %d a side)", who, (long long)buckets, kMaxSide);
    DT_REQUIRE(distance > side / 2 && distance <= kMaxDistance,
               "%s: relative position distance %lld outside %lld..%d", who, (long long)distance, (long long)(side / 2 + 1),
               kMaxDistance);
    return DT_OK;
}

}  // namespace

int check_rows(const dt_attn_args* x, const void* p, const int64_t* strides, int64_t heads, int64_t seq, bool out,
               const char* name, const char* who) {
    if (x->batch == 0 || heads == 0 || seq == 0) return DT_OK;  // no element
    DT_REQUIRE(p != nullptr && strides != nullptr, "%s: null %s", who, name);
    DT_REQUIRE(aligned16(p), "%s: %s must be 16-byte aligned", who, name);
    const int64_t n[3] = {x->batch, seq, heads}, step = x->io_type == DT_TYPE_F32 ? 4 : 8;  // elements of 16 bytes
    int64_t reach = x->head_dim;  // of the dimensions with smaller strides
    bool done[3] = {false, false, false};
    for (int pass = 0; pass < 3; ++pass) {
        int at = -1;
        for (int i = 0; i < 3; ++i)
            if (!done[i] && (at < 0 || strides[i] < strides[at])) at = i;
        done[at] = true;
        if (n[at] == 1) continue;
        const int64_t s = strides[at];
        DT_REQUIRE(s % step == 0, "%s: %s strides must keep rows 16-byte aligned", who, name);
        DT_REQUIRE(s >= 0 && s < (at == 1 ? kMaxRowBytes / 16 * step : 1ll << 40), "%s: %s stride %lld unsupported", who, name, (long long)s);
        if (!out) continue;
        DT_REQUIRE(s >= reach, "%s: elements of %s overlap", who, name);
        reach = s * (n[at] - 1) + reach;
    }
    return DT_OK;
}

int prepare_in(const dt_attn_args* x, const char* who, AttnIn* out) {
    DT_REQUIRE(x != nullptr, "%s: null arguments", who);
    DT_REQUIRE(is_io_type(x->io_type), "%s: io_type %d unsupported", who, x->io_type);
    DT_REQUIRE(x->batch >= 0 && x->heads >= 0 && x->kv_heads >= 0 && x->seq_q >= 0 && x->seq_kv >= 0, "%s: negative size", who);
    DT_REQUIRE(x->head_dim > 0 && x->head_dim <= 128 && x->head_dim % 8 == 0,
               "%s: head_dim %lld unsupported (a multiple of 8 up to 128)", who, (long long)x->head_dim);
    DT_REQUIRE(x->heads == 0 || (x->kv_heads > 0 && x->heads % x->kv_heads == 0),
               "%s: %lld query heads do not share %lld key heads evenly", who, (long long)x->heads, (long long)x->kv_heads);
    DT_REQUIRE(x->batch < (1 << 20) && x->heads < (1 << 16) && x->seq_q < kMaxSeq && x->seq_kv < kMaxSeq &&
                   x->seq_q * (x->heads == 0 ? 1 : x->heads / x->kv_heads) < (1ll << 30), "%s: size too large", who);
    DT_REQUIRE(x->scale >= 0.f && x->scale < INFINITY, "%s: scale must be >= 0 and finite (got %g)", who, (double)x->scale);
    int rc = check_rows(x, x->q, x->q_strides, x->heads, x->seq_q, false, "q", who);
    if (!rc) rc = check_rows(x, x->k, x->k_strides, x->kv_heads, x->seq_kv, false, "k", who);
    if (!rc) rc = check_rows(x, x->v, x->v_strides, x->kv_heads, x->seq_kv, false, "v", who);
    if (rc) return rc;
    DT_REQUIRE(((uintptr_t)x->kv_len & 3) == 0 && ((uintptr_t)x->q_pos & 3) == 0, "%s: kv_len and q_pos must be 4-byte aligned", who);
    DT_REQUIRE(!x->kv_mask || x->batch <= 1 || x->kv_mask_stride >= 0, "%s: negative kv_mask_stride", who);
    AttnIn a{};
    a.q = x->q;
    a.k = x->k;
    a.v = x->v;
    for (int i = 0; i < 3; ++i) {
        a.qs[i] = x->q_strides[i];
        a.ks[i] = x->k_strides[i];
        a.vs[i] = x->v_strides[i];
    }
    a.batch = (int32_t)x->batch;
    a.heads = (int32_t)x->heads;
    a.kv_heads = (int32_t)x->kv_heads;
    a.shared = x->kv_heads ? (int32_t)(x->heads / x->kv_heads) : 1;
    a.seq_q = (int32_t)x->seq_q;
    a.seq_kv = (int32_t)x->seq_kv;
    a.dim = (int32_t)x->head_dim;
    a.kv_len = x->kv_len;
    a.kv_mask = x->kv_mask;
    a.mask_stride = x->kv_mask_stride;
    a.scale = x->scale;
    // A scale of 0 as the least normal number: -inf times it is still -inf, and every finite
    // score still next to 0.
    a.scale_log2 = x->scale * kLog2e > FLT_MIN ? x->scale * kLog2e : FLT_MIN;
    if (x->rel_table) {
        rc = check_rel(x->rel_buckets, x->rel_distance, x->rel_two_sided, who);
        if (rc) return rc;
        DT_REQUIRE(((uintptr_t)x->rel_table & 3) == 0 && x->rel_table_stride >= x->heads,
                   "%s: rel_table must be 4-byte aligned with rows of at least heads", who);
        RelArgs& r = a.rel;
        r.table = x->rel_table;
        r.table_stride = x->rel_table_stride;
        r.q_pos = x->q_pos;
        r.two_sided = x->rel_two_sided != 0;
        r.side = r.two_sided ? x->rel_buckets / 2 : x->rel_buckets;
        bucket_starts(r.side, x->rel_distance, r.start);
        r.reach = r.start[r.side - 1];
    }
    *out = a;
    return DT_OK;
}

}  // namespace attn
}  // namespace dit

extern "C" int dt_rel_bucket_fill(int32_t* bucket, int64_t n, int32_t buckets, int32_t distance, int32_t two_sided) {
    using namespace dit;
    using namespace dit::attn;
    const char* who = "dt_rel_bucket_fill";
    DT_REQUIRE(n >= 0 && (bucket || n == 0), "%s: null bucket list", who);
    const int rc = check_rel(buckets, distance, two_sided, who);
    if (rc) return rc;
    const int side = two_sided ? buckets / 2 : buckets;
    int32_t start[kMaxSide];
    bucket_starts(side, distance, start);
    int t = 0;  // of distance d
    for (int64_t d = 0; d < n; ++d) {
        while (t + 1 < side && d >= start[t + 1]) ++t;
        bucket[n - 1 - d] = t;
        bucket[n - 1 + d] = !two_sided ? 0 : d ? side + t : t;
    }
    return DT_OK;
}

extern "C" size_t dt_attn_fwd_workspace_bytes(const dt_attn_args* x) {
    using namespace dit;
    using namespace dit::attn;
    AttnIn in;
    if (prepare_in(x, "dt_attn_fwd_workspace_bytes", &in)) return 0;
    if (in.batch == 0 || in.heads == 0 || in.seq_q == 0) return 0;
    return (size_t)plan(in, x->io_type == DT_TYPE_BF16, cu_count()).part_floats * sizeof(float);
}

extern "C" int dt_attn_fwd(const dt_attn_args* x, void* o, const int64_t* o_strides, float* lse, void* workspace,
                           size_t workspace_bytes, dt_stream_t stream) {
    using namespace dit;
    using namespace dit::attn;
    const char* who = "dt_attn_fwd";
    FwdArgs a{};
    int rc = prepare_in(x, who, &a.in);
    if (!rc) rc = check_rows(x, o, o_strides, x->heads, x->seq_q, true, "o", who);
    if (rc) return rc;
    DT_REQUIRE(((uintptr_t)lse & 3) == 0, "%s: lse must be 4-byte aligned", who);
    if (a.in.batch == 0 || a.in.heads == 0 || a.in.seq_q == 0) return DT_OK;
    a.o = o;
    for (int i = 0; i < 3; ++i) a.os[i] = o_strides[i];
    a.lse = lse;
    Plan p = plan(a.in, x->io_type == DT_TYPE_BF16, cu_count());
    if (p.splits > 1 && (!workspace || workspace_bytes < (size_t)p.part_floats * sizeof(float) || !aligned16(workspace))) p.splits = 1;
    DT_REQUIRE((int64_t)p.row_blocks * p.splits * p.groups * a.in.batch < (1ll << 31) &&
                   (int64_t)a.in.batch * a.in.heads * a.in.seq_q < (1ll << 36), "%s: grid too large", who);
    a.pack = p.pack;
    a.pack_div = make_fastdiv((uint32_t)p.pack);
    a.rows = p.rows;
    a.row_blocks = p.row_blocks;
    a.groups = p.groups;
    a.splits = p.splits;
    a.part_o = (float*)workspace;
    if (p.splits > 1) a.part_ml = a.part_o + (int64_t)p.splits * a.in.batch * p.groups * p.rows * padded_dim(a.in.dim);
    const hipStream_t st = (hipStream_t)stream;
    if (x->io_type == DT_TYPE_F32)
        return padded_dim(a.in.dim) == 64 ? launch_bias<float, 64>(a, p, st) : launch_bias<float, 128>(a, p, st);
    return padded_dim(a.in.dim) == 64 ? launch_bias<bf16, 64>(a, p, st) : launch_bias<bf16, 128>(a, p, st);
}
