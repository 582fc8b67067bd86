// cross_attention_bwd.hip -- the gradients of cross_attention.hip's attention:
//   P_ij = exp(s_ij - lse_i),  dP_ij = <dO_i, v_j>,  delta_i = sum_j P_ij dP_ij,
//   dS = P (dP - delta),  dQ_i = scale sum_j dS_ij k_j,
//   dK_j = scale sum_i dS_ij q_i,  dV_j = sum_i P_ij dO_i  (i over the query heads
//   that share the key head),  dtable[t][h] = sum of dS over the pairs of bucket t.
//
// Two kernels recompute P instead of one that adds into dQ with atomics, so every sum
// has a fixed order and a call gives the same bits each time:
//  * queries: 128 rows per workgroup, a query per lane, keys streamed -- dQ, delta
//    and the table's gradient (transposed products, dS^T straight into dQ^T += K^T dS^T);
//  * keys: 128 keys per workgroup, a key per lane, queries streamed -- dK and dV
//    (S = Q K^T, P and dS straight into dV^T += dO^T P and dK^T += Q^T dS).
//    Too few key blocks for the chip share the queries in ranges, whose fp32 partial
//    sums are added in range order by a third launch.
#include <type_traits>

#include "attn_tiles.hpp"

namespace dit {
namespace attn {
namespace {

struct BwdArgs {
    AttnIn in;
    const void* d_o;
    const void* o;
    int64_t dos[3], os[3];
    const float* lse;   // [batch][heads][seq_q]
    void* dq;
    void* dk;
    void* dv;
    int64_t dqs[3], dks[3], dvs[3];
    float* ref;         // [batch][heads][seq_q]: lse in log2, +inf for a query without kept keys
    float* delta;       // [batch][heads][seq_q]
    float* part_table;  // [batch][heads][row_blocks][buckets]
    float* part_kv;     // [ranges][2][batch][kv_heads][seq_kv][DP]
    float* d_table;
    int64_t d_table_stride;
    int32_t row_blocks, key_blocks, ranges, buckets, table_blocks;
};

// 32-row halves of a wave's part of a tile with four waves side by side; waves that share rows
// when there are few.
template <typename T, int DP>
constexpr int halves() {
    return sizeof(T) == 4 && DP == 128 ? 1 : 2;
}
template <typename T, int DP, bool BIAS>
constexpr int few_waves() {
    return Tile<T, DP>::RB <= 128 || (Tile<T, DP>::RB == 256 && !BIAS) ? 4 : Tile<T, DP>::RB == 256 || !BIAS ? 2 : 1;
}

// delta = <dO, o> is off by the rounding of a bf16 o, and P spreads that over the row's dS: the
// fewer the keys, the less it is averaged (error of dq and dk against 64 bits, in errors
// of one rounding to bf16; two independent ones, of dS and of the result, are
// 1.41: 9 keys 1.67, 16 keys 1.58, 40 keys 1.50, 77 keys 1.46, 200 keys 1.45).  Up to one tile
// of keys sums P dP first (9 to 64 keys: 1.43); up to two would take 42.2 instead of 38.9 us for
// a step of 1024 queries and 77 keys.
constexpr int kExactKeys = 64;
// So do rows of more keys of which a mask keeps few, wherever they lie (9 of 500 1.63 -> 1.42, 32
// 1.50 -> 1.42): the tiles that hold them are walked twice (1024 queries x 16 heads x 4, 32 of 500
// keys in every tile, bwd 51.1 -> 63.1 us, side by side 39.8 -> 43.5; the count alone 0.2).
constexpr int kExactKept = 32;

// A wave's dS block as its 63 diagonals (offsets -31 .. 31), each a row of 32 queries; what
// lies outside the block stays 0.  Rows padded to 36: the block's writes (a step of 35
// floats a lane) and a lane's reads of its row in 16 bytes spread over all banks.
constexpr int kDiag = 36, kScratch = 63 * kDiag;

// The keys kept of 64 N mask bytes, fetched ahead of their count.
template <int N>
struct KeptCount {
    uint32_t m[N];
    __device__ __forceinline__ void fetch(const uint8_t* mask, int from, int len, int lane) {
#pragma unroll
        for (int w = 0; w < N; ++w) m[w] = from + 64 * w + lane < len ? mask[from + 64 * w + lane] : 0u;
    }
    __device__ __forceinline__ int count() const {
        int n = 0;
#pragma unroll
        for (int w = 0; w < N; ++w) n += __builtin_popcountll(__builtin_amdgcn_ballot_w64(m[w] != 0));
        return n;
    }
};

// ---- dQ, delta, the table's gradient ---------------------------------------------------
// WR waves of 32 rows each, times WK that share the rows and take HALVES x 32 keys each of
// a tile; their results meet in LDS in wave order.
template <typename T, int DP, bool BIAS, int WR, int WK, int HALVES>
__global__ __launch_bounds__(64 * WR * WK, sizeof(T) == 2 ? 2 : 1) void attn_dq_kernel(const BwdArgs a) {
    typedef Tile<T, DP> Tl;
    constexpr int MY = 32 * HALVES, KB = MY * WK, TILE = KB * Tl::RB, NW = WR * WK;
    static_assert(WR * (WK - 1) * (Tl::BLOCKS * 16 + 1) * 256 <= 4 * TILE, "the waves' results take the tiles' place");
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];  // [buffer][K | V], scratch, bias line, gradient lines
    const AttnIn& in = a.in;
    const int reach = in.rel.reach;
    const int line_len = rel_line_len(reach), mid = reach + kMargin;
    float* const scratch = reinterpret_cast<float*>(smem + 4 * TILE);
    float* const line = scratch + NW * kScratch;
    // Then the waves' table gradients, a line each as the bias's; scratch first, for its alignment.
    float* const grad = line + line_len;
    __shared__ float far_sum[2][NW], part_delta[NW][32];

    const uint32_t bid = xcd_block();
    const int blk = (int)(bid % (uint32_t)a.row_blocks), bh = (int)(bid / (uint32_t)a.row_blocks);
    const int b = bh % in.batch, h = bh / in.batch, kvh = h / in.shared;  // batch entries innermost, as in the forward pass
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 31, g = lane >> 5, wr = wave % WR, wk = wave / WR;
    const int row0 = (blk * WR + wr) * 32, row = row0 + r;
    const bool live = row < in.seq_q;
    const int tok = live ? row : 0;
    float* const my_grad = grad + wave * line_len;
    float* const my_scratch = scratch + wave * kScratch;

    const T* Kp = reinterpret_cast<const T*>(in.k) + b * in.ks[0] + kvh * in.ks[2];
    const T* Vp = reinterpret_cast<const T*>(in.v) + b * in.vs[0] + kvh * in.vs[2];
    typename Tl::template Loads<KB, NW> kl, vl;
    kl.init(in.ks[1], in.dim, wave, lane);
    vl.init(in.vs[1], in.dim, wave, lane);
    auto issue = [&](int t, const uint64_t (&word)[(KB + 63) / 64], int buf) {
        uint8_t* kb = smem + buf * 2 * TILE;
        const T* ks = Kp + (int64_t)t * KB * in.ks[1];
        const T* vs = Vp + (int64_t)t * KB * in.vs[1];
        if (all_kept<KB>(word)) {
            kl.issue_all(ks, kb, wave);
            vl.issue_all(vs, kb + TILE, wave);
        } else {
            const auto keep = [&](int i) { return kept_row(word, i); };
            kl.issue(ks, kb, wave, lane, keep);
            vl.issue(vs, kb + TILE, wave, lane, keep);
        }
    };

    Kept<KB> kept;
    const int len = kept_len(in, b);
    auto first_tile = [&]() {
        kept.start(in, b, len, 0, in.seq_kv, 1, lane);
        return kept.next(lane);
    };
    // Which of this wave's keys of the tile are kept.
    auto mine = [&]() { return (MY * wk < 64 ? kept.word[0] : kept.word[Kept<KB>::W - 1]) >> (MY * wk & 63); };
    int t = first_tile(), buf = 0;
    uint64_t word = mine();
    if (t >= 0) issue(t, kept.word, 0);

    const bool counted = sizeof(T) == 2 && !BIAS && in.kv_mask && len > kExactKeys;
    const uint8_t* const mask = in.kv_mask + b * in.mask_stride;
    KeptCount<4> head;
    if (counted) head.fetch(mask, 0, len, lane);
    typename Tl::Frag qf[Tl::STEPS], of[Tl::STEPS];
    const int64_t stat = ((int64_t)b * in.heads + h) * in.seq_q + tok;
    float ref = a.lse[stat] * kLog2e;
    if (!live || ref == -INFINITY) ref = INFINITY;
    float delta = 0.f;
    {
        const T* qp = reinterpret_cast<const T*>(in.q) + b * in.qs[0] + (int64_t)tok * in.qs[1] + h * in.qs[2];
        const T* gp = reinterpret_cast<const T*>(a.d_o) + b * a.dos[0] + (int64_t)tok * a.dos[1] + h * a.dos[2];
        const T* op = reinterpret_cast<const T*>(a.o) + b * a.os[0] + (int64_t)tok * a.os[1] + h * a.os[2];
#pragma unroll
        for (int c = 0; c < Tl::STEPS; ++c) {
            qf[c] = live ? frag_global<T>(qp, c, g, in.dim) : frag_zero<T>();
            of[c] = live ? frag_global<T>(gp, c, g, in.dim) : frag_zero<T>();
            delta += frag_dot(of[c], live ? frag_global<T>(op, c, g, in.dim) : frag_zero<T>());
        }
        delta += swap32(delta);
    }
    if constexpr (BIAS) {  // read after the first tile's barrier
        rel_line(in.rel, h, line, tid, 64 * NW);
        for (int i = tid; i < NW * line_len; i += 64 * NW) grad[i] = 0.f;
        for (int i = tid; i < NW * kScratch; i += 64 * NW) scratch[i] = 0.f;
    }
    const typename Tl::Cols cols = Tl::cols(lane);
    const int at = row + (BIAS ? rel_position(in.rel, b) : 0);  // rows past the last one too: the block's offsets stay together

    // S and dP of one 32-key half of a tile.
    auto scores = [&](const uint8_t* Kt, const uint8_t* Vt, int hh, f32x16_t& s, f32x16_t& d, auto vc, auto side) {
        s = d = zero16();
        products<T, 2 * Tl::STEPS, 1, decltype(vc)::value>(
            [&](int i) { return Tl::row_frag(i & 1 ? Vt : Kt, 32 * hh + r, i / 2, g); },
            [&](int i, const typename Tl::Frag& f) {
                if (i & 1) d = mma(f, of[i / 2], d);
                else s = mma(f, qf[i / 2], s);
            },
            side);
    };
    // dS in d from S and dP, elements 4 i4 .. + 3: keys 8 i4 + 4 g + e of the 32 from offset `off`.
    auto weights = [&](const f32x16_t& s, f32x16_t& d, int off, int i4) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = 4 * i4 + e;
            float c = -ref;
            if constexpr (BIAS) c += rel_at(line, reach, off + 4 * g)[8 * i4 + e];
            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], in.scale_log2, c));
            d[i] = p * (d[i] - delta);
        }
    };
    auto drop = [&](f32x16_t& d, uint32_t word) {  // keys that are not kept
        if (word == 0xFFFFFFFFu) return;
        const uint32_t w = word >> (4 * g);
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (!(w & (1u << (8 * (i >> 2) + (i & 3))))) d[i] = 0.f;
    };
    // A pass over the tiles with a kept key, the next one's DMA in flight behind each (behind the
    // last one the next pass's first); body has this wave's rows of K and V, its first key
    // and which of its keys are kept.
    auto walk = [&](auto body, bool again) {
        bool more = t >= 0;
        while (more) {
            wait_vmem<0>();
            wait_lds();
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_sched_barrier(0);
            int t_next = kept.next(lane);
            if (t_next < 0) {
                more = false;
                if (again) t_next = first_tile();
            }
            if (t_next >= 0) issue(t_next, kept.word, buf ^ 1);
            const uint8_t* Kt = smem + buf * 2 * TILE + MY * wk * Tl::RB;
            if (WK == 1 || (HALVES == 2 ? word != 0 : (uint32_t)word != 0)) body(Kt, Kt + TILE, t * KB + MY * wk, word);
            t = t_next;
            word = mine();
            buf ^= 1;
        }
    };

    // dS of a tile's halves: the first half's weights between the second one's products.
    using None = std::integral_constant<int, 0>;
    using SV = std::integral_constant<int, DP == 64 ? 18 : 9>;  // vector instructions per product
    auto each = [&](const uint8_t* Kt, const uint8_t* Vt, int key, f32x16_t (&s)[HALVES], f32x16_t (&d)[HALVES]) {
        const int off = key - at;
        scores(Kt, Vt, 0, s[0], d[0], None{}, NoSide{});
        if constexpr (HALVES == 2)
            scores(Kt, Vt, 1, s[1], d[1], SV{}, [&](int part, int of) {
#pragma unroll
                for (int i4 = 0; i4 < 4; ++i4)
                    if (i4 * of / 4 == part) weights(s[0], d[0], off, i4);
            });
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) weights(s[HALVES - 1], d[HALVES - 1], off + 32 * (HALVES - 1), i4);
    };

    // The table's gradient is kept in fp32, and a whole row's dS cancels in it: delta
    // from the rounded output (off by its rounding and P's) would show there, so it is
    // summed from P and dP first; so it is for few keys.
    bool exact = BIAS || len <= kExactKeys;
    if (counted) {
        int n = head.count();
        for (int from = 256; n <= kExactKept && from < len; from += 1024) {
            KeptCount<16> c;
            c.fetch(mask, from, len, lane);
            n += c.count();
        }
        exact = n <= kExactKept;
    }
    if (sizeof(T) == 2 && exact) {
        float sum = 0.f;
        delta = 0.f;
        walk([&](const uint8_t* Kt, const uint8_t* Vt, int key, uint64_t word) {
            f32x16_t s[HALVES], d[HALVES];
            each(Kt, Vt, key, s, d);
#pragma unroll
            for (int hh = 0; hh < HALVES; ++hh) {
                drop(d[hh], (uint32_t)(word >> (32 * hh)));
#pragma unroll
                for (int i = 0; i < 16; ++i) sum += d[hh][i];
            }
        }, true);
        delta = sum + swap32(sum);
        if constexpr (WK > 1) {  // of all keys, in wave order
            if (g == 0) part_delta[wave][r] = delta;
            __syncthreads();
            delta = part_delta[wr][r];
#pragma unroll
            for (int w = 1; w < WK; ++w) delta += part_delta[w * WR + wr][r];
        }
    }
    if (live && g == 0 && wk == 0) {
        a.ref[stat] = ref;
        a.delta[stat] = delta;
    }

    f32x16_t dq[Tl::BLOCKS];
#pragma unroll
    for (int d = 0; d < Tl::BLOCKS; ++d) dq[d] = zero16();
    float far[2] = {0.f, 0.f};  // keys behind, keys ahead, out of reach
    walk([&](const uint8_t* Kt, const uint8_t* Vt, int key, uint64_t word) {
        f32x16_t s[HALVES], dsv[HALVES];
        each(Kt, Vt, key, s, dsv);
#pragma unroll
        for (int hh = 0; hh < HALVES; ++hh) {
            f32x16_t& ds = dsv[hh];
            drop(ds, (uint32_t)(word >> (32 * hh)));
            if constexpr (BIAS) {
                // Offsets of this 32 x 32 block: off0 + [-31, 31].  A block that is out
                // of reach as a whole has one bucket (per side: reach may be small).
                const int off0 = key + 32 * hh - row0 - (at - row);
                if (off0 - 31 >= reach || off0 + 31 <= -reach) {
                    float sum = 0.f;
#pragma unroll
                    for (int i = 0; i < 16; ++i) sum += ds[i];
                    far[0] += off0 > 0 ? 0.f : sum;
                    far[1] += off0 > 0 ? sum : 0.f;
                } else {
                    // Diagonal key - query + 31 of each element, then a lane sums its diagonal in four parts.
                    float* to = my_scratch + (31 + 4 * g) * kDiag - (kDiag - 1) * r;
#pragma unroll
                    for (int i = 0; i < 16; ++i) to[(8 * (i >> 2) + (i & 3)) * kDiag] = ds[i];
                    wait_lds();
                    __builtin_amdgcn_sched_barrier(0);
                    const float4* from = reinterpret_cast<const float4*>(my_scratch + min(lane, 62) * kDiag);
                    float4 sum = from[0];
#pragma unroll
                    for (int i = 1; i < 8; ++i) {
                        const float4 x = from[i];
                        sum.x += x.x;
                        sum.y += x.y;
                        sum.z += x.z;
                        sum.w += x.w;
                    }
                    if (lane < 63) my_grad[mid + off0 + lane - 31] += (sum.x + sum.y) + (sum.z + sum.w);
                    wait_lds();
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            typename Tl::Frag f2[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) acc_frag<T>(ds, j, f2[j]);
            products<T, 2 * Tl::BLOCKS, 2>(
                [&](int i) { return Tl::col_frag(Kt, 32 * hh + 16 * (i / Tl::BLOCKS), i % Tl::BLOCKS, cols); },
                [&](int i, const typename Tl::Frag& f) { dq[i % Tl::BLOCKS] = mma(f, f2[i / Tl::BLOCKS], dq[i % Tl::BLOCKS]); });
        }
    }, false);

    if constexpr (WK > 1) {  // the other waves' sums, in wave order
        float* part = reinterpret_cast<float*>(smem) + lane;
        constexpr int N = Tl::BLOCKS * 16 * 64;
        __syncthreads();  // every wave has read its last tile
        if (wk > 0) {
#pragma unroll
            for (int d = 0; d < Tl::BLOCKS; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) part[((wk - 1) * WR + wr) * N + (16 * d + e) * 64] = dq[d][e];
        }
        __syncthreads();
        if (wk == 0) {
#pragma unroll
            for (int w = 0; w < WK - 1; ++w)
#pragma unroll
                for (int d = 0; d < Tl::BLOCKS; ++d)
#pragma unroll
                    for (int e = 0; e < 16; ++e) dq[d][e] += part[(w * WR + wr) * N + (16 * d + e) * 64];
        }
    }
    if (live && wk == 0) {
        T* op = reinterpret_cast<T*>(a.dq) + b * a.dqs[0] + (int64_t)tok * a.dqs[1] + h * a.dqs[2];
#pragma unroll
        for (int d = 0; d < Tl::BLOCKS; ++d)
#pragma unroll
            for (int i4 = 0; i4 < 4; ++i4) {
                const int e0 = 32 * d + 8 * i4 + 4 * g;
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = dq[d][4 * i4 + e] * in.scale;
                if (e0 < in.dim) put4(op + e0, v);
            }
    }
    if constexpr (BIAS) {
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            const float f = wave_sum(far[side]);
            if (lane == 0) far_sum[side][wave] = f;
        }
        __syncthreads();
        // The waves' lines, in wave order, into the first.
        const int n = line_len;
        for (int i = tid; i < n; i += 64 * NW) {
            float sum = grad[i];
#pragma unroll
            for (int w = 1; w < NW; ++w) sum += grad[w * n + i];
            grad[i] = sum;
        }
        __syncthreads();
        // Sixteen lanes a bucket, its offsets over them.
        float* out = a.part_table + (((int64_t)b * in.heads + h) * a.row_blocks + blk) * a.buckets;
        for (int t0 = 0; t0 < a.buckets; t0 += 4 * NW) {
            const int bucket = t0 + (tid >> 4), t = min(bucket, a.buckets - 1), i = tid & 15;
            const bool ahead = in.rel.two_sided && t >= in.rel.side;
            const int u = ahead ? t - in.rel.side : t;
            const bool last = u == in.rel.side - 1, rest = !in.rel.two_sided && u == 0;
            // Distances [lo, hi) of the bucket.  Without the two sides every key ahead is at distance 0.
            const int lo = in.rel.start[u], hi = last ? mid + 1 : in.rel.start[u + 1];
            float sum = 0.f;
            for (int dist = lo + i; dist < hi; dist += 16)
                if (!ahead || dist > 0) sum += grad[mid + (ahead ? dist : -dist)];
            if (rest)
                for (int dist = 1 + i; dist <= mid; dist += 16) sum += grad[mid + dist];
            sum = row16_sum(sum);
            if (i == 0 && bucket < a.buckets) {
                if (last)
                    for (int w = 0; w < NW; ++w) sum += far_sum[ahead][w];
                if (rest)
                    for (int w = 0; w < NW; ++w) sum += far_sum[1][w];
                out[t] = sum;
            }
        }
    }
}

// dtable[t][h] = the sum of its partial sums over batch entries and row blocks: a wave per (t, h), in 64 bits.
__device__ __forceinline__ void sum_table(const BwdArgs& a, int id, int lane) {
    if (id >= a.buckets * a.in.heads) return;
    const int t = id % a.buckets, h = id / a.buckets;
    double sum = 0.0;
    const int n = a.in.batch * a.row_blocks;
    for (int i = lane; i < n; i += 64) {
        const int b = i / a.row_blocks, blk = i - b * a.row_blocks;
        sum += (double)a.part_table[(((int64_t)b * a.in.heads + h) * a.row_blocks + blk) * a.buckets + t];
    }
    sum = wave_sum_f64(sum);
    if (lane == 0) a.d_table[t * a.d_table_stride + h] = (float)sum;
}

// ---- dK, dV ----------------------------------------------------------------------------
// WR waves of 32 keys each, times WK that share the keys and take HALVES x 32 queries each
// of a tile; their results meet in LDS in wave order.
template <typename T, int DP, bool BIAS, int WR, int WK, int HALVES>
__global__ __launch_bounds__(64 * WR * WK, sizeof(T) == 2 && DP == 64 ? 2 : 1) void attn_dkv_kernel(const BwdArgs a) {
    typedef Tile<T, DP> Tl;
    constexpr int MY = 32 * HALVES, QB = MY * WK, TILE = QB * Tl::RB, NW = WR * WK, SL = QB < 64 ? 64 : QB;
    static_assert(WR * (WK - 1) * 2 * Tl::BLOCKS * 16 * 256 <= 4 * TILE, "the waves' results take the tiles' place");
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];  // [buffer][Q | dO], [buffer][ref | delta], bias line
    const AttnIn& in = a.in;
    float* const stats = reinterpret_cast<float*>(smem + 4 * TILE);  // [buffer][2][SL]
    float* const line = stats + 2 * 2 * SL;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // The launch's first workgroups add up the table's gradient.
    if (BIAS && blockIdx.x < (uint32_t)a.table_blocks) {
        sum_table(a, (int)blockIdx.x * NW + wave, lane);
        return;
    }
    const uint32_t bid = BIAS ? blockIdx.x - a.table_blocks : xcd_block();
    const int blk = (int)(bid % (uint32_t)a.key_blocks), rest = (int)(bid / (uint32_t)a.key_blocks);
    const int range = rest % a.ranges, bh = rest / a.ranges, b = bh % in.batch, kvh = bh / in.batch;
    const int r = lane & 31, g = lane >> 5, wr = wave % WR, wk = wave / WR;
    const int key = (blk * WR + wr) * 32 + r, len = kept_len(in, b);
    const bool keep = key < len && (!in.kv_mask || in.kv_mask[b * in.mask_stride + key] != 0);
    const bool inside = key < in.seq_kv;

    typename Tl::Frag kf[Tl::STEPS], vf[Tl::STEPS];
    {
        // A key that is not kept is taken as zeros: what it holds reaches no product.
        const int64_t n = keep ? key : 0;
        const T* kp = reinterpret_cast<const T*>(in.k) + b * in.ks[0] + n * in.ks[1] + kvh * in.ks[2];
        const T* vp = reinterpret_cast<const T*>(in.v) + b * in.vs[0] + n * in.vs[1] + kvh * in.vs[2];
#pragma unroll
        for (int c = 0; c < Tl::STEPS; ++c) {
            kf[c] = keep ? frag_global<T>(kp, c, g, in.dim) : frag_zero<T>();
            vf[c] = keep ? frag_global<T>(vp, c, g, in.dim) : frag_zero<T>();
        }
    }
    f32x16_t dk[Tl::BLOCKS], dv[Tl::BLOCKS];
#pragma unroll
    for (int d = 0; d < Tl::BLOCKS; ++d) dk[d] = dv[d] = zero16();
    const typename Tl::Cols cols = Tl::cols(lane);

    // Query tiles of the heads that share this key head, one after another; this range's.
    const int tiles = (in.seq_q + QB - 1) / QB;
    const int64_t total = (int64_t)tiles * in.shared;
    int first = (int)(total * range / a.ranges), last = (int)(total * (range + 1) / a.ranges);
    if (__syncthreads_or(keep) == 0) last = first;  // no kept key in the block
    const int pos = BIAS ? rel_position(in.rel, b) : 0;

    typename Tl::template Loads<QB, NW> ql, gl;
    ql.init(in.qs[1], in.dim, wave, lane);
    gl.init(a.dos[1], in.dim, wave, lane);
    auto issue = [&](int n, int buf) {
        const int h = kvh * in.shared + n / tiles, q0 = (n % tiles) * QB;
        const int left = in.seq_q - q0;
        uint8_t* qb = smem + buf * 2 * TILE;
        const T* qp = reinterpret_cast<const T*>(in.q) + b * in.qs[0] + (int64_t)q0 * in.qs[1] + h * in.qs[2];
        const T* gp = reinterpret_cast<const T*>(a.d_o) + b * a.dos[0] + (int64_t)q0 * a.dos[1] + h * a.dos[2];
        if (left >= QB) {
            ql.issue_all(qp, qb, wave);
            gl.issue_all(gp, qb + TILE, wave);
        } else {
            const auto keep = [&](int i) { return i < left; };
            ql.issue(qp, qb, wave, lane, keep);
            gl.issue(gp, qb + TILE, wave, lane, keep);
        }
#pragma unroll
        for (int i = 0; i < 2 * SL / 64; ++i) {  // 64 floats an instruction: ref's, then delta's
            if (i % NW != wave) continue;
            const int which = i / (SL / 64), at = i % (SL / 64) * 64 + lane;
            const float* src = (which == 0 ? a.ref : a.delta) + ((int64_t)b * in.heads + h) * in.seq_q + q0;
            lds_dma4(src, at < min(left, QB) ? 4 * at : kOutOfBuffer, stats + (buf * 2 + which) * SL + i % (SL / 64) * 64);
        }
    };
    int cur = -1, buf = 0;
    if (first < last) issue(first, 0);
    for (int n = first; n < last; ++n) {
        wait_vmem<0>();
        wait_lds();
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (BIAS) {
            if (n / tiles != cur) {  // every wave has finished with the last head's line
                cur = n / tiles;
                rel_line(in.rel, kvh * in.shared + cur, line, tid, 64 * NW);
                __syncthreads();
            }
            // Queries past the last one: their weight is 0 by a reference of +inf.  The bias of their
            // offset is finite, but alone above 88.7 exp of it is not.
            const int left = in.seq_q - (n % tiles) * QB;
            if (left < QB) {
                float* ref = stats + buf * 2 * SL;
                for (int i = left + tid; i < QB; i += 64 * NW) ref[i] = INFINITY;
                __syncthreads();
            }
        }
        if (n + 1 < last) issue(n + 1, buf ^ 1);
        const uint8_t* Qt = smem + buf * 2 * TILE + MY * wk * Tl::RB;
        const uint8_t* Gt = Qt + TILE;
        const float* st = stats + buf * 2 * SL + MY * wk;
        const int q0 = (n % tiles) * QB + MY * wk;
        f32x16_t s[HALVES], ds[HALVES];
        FragParts<T> pf[HALVES][2], df[HALVES][2];
        auto scores = [&](auto hc, auto vc, auto side) {
            constexpr int hh = decltype(hc)::value;
            s[hh] = ds[hh] = zero16();
            products<T, 2 * Tl::STEPS, 1, decltype(vc)::value>(
                [&](int i) { return Tl::row_frag(i & 1 ? Gt : Qt, 32 * hh + r, i / 2, g); },
                [&](int i, const typename Tl::Frag& f) {
                    if (i & 1) ds[hh] = mma(f, vf[i / 2], ds[hh]);
                    else s[hh] = mma(f, kf[i / 2], s[hh]);
                },
                side);
        };
        // P and dS of elements 4 i4 .. + 3: queries q0 + 32 hh + 8 i4 + 4 g + e.  A query past the
        // last one is a row of zeros with weight 1 (its ref and delta are 0 too), with a bias of
        // weight 0: it adds nothing; a key that is not kept has a lane of its own, which is not stored.
        auto weights = [&](auto hc, int i4) {
            constexpr int hh = decltype(hc)::value;
            const int i0 = 32 * hh + 4 * g + 8 * i4;
            const float4 rf = *reinterpret_cast<const float4*>(st + i0);
            const float4 dl = *reinterpret_cast<const float4*>(st + SL + i0);
            const float ref[4] = {rf.x, rf.y, rf.z, rf.w}, delta[4] = {dl.x, dl.y, dl.z, dl.w};
            float p[4], d[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float c = -ref[e];
                // Offsets fall by one from query to query.
                if constexpr (BIAS) c += rel_at(line, in.rel.reach, key - (q0 + 32 * hh + 4 * g) - pos - 27)[27 - 8 * i4 - e];
                p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[hh][4 * i4 + e], in.scale_log2, c));
                d[e] = p[e] * (ds[hh][4 * i4 + e] - delta[e]);
            }
            pf[hh][i4 / 2].set(i4 & 1, p);
            df[hh][i4 / 2].set(i4 & 1, d);
        };
        auto some = [&](auto hc) {
            return [&, hc](int part, int of) {
#pragma unroll
                for (int i4 = 0; i4 < 4; ++i4)
                    if (i4 * of / 4 == part) weights(hc, i4);
            };
        };
        auto grads = [&](auto hc, auto vc, auto side) {
            constexpr int hh = decltype(hc)::value;
            products<T, 4 * Tl::BLOCKS, 2, decltype(vc)::value>(
                [&](int i) { return Tl::col_frag(i & 1 ? Qt : Gt, 32 * hh + 16 * (i / 2 / Tl::BLOCKS), i / 2 % Tl::BLOCKS, cols); },
                [&](int i, const typename Tl::Frag& f) {
                    const int j = i / 2 / Tl::BLOCKS, d = i / 2 % Tl::BLOCKS;
                    if (i & 1) dk[d] = mma(f, df[hh][j].frag(), dk[d]);
                    else dv[d] = mma(f, pf[hh][j].frag(), dv[d]);
                },
                side);
        };
        // One half's weights between the other half's products.
        using H0 = std::integral_constant<int, 0>;
        using H1 = std::integral_constant<int, HALVES - 1>;
        using None = std::integral_constant<int, 0>;
        using SV = std::integral_constant<int, DP == 64 ? 18 : 9>;   // vector instructions per product
        using GV = std::integral_constant<int, DP == 64 ? 18 : 9>;
        scores(H0{}, None{}, NoSide{});
        if constexpr (HALVES == 2) {
            scores(H1{}, SV{}, some(H0{}));
            grads(H0{}, GV{}, some(H1{}));
        } else {
#pragma unroll
            for (int i4 = 0; i4 < 4; ++i4) weights(H0{}, i4);
        }
        grads(H1{}, None{}, NoSide{});
        buf ^= 1;
    }
    if constexpr (WK > 1) {  // the other waves' sums, in wave order
        float* part = reinterpret_cast<float*>(smem) + lane;
        constexpr int N = 2 * Tl::BLOCKS * 16 * 64;
        __syncthreads();  // every wave has read its last tile
        if (wk > 0) {
#pragma unroll
            for (int d = 0; d < Tl::BLOCKS; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    part[((wk - 1) * WR + wr) * N + (32 * d + e) * 64] = dk[d][e];
                    part[((wk - 1) * WR + wr) * N + (32 * d + 16 + e) * 64] = dv[d][e];
                }
        }
        __syncthreads();
        if (wk > 0) return;
#pragma unroll
        for (int w = 0; w < WK - 1; ++w)
#pragma unroll
            for (int d = 0; d < Tl::BLOCKS; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    dk[d][e] += part[(w * WR + wr) * N + (32 * d + e) * 64];
                    dv[d][e] += part[(w * WR + wr) * N + (32 * d + 16 + e) * 64];
                }
    }
    if (!inside) return;
    if (!keep) {
#pragma unroll
        for (int d = 0; d < Tl::BLOCKS; ++d) dk[d] = dv[d] = zero16();
    }
    if (a.ranges > 1) {
        const int64_t plane = (int64_t)in.batch * in.kv_heads * in.seq_kv * DP;
        float* pk = a.part_kv + (int64_t)range * 2 * plane + (((int64_t)b * in.kv_heads + kvh) * in.seq_kv + key) * DP;
#pragma unroll
        for (int d = 0; d < Tl::BLOCKS; ++d)
#pragma unroll
            for (int i4 = 0; i4 < 4; ++i4) {
                const int e0 = 32 * d + 8 * i4 + 4 * g;
                const float x[4] = {dk[d][4 * i4], dk[d][4 * i4 + 1], dk[d][4 * i4 + 2], dk[d][4 * i4 + 3]};
                const float y[4] = {dv[d][4 * i4], dv[d][4 * i4 + 1], dv[d][4 * i4 + 2], dv[d][4 * i4 + 3]};
                if (e0 < in.dim) {
                    put4(pk + e0, x);
                    put4(pk + plane + e0, y);
                }
            }
        return;
    }
    T* kp = reinterpret_cast<T*>(a.dk) + b * a.dks[0] + (int64_t)key * a.dks[1] + kvh * a.dks[2];
    T* vp = reinterpret_cast<T*>(a.dv) + b * a.dvs[0] + (int64_t)key * a.dvs[1] + kvh * a.dvs[2];
#pragma unroll
    for (int d = 0; d < Tl::BLOCKS; ++d)
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) {
            const int e0 = 32 * d + 8 * i4 + 4 * g;
            float x[4], y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[e] = dk[d][4 * i4 + e] * in.scale;
                y[e] = dv[d][4 * i4 + e];
            }
            if (e0 < in.dim) {
                put4(kp + e0, x);
                put4(vp + e0, y);
            }
        }
}

// The ranges' dK and dV of one key, added in range order: a thread per four elements.
template <typename T, int DP>
__global__ __launch_bounds__(256) void attn_dkv_join_kernel(const BwdArgs a) {
    const AttnIn& in = a.in;
    constexpr int TPR = DP / 4;
    const int64_t n = (int64_t)in.batch * in.kv_heads * in.seq_kv, id = ((int64_t)blockIdx.x * 256 + threadIdx.x) / TPR;
    const int d = (int)(threadIdx.x % TPR) * 4;
    if (id >= n || d >= in.dim) return;
    const int key = (int)(id % in.seq_kv), bh = (int)(id / in.seq_kv), kvh = bh % in.kv_heads, b = bh / in.kv_heads;
    float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < a.ranges; ++s) {
        const float* p = a.part_kv + ((int64_t)s * 2 * n + id) * DP + d;
        const float4 u = *reinterpret_cast<const float4*>(p), w = *reinterpret_cast<const float4*>(p + n * DP);
        x[0] += u.x;
        x[1] += u.y;
        x[2] += u.z;
        x[3] += u.w;
        y[0] += w.x;
        y[1] += w.y;
        y[2] += w.z;
        y[3] += w.w;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] *= in.scale;
    put4(reinterpret_cast<T*>(a.dk) + b * a.dks[0] + (int64_t)key * a.dks[1] + kvh * a.dks[2] + d, x);
    put4(reinterpret_cast<T*>(a.dv) + b * a.dvs[0] + (int64_t)key * a.dvs[1] + kvh * a.dvs[2] + d, y);
}

// ---- launch ------------------------------------------------------------------------------
struct Plan {
    int row_high, key_high;     // rows (keys) of a workgroup: 128, or 32 with waves that share them
    bool row_pairs;             // 128 rows by eight waves
    int row_blocks, key_blocks, ranges;
    int64_t stat_floats, table_floats, kv_floats;  // workspace, in this order (ref and delta first)
};

int64_t up4(int64_t n) { return (n + 3) / 4 * 4; }

Plan plan(const AttnIn& in, bool bf16_io, int buckets, int cus) {
    Plan p{};
    const int dp = in.dim <= 64 ? 64 : 128;
    const int64_t rows = (int64_t)in.heads * in.batch, keys = (int64_t)in.kv_heads * in.batch;
    // 128 rows a workgroup while that gives half the CUs one (bwd, 16 heads x 128, 512 keys: 128 blocks
    // 43.0 us, in 32 rows 48.5; 64 blocks 36.9 and 30.8; 128 blocks at 2048 keys 93 and 102, with a
    // bias 187 and 207; but 128 blocks at width 64 59 and 53, in fp32 366 and 293, and 96 at width
    // 128 84 and 91); up to one per CU by eight waves (bf16 without a bias, whose lines take the
    // second tile's place).
    const int64_t wide = (int64_t)((in.seq_q + 127) / 128) * rows;
    p.row_high = wide * 2 >= cus ? 128 : 32;
    p.row_pairs = p.row_high == 128 && wide <= cus && bf16_io && buckets == 0 && in.seq_kv > 64;
    p.row_blocks = (in.seq_q + p.row_high - 1) / p.row_high;
    // 128 keys, whose queries can be shared in up to 16 ranges of at least 128, while that gives
    // every CU a workgroup.
    const int64_t tall = (int64_t)((in.seq_kv + 127) / 128) * keys;
    int64_t most = (int64_t)((in.seq_q + 127) / 128) * in.shared;
    if (most > 16) most = 16;
    p.key_high = tall * most >= cus ? 128 : 32;
    // bf16 with up to 2048 queries whose 32-key blocks give half the CUs a workgroup: those, with no
    // ranges to join (16 heads x 4 batch entries, 64 wide, bwd: 1024 queries, 77 keys
    // 28.2 -> 25.1 us; 2048, 512 keys, one entry 42.8 -> 35.4; 2048, 77 keys 44.8 -> 45.8; 4096, 77
    // keys would be 72.1 -> 81.2: the four waves' query tiles are four times the loads).
    const int64_t narrow = (int64_t)((in.seq_kv + 31) / 32) * keys;
    if (bf16_io && (int64_t)in.seq_q * in.shared <= 2048 && tall * 2 <= cus && narrow * 2 >= cus) p.key_high = 32;
    p.key_blocks = (in.seq_kv + p.key_high - 1) / p.key_high;
    const int64_t blocks = p.key_blocks * keys;
    int64_t s = blocks > 0 ? cus / blocks : 1;
    if (s > most) s = most;
    p.ranges = s < 2 ? 1 : (int)s;
    p.stat_floats = up4(rows * in.seq_q);
    p.table_floats = buckets ? up4(rows * p.row_blocks * buckets) : 0;
    p.kv_floats = p.ranges > 1 ? (int64_t)p.ranges * 2 * keys * in.seq_kv * dp : 0;
    return p;
}

template <typename T, int DP, bool BIAS, int WR, int WK, int HALVES>
void launch_dq(const BwdArgs& a, int64_t blocks, hipStream_t st) {
    const size_t lds = 4 * 32 * HALVES * WK * Tile<T, DP>::RB +
                       (BIAS ? (1 + WR * WK) * rel_line_len(a.in.rel.reach) + WR * WK * kScratch : 0) * sizeof(float);
    hipLaunchKernelGGL((attn_dq_kernel<T, DP, BIAS, WR, WK, HALVES>), dim3((unsigned)blocks), dim3(64 * WR * WK), lds, st, a);
}
template <typename T, int DP, bool BIAS, int WR, int WK, int HALVES>
void launch_dkv(const BwdArgs& a, int64_t blocks, hipStream_t st) {
    constexpr int QB = 32 * HALVES * WK;
    const size_t lds = 4 * QB * Tile<T, DP>::RB + (4 * (QB < 64 ? 64 : QB) + (BIAS ? rel_line_len(a.in.rel.reach) : 0)) * sizeof(float);
    hipLaunchKernelGGL((attn_dkv_kernel<T, DP, BIAS, WR, WK, HALVES>), dim3((unsigned)blocks), dim3(64 * WR * WK), lds, st, a);
}

template <typename T, int DP, bool BIAS>
int launch(const BwdArgs& a, const Plan& p, hipStream_t st) {
    const char* who = "dt_attn_bwd";
    const AttnIn& in = a.in;
    const int64_t dq_blocks = (int64_t)p.row_blocks * in.heads * in.batch;
    const int64_t dkv_blocks = (int64_t)p.key_blocks * p.ranges * in.kv_heads * in.batch;
    DT_REQUIRE(dq_blocks < (1ll << 31) && dkv_blocks < (1ll << 31), "%s: grid too large", who);
    constexpr int H = halves<T, DP>(), FEW = few_waves<T, DP, BIAS>();
    int rc = DT_OK;
    if (dq_blocks > 0) {
        if (p.row_high == 32) {
            launch_dq<T, DP, BIAS, 1, FEW, 1>(a, dq_blocks, st);
        } else if (p.row_pairs) {
            if constexpr (sizeof(T) == 2 && !BIAS) launch_dq<T, DP, BIAS, 4, 2, 2>(a, dq_blocks, st);
        } else {
            launch_dq<T, DP, BIAS, 4, 1, H>(a, dq_blocks, st);
        }
        rc = check_launch(who);
    }
    constexpr int KW = Tile<T, DP>::RB <= 256 ? 4 : 2;
    BwdArgs k = a;
    const int waves = p.key_high == 32 ? KW : 4;
    k.table_blocks = BIAS && a.d_table ? (a.buckets * in.heads + waves - 1) / waves : 0;
    const int64_t blocks = dkv_blocks + k.table_blocks;
    DT_REQUIRE(blocks < (1ll << 31), "%s: grid too large", who);
    if (rc || blocks == 0) return rc;
    if (p.key_high == 32) launch_dkv<T, DP, BIAS, 1, KW, 1>(k, blocks, st);
    else launch_dkv<T, DP, BIAS, 4, 1, H>(k, blocks, st);
    rc = check_launch(who);
    if (rc || p.ranges == 1 || dkv_blocks == 0) return rc;
    const int64_t n = (int64_t)in.batch * in.kv_heads * in.seq_kv * (DP / 4);
    hipLaunchKernelGGL((attn_dkv_join_kernel<T, DP>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, a);
    return check_launch(who);
}

template <typename T, int DP>
int launch_bias(const BwdArgs& a, const Plan& p, hipStream_t st) {
    return a.in.rel.table ? launch<T, DP, true>(a, p, st) : launch<T, DP, false>(a, p, st);
}

int64_t total_floats(const Plan& p) { return 2 * p.stat_floats + p.table_floats + p.kv_floats; }

}  // namespace
}  // namespace attn
}  // namespace dit

extern "C" size_t dt_attn_bwd_workspace_bytes(const dt_attn_args* x) {
    using namespace dit;
    using namespace dit::attn;
    AttnIn in;
    if (prepare_in(x, "dt_attn_bwd_workspace_bytes", &in)) return 0;
    return (size_t)total_floats(plan(in, x->io_type == DT_TYPE_BF16, x->rel_table ? x->rel_buckets : 0, cu_count())) * sizeof(float);
}

extern "C" int dt_attn_bwd(const dt_attn_args* x, const dt_attn_grads* y, void* workspace, size_t workspace_bytes,
                           dt_stream_t stream) {
    using namespace dit;
    using namespace dit::attn;
    const char* who = "dt_attn_bwd";
    BwdArgs a{};
    int rc = prepare_in(x, who, &a.in);
    if (rc) return rc;
    DT_REQUIRE(y != nullptr, "%s: null gradients", who);
    rc = check_rows(x, y->d_o, y->d_o_strides, x->heads, x->seq_q, false, "d_o", who);
    if (!rc) rc = check_rows(x, y->o, y->o_strides, x->heads, x->seq_q, false, "o", who);
    if (!rc) rc = check_rows(x, y->dq, y->dq_strides, x->heads, x->seq_q, true, "dq", who);
    if (!rc) rc = check_rows(x, y->dk, y->dk_strides, x->kv_heads, x->seq_kv, true, "dk", who);
    if (!rc) rc = check_rows(x, y->dv, y->dv_strides, x->kv_heads, x->seq_kv, true, "dv", who);
    if (rc) return rc;
    const AttnIn& in = a.in;
    const bool rows = in.batch > 0 && in.heads > 0 && in.seq_q > 0;
    DT_REQUIRE(!rows || (y->lse && ((uintptr_t)y->lse & 3) == 0), "%s: lse must be given, 4-byte aligned", who);
    DT_REQUIRE(!x->rel_table || !y->d_rel_table || (((uintptr_t)y->d_rel_table & 3) == 0 && y->d_rel_table_stride >= x->heads),
               "%s: d_rel_table must be 4-byte aligned with rows of at least heads", who);
    a.buckets = x->rel_table ? x->rel_buckets : 0;
    const Plan p = plan(in, x->io_type == DT_TYPE_BF16, a.buckets, cu_count());
    const size_t need = (size_t)total_floats(p) * sizeof(float);
    DT_REQUIRE(need == 0 || (workspace && aligned16(workspace) && workspace_bytes >= need),
               "%s: workspace of %zu bytes (16-byte aligned) needed, %zu given", who, need, workspace ? workspace_bytes : 0);
    a.d_o = y->d_o;
    a.o = y->o;
    a.lse = y->lse;
    a.dq = y->dq;
    a.dk = y->dk;
    a.dv = y->dv;
    for (int i = 0; i < 3; ++i) {
        a.dos[i] = y->d_o_strides[i];
        a.os[i] = y->o_strides[i];
        a.dqs[i] = y->dq_strides[i];
        a.dks[i] = y->dk_strides[i];
        a.dvs[i] = y->dv_strides[i];
    }
    a.ref = (float*)workspace;
    a.delta = a.ref + p.stat_floats;
    a.part_table = a.delta + p.stat_floats;
    a.part_kv = a.part_table + p.table_floats;
    a.d_table = y->d_rel_table;
    a.d_table_stride = y->d_rel_table_stride;
    a.row_blocks = p.row_blocks;
    a.key_blocks = p.key_blocks;
    a.ranges = p.ranges;
    const hipStream_t st = (hipStream_t)stream;
    if (x->io_type == DT_TYPE_F32) return in.dim <= 64 ? launch_bias<float, 64>(a, p, st) : launch_bias<float, 128>(a, p, st);
    return in.dim <= 64 ? launch_bias<bf16, 64>(a, p, st) : launch_bias<bf16, 128>(a, p, st);
}
