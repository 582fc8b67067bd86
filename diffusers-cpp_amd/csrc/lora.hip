// lora.hip -- the down projection of dt_lora_gemm: T[m, r] = scale_a sum_k x[m, k]
// A_a[r, k], a = adapter of row m, as two bf16 parts for the product's
// kernels (gemm.hip).
//
// A stream of x and of the used adapters with next to no arithmetic.  A workgroup takes 16
// or 32 rows and 16 or 32 ranks; its waves take every NW-th 64 k and meet in LDS, in wave order.  Each
// streams its rows and ranks x 64 of x and of the adapter through LDS buffers of its own by
// direct DMA, whole 128-byte lines of a row side by side: read straight into the MFMA's
// registers, lanes next to each other lie in different rows, and the vector cache
// looks up every lane for itself, 16 bytes a cycle (4608 rows x 4096, rank 32: 27 us; so 16.5).
// The adapters of the 16 rows are found by ballot and taken one after another, or,
// when there are few rows, by workgroups of their own.
#include "capi_util.hpp"
#include "common.hpp"
#include "kernels.hpp"

namespace dit {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

struct DownArgs {
    const uint16_t* x;
    int64_t ldx;
    const uint16_t* a;
    int64_t lda, a_stride;
    const float* scale;
    const int32_t* row_adapter;
    uint16_t* t;  // [M][2][rp]
    int M, K, adapters, rank, rp, slots;
};

// Elements k .. k + 7 of a row of K; zeros past its end.
__device__ __forceinline__ uint4 load8(const uint16_t* row, int k, int K) {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t lo = k + 2 * e < K ? row[k + 2 * e] : 0u, hi = k + 2 * e + 1 < K ? row[k + 2 * e + 1] : 0u;
        w[e] = lo | hi << 16;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

constexpr int kLine = 64;   // k a wave takes at a time

struct Out {  // a thread's element of T: row tid / RANKS, rank tid % RANKS
    const DownArgs& p;
    int m, rank, theirs;
    __device__ __forceinline__ void put(float v) const {
        const uint32_t hi = f32_to_bf16_bits(v);
        const float h = __uint_as_float(hi << 16);
        // The rest; none behind a value beyond bf16's range.
        const float lo = (hi & 0x7FFFu) < 0x7F80u ? v - h : 0.f;
        uint16_t* o = p.t + (int64_t)m * 2 * p.rp + rank;
        o[0] = (uint16_t)hi;
        o[p.rp] = (uint16_t)f32_to_bf16_bits(lo);
    }
};

// VEC: rows in whole 16-byte chunks, through LDS.  Else element by element, for any layout.
template <bool VEC, int ROWS, int NW, int NB, int RANKS>
__global__ __launch_bounds__(64 * NW) void lora_down_kernel(const DownArgs p) {
    constexpr int ROWB = kLine * 2, BUF = (ROWS + RANKS) * ROWB, RF = ROWS / 16, AF = RANKS / 16;  // NB buffers of a wave
    constexpr int DMAS = BUF / 1024, PARTB = NW * ROWS * (RANKS + 1) * 4;
    __shared__ __attribute__((aligned(16))) uint8_t smem[VEC && NW * NB * BUF > PARTB ? NW * NB * BUF : PARTB];
    float(*const part)[ROWS][RANKS + 1] = reinterpret_cast<float(*)[ROWS][RANKS + 1]>(smem);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, g = lane >> 4;
    const int m0 = blockIdx.x * ROWS, r0 = blockIdx.y * RANKS, slot = blockIdx.z;
    // Lane i < ROWS has row i's adapter.
    int mine = lane < ROWS && m0 + lane < p.M ? p.row_adapter[m0 + lane] : -1;
    if (mine >= p.adapters) mine = -1;
    const int lines = (p.K + kLine - 1) / kLine;
    constexpr int STEP = 64 * NW / RANKS, OUTS = ROWS / STEP > 1 ? ROWS / STEP : 1;  // elements of T a thread has
    auto each_out = [&](auto f) {
#pragma unroll
        for (int o = 0; o < OUTS; ++o) {
            const int row = tid / RANKS + STEP * o;
            const int theirs = __shfl(mine, row & (ROWS - 1));
            if (row < ROWS && m0 + row < p.M) f(Out{p, m0 + row, r0 + tid % RANKS, theirs}, row);
        }
    };
    if (slot == 0)
        each_out([](const Out& o, int) {
            if (o.theirs < 0) o.put(0.f);
        });

    uint64_t left = __builtin_amdgcn_ballot_w64(mine >= 0);
    for (int turn = 0; left; ++turn) {
        const int a = __builtin_amdgcn_readlane(mine, (int)__builtin_ctzll(left));
        const uint64_t of = __builtin_amdgcn_ballot_w64(mine == a);
        left &= ~of;
        if (turn % p.slots != slot) continue;
        f32x4_t acc[RF][AF];
#pragma unroll
        for (int f = 0; f < RF; ++f)
#pragma unroll
            for (int h = 0; h < AF; ++h) acc[f][h] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        auto multiply = [&](const uint4 (&v)[RF + AF]) {  // 16 rows of x each, then 16 of the adapter each
#pragma unroll
            for (int f = 0; f < RF; ++f)
#pragma unroll
                for (int h = 0; h < AF; ++h)
                    acc[f][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, v[RF + h]),
                                                                        __builtin_bit_cast(bf16x8_t, v[f]), acc[f][h], 0, 0, 0);
        };
        if constexpr (VEC) {
            // Instruction j covers buffer rows 8 j .. + 7 (x, then the adapter), lane i chunk
            // i % 8 of row i / 8, stored at chunk ^ (row & 7).  Rows past the ends, of other
            // adapters, and k past K are zeros.
            uint8_t* const mem = smem + wave * NB * BUF;
            const uint16_t* xb = p.x + (int64_t)m0 * p.ldx;
            const uint16_t* ab = p.a + a * p.a_stride + (int64_t)r0 * p.lda;
            const int chunk = (lane & 7) ^ (lane >> 3);
            uint32_t off[DMAS];
#pragma unroll
            for (int j = 0; j < DMAS; ++j) {
                const int row = 8 * j + (lane >> 3), rank = row - ROWS;
                const bool there = row < ROWS ? (of >> row) & 1 : r0 + rank < p.rank;
                off[j] = there ? (uint32_t)((row < ROWS ? row * p.ldx : rank * p.lda) * 2 + chunk * 16) : kOutOfBuffer;
            }
            auto issue = [&](int line, int buf) {
                const bool tail = line * kLine + chunk * 8 >= p.K;  // lines past the last one too
#pragma unroll
                for (int j = 0; j < DMAS; ++j)
                    lds_dma16((8 * j < ROWS ? xb : ab) + (int64_t)line * kLine, tail ? kOutOfBuffer : off[j], mem + buf * BUF + 1024 * j);
            };
#pragma unroll
            for (int i = 0; i < NB - 1; ++i) issue(wave + i * NW, i);
            int buf = 0;
            for (int line = wave; line < lines; line += NW) {
                issue(line + (NB - 1) * NW, buf == 0 ? NB - 1 : buf - 1);  // the one read last
                __builtin_amdgcn_s_waitcnt(((NB - 1) * DMAS & 15) | (((NB - 1) * DMAS >> 4) << 14) | 0x0F70);
                __builtin_amdgcn_sched_barrier(0);
                const uint8_t* t = mem + buf * BUF;
                uint4 v[2][RF + AF];
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int h = 0; h < RF + AF; ++h)
                        v[s][h] = *reinterpret_cast<const uint4*>(t + (16 * h + r) * ROWB + (((4 * s + g) ^ (r & 7)) << 4));
#pragma unroll
                for (int s = 0; s < 2; ++s) multiply(v[s]);
                __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the buffer is read
                __builtin_amdgcn_sched_barrier(0);
                buf = buf == NB - 1 ? 0 : buf + 1;
            }
            __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): the DMA past the end is in LDS before it is used again
        } else {
            const uint16_t* row[RF + AF];
#pragma unroll
            for (int h = 0; h < RF + AF; ++h)
                row[h] = h < RF ? p.x + (int64_t)min(m0 + 16 * h + r, p.M - 1) * p.ldx
                                : p.a + a * p.a_stride + (int64_t)min(r0 + 16 * (h - RF) + r, p.rank - 1) * p.lda;
            for (int line = wave; line < lines; line += NW)
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    uint4 v[RF + AF];
#pragma unroll
                    for (int h = 0; h < RF + AF; ++h) v[h] = load8(row[h], line * kLine + 32 * s + 8 * g, p.K);
                    multiply(v);
                }
        }
        __syncthreads();
#pragma unroll
        for (int f = 0; f < RF; ++f)
#pragma unroll
            for (int h = 0; h < AF; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) part[wave][16 * f + r][16 * h + 4 * g + i] = acc[f][h][i];
        __syncthreads();
        each_out([&](const Out& o, int row) {
            if (o.theirs != a) return;
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < NW; ++w) v += part[w][row][tid % RANKS];
            if (o.rank >= p.rank) v = 0.f;
            o.put(p.scale ? v * p.scale[a] : v);
        });
        __syncthreads();  // the sums have been read
    }
}

}  // namespace

int lora_down(const uint16_t* x, int64_t ldx, int64_t M, int64_t K, const dt_lora& l, uint16_t* t, hipStream_t st) {
    DownArgs p{};
    p.x = x;
    p.ldx = ldx;
    p.a = (const uint16_t*)l.a;
    p.lda = l.lda;
    p.a_stride = l.a_stride;
    p.scale = l.scale;
    p.row_adapter = l.row_adapter;
    p.t = t;
    p.M = (int)M;
    p.K = (int)K;
    p.adapters = (int)l.adapters;
    p.rank = (int)l.rank;
    p.rp = (int)lora_rank_padded(l.rank);
    // Rows in whole chunks, a tile's within 2^31 bytes.
    const bool vec = K % 8 == 0 && ldx % 8 == 0 && l.lda % 8 == 0 && (l.a_stride % 8 == 0 || l.adapters == 1) &&
                     aligned16(x) && aligned16(l.a) && ldx < (1 << 25) && l.lda < (1 << 25);
    // 16 rows a workgroup while that gives each CU one at most, else 32: the adapter is read
    // again for every workgroup.  While 16 rows x 16 ranks give half the CUs one at most, those, by
    // sixteen waves (K 4096, cold: 16 rows with 16 adapters of rank 64 11.8 -> 8.8 us, one row 8.5 -> 6.0;
    // 1628 rows x 2560 would be 7.2 -> 8.6: x is read again for every 16 ranks).
    const int64_t few = (M + 15) / 16;
    const bool small = vec && few * (p.rp / 32) <= cu_count(), tiny = vec && few * (p.rp / 16) * 2 <= cu_count();
    const int64_t high = small ? 16 : 32, tiles = (M + high - 1) / high, blocks = p.rp / (tiny ? 16 : 32);
    // Adapters of a tile side by side until the chip is full: at most one for each of its rows.
    int64_t slots = cu_count() / (tiles * blocks);
    const int64_t rows = M < high ? M : high, most = l.adapters < rows ? l.adapters : rows;
    slots = slots < 1 ? 1 : slots < most ? slots : most;
    p.slots = (int)slots;
    const dim3 grid((unsigned)tiles, (unsigned)blocks, (unsigned)slots);
    if (!vec) hipLaunchKernelGGL((lora_down_kernel<false, 32, 8, 1, 32>), grid, dim3(512), 0, st, p);
    else if (tiny) hipLaunchKernelGGL((lora_down_kernel<true, 16, 16, 2, 16>), grid, dim3(1024), 0, st, p);
    else if (small) hipLaunchKernelGGL((lora_down_kernel<true, 16, 8, 3, 32>), grid, dim3(512), 0, st, p);
    else hipLaunchKernelGGL((lora_down_kernel<true, 32, 8, 2, 32>), grid, dim3(512), 0, st, p);
    return check_launch("dt_lora_gemm");
}

}  // namespace dit
