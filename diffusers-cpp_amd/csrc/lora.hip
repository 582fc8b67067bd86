// lora.hip -- the down projection of dt_lora_gemm: T[m, r] = scale_a sum_k x[m, k]
// A_a[r, k], a = adapter of row m, as two bf16 parts for the product's epilogue
// (lora_add in gemm.hip).
//
// A stream of x and of the used adapters with next to no arithmetic.  A workgroup takes 32
// rows and 32 ranks; its sixteen waves share K, read both operands straight into
// the MFMA's registers (v_mfma_f32_32x32x16_bf16, the adapter's rows as A, the rows of x
// as B) and meet in LDS, in wave order.  The adapters of the 32 rows are found by ballot
// and taken one after another, or, when there are few rows, by workgroups of their own.
#include "capi_util.hpp"
#include "common.hpp"
#include "kernels.hpp"

namespace dit {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));

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
template <bool VEC>
__device__ __forceinline__ uint4 load8(const uint16_t* row, int k, int K) {
    if constexpr (VEC) return k < K ? *reinterpret_cast<const uint4*>(row + k) : make_uint4(0, 0, 0, 0);
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t lo = k + 2 * e < K ? row[k + 2 * e] : 0u, hi = k + 2 * e + 1 < K ? row[k + 2 * e + 1] : 0u;
        w[e] = lo | hi << 16;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

template <bool VEC>
__global__ __launch_bounds__(1024) void lora_down_kernel(const DownArgs p) {
    constexpr int NW = 16, STEPS = 4;  // waves; 16-k steps loaded together (a 128-byte line of each row)
    __shared__ float part[NW][32][33];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 31, g = lane >> 5;
    const int m0 = blockIdx.x * 32, r0 = blockIdx.y * 32, slot = blockIdx.z;
    const bool row = m0 + r < p.M;
    const int mine = row ? p.row_adapter[m0 + r] : -1;
    const bool valid = mine >= 0 && mine < p.adapters;
    const uint16_t* xr = p.x + (int64_t)min(m0 + r, p.M - 1) * p.ldx;
    // A thread's output: row tid / 32, rank tid % 32.
    const int om = tid >> 5, orank = tid & 31;
    const int theirs = __shfl(mine, om);
    auto put = [&](float v) {
        const uint32_t hi = f32_to_bf16_bits(v);
        const float h = __uint_as_float(hi << 16);
        // The rest; none behind a value beyond bf16's range.
        const float lo = (hi & 0x7FFFu) < 0x7F80u ? v - h : 0.f;
        uint16_t* o = p.t + (int64_t)(m0 + om) * 2 * p.rp + r0 + orank;
        o[0] = (uint16_t)hi;
        o[p.rp] = (uint16_t)f32_to_bf16_bits(lo);
    };
    if (slot == 0 && m0 + om < p.M && !(theirs >= 0 && theirs < p.adapters)) put(0.f);

    // Whole lines per wave: K in ranges of 64.
    const int lines = (p.K + 63) / 64, per = (lines + NW - 1) / NW;
    const int k0 = wave * per * 64, k1 = min(k0 + per * 64, p.K);
    uint64_t left = __builtin_amdgcn_ballot_w64(valid) & 0xFFFFFFFFull;
    for (int turn = 0; left; ++turn) {
        const int a = __builtin_amdgcn_readlane(mine, (int)__builtin_ctzll(left));
        left &= ~__builtin_amdgcn_ballot_w64(mine == a);
        if (turn % p.slots != slot) continue;
        const uint16_t* ar = p.a + a * p.a_stride + (int64_t)min(r0 + r, p.rank - 1) * p.lda;
        f32x16_t acc;
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[e] = 0.f;
        for (int k = k0; k < k1; k += 16 * STEPS) {
            uint4 xv[STEPS], av[STEPS];
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
                xv[s] = load8<VEC>(xr, k + 16 * s + 8 * g, p.K);
                av[s] = load8<VEC>(ar, k + 16 * s + 8 * g, p.K);
            }
#pragma unroll
            for (int s = 0; s < STEPS; ++s)
                acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, av[s]),
                                                              __builtin_bit_cast(bf16x8_t, xv[s]), acc, 0, 0, 0);
        }
        __syncthreads();  // the last adapter's sums have been read
#pragma unroll
        for (int i = 0; i < 16; ++i) part[wave][r][8 * (i >> 2) + 4 * g + (i & 3)] = acc[i];
        __syncthreads();
        if (theirs == a && m0 + om < p.M) {
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < NW; ++w) v += part[w][om][orank];
            if (r0 + orank >= p.rank) v = 0.f;
            put(p.scale ? v * p.scale[a] : v);
        }
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
    const int64_t tiles = (M + 31) / 32, blocks = p.rp / 32;
    // Adapters of a tile side by side until the chip is full: at most the 32 its rows can have.
    int64_t slots = cu_count() / (tiles * blocks);
    const int64_t most = l.adapters < (M < 32 ? M : 32) ? l.adapters : (M < 32 ? M : 32);
    slots = slots < 1 ? 1 : slots < most ? slots : most;
    p.slots = (int)slots;
    const bool vec = K % 8 == 0 && ldx % 8 == 0 && l.lda % 8 == 0 && (l.a_stride % 8 == 0 || l.adapters == 1) &&
                     aligned16(x) && aligned16(l.a);
    const dim3 grid((unsigned)tiles, (unsigned)blocks, (unsigned)slots);
    if (vec) hipLaunchKernelGGL((lora_down_kernel<true>), grid, dim3(1024), 0, st, p);
    else hipLaunchKernelGGL((lora_down_kernel<false>), grid, dim3(1024), 0, st, p);
    return check_launch("dt_lora_gemm");
}

}  // namespace dit
