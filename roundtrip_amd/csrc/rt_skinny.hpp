// rt_skinny.hpp — the feed-forward block's products for few rows (one token, a small serving batch): the weights are read
// once, straight into registers, and that is what bounds it.
//
//   C[m][n] = sum over k of X[m][k] W[k][n],     M <= 16 MT,   W [K][N] with n contiguous
//
// A workgroup of 8 waves makes 64 columns.  In a step of 32 k's lane (g = lane / 16, i = lane % 16) loads the four columns
// 4 i .. of the eight rows 8 g ..: 128-byte (16-bit) or 256-byte runs of W, eight loads of 64 lanes before the first is
// needed, the next step's behind them.  For column c of the four, the eight rows are an operand of one 16x16x32
// matrix instruction as they are (16-bit: after one v_perm for every two values), so nothing passes through LDS; rows of X
// that do not exist are zeros.  Steps are dealt to the waves of all splits in turn; the waves' sums meet in LDS in a fixed
// order, the splits' in gemm_join_kernel.
#pragma once
#include "rt_gemm.hpp"

constexpr int SK_WAVES = 8, SK_COLS = 64;

template <int DT, int DUAL>
struct SkinnyStep {
    typedef typename Elem<DT>::T T;
    struct __attribute__((aligned(4 * ES<DT>))) Four { T t[4]; };
    Four w[DUAL][8];

    // rows k0 + 8 g + j of the lane's four columns, which start at p in row 0
    __device__ __forceinline__ void load(const char* const (&p)[DUAL], long long ld, int k0, int K, int g) {
        if (k0 + 32 <= K) {
#pragma unroll
            for (int d = 0; d < DUAL; ++d)
#pragma unroll
                for (int j = 0; j < 8; ++j) w[d][j] = *(const Four*)(p[d] + (k0 + 8 * g + j) * ld);
        } else {
#pragma unroll
            for (int d = 0; d < DUAL; ++d)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int k = k0 + 8 * g + j;
                    w[d][j] = Four{};
                    if (k < K) w[d][j] = *(const Four*)(p[d] + k * ld);
                }
        }
    }
};

template <int DT, int EPI, int MT>
__global__ __launch_bounds__(64 * SK_WAVES) void skinny_kernel(GemmArgs a) {
    constexpr int DUAL = EPI == EPI_GATED ? 2 : 1;
    typedef SkinnyStep<DT, DUAL> Step;
    __shared__ float sm[SK_WAVES][DUAL][SK_COLS / 4][16][4];          // [wave][..][quad of columns][row][column]: one row tile
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * SK_COLS, split = blockIdx.y, K = (int)a.K, steps = (K + 31) >> 5;
    const int stride = gridDim.y * SK_WAVES;

    const char* p[DUAL];
#pragma unroll
    for (int d = 0; d < DUAL; ++d)
        p[d] = a.w[d] + (long long)(n0 + 4 * i < a.N ? n0 + 4 * i : n0) * ES<DT>;     // columns behind N: any, they are dropped
    f32x4 acc[MT][DUAL][4];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int d = 0; d < DUAL; ++d)
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[t][d][c] = f32x4{0, 0, 0, 0};

    auto use = [&](const Step& s, int k0) __attribute__((always_inline)) {
        u32x4 x[MT][2];                 // k0 + 8 g .. + 7 of row 16 t + i
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const int m = 16 * t + i, k = k0 + 8 * g;
            x[t][0] = x[t][1] = u32x4{0, 0, 0, 0};
            if (m < a.M) {
                const char* q = a.x[0] + m * a.ldx[0] + (long long)k * ES<DT>;
                if (k < K) x[t][0] = load_chunk<DT, false>(q, K - k);
                if (ES<DT> == 4 && k + 4 < K) x[t][1] = load_chunk<DT, false>(q + 16, K - k - 4);
            }
        }
#pragma unroll
        for (int d = 0; d < DUAL; ++d)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                if constexpr (ES<DT> == 4) {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
#pragma unroll
                        for (int t = 0; t < MT; ++t) {
                            const f32x4 xf = __builtin_bit_cast(f32x4, x[t][j >> 2]);
                            acc[t][d][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(s.w[d][j].t[c], xf[j & 3], acc[t][d][c], 0, 0, 0);
                        }
                } else {
                    u32x4 w;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint2 lo = __builtin_bit_cast(uint2, s.w[d][2 * j]), hi = __builtin_bit_cast(uint2, s.w[d][2 * j + 1]);
                        w[j] = __builtin_amdgcn_perm(c < 2 ? hi.x : hi.y, c < 2 ? lo.x : lo.y, c & 1 ? 0x07060302u : 0x05040100u);
                    }
#pragma unroll
                    for (int t = 0; t < MT; ++t) acc[t][d][c] = mfma_step<DT>(w, x[t][0], acc[t][d][c]);
                }
            }
    };

    Step s0, s1;
    int t = split * SK_WAVES + wave;
    if (t < steps) s0.load(p, a.ldw[0], t * 32, K, g);
    for (; t < steps; t += 2 * stride) {
        if (t + stride < steps) s1.load(p, a.ldw[0], (t + stride) * 32, K, g);
        use(s0, t * 32);
        if (t + stride >= steps) break;
        if (t + 2 * stride < steps) s0.load(p, a.ldw[0], (t + 2 * stride) * 32, K, g);
        use(s1, (t + stride) * 32);
    }

    // acc[t][d][c][j] is row 16 t + i, column 4 (4 g + j) + c
#pragma unroll
    for (int t16 = 0; t16 < MT; ++t16) {
        if (t16) __syncthreads();
        if (16 * t16 + i < a.M) {
#pragma unroll
            for (int d = 0; d < DUAL; ++d)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    *(f32x4*)sm[wave][d][4 * g + j][i] = f32x4{acc[t16][d][0][j], acc[t16][d][1][j], acc[t16][d][2][j], acc[t16][d][3][j]};
        }
        __syncthreads();
        // 16 quads of columns x 16 rows: one of 256 threads each
        const int q = threadIdx.x & 15, r = threadIdx.x >> 4, n = n0 + 4 * q;
        const long long m = 16 * t16 + r;
        if (r < 16 && m < a.M && n < a.N) {
            f32x4 v[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
            for (int d = 0; d < DUAL; ++d)
#pragma unroll
                for (int w = 0; w < SK_WAVES; ++w) v[d] += *(const f32x4*)sm[w][d][q][r];
            if (gridDim.y > 1) {
#pragma unroll
                for (int d = 0; d < DUAL; ++d) *(f32x4*)(a.part + (((long long)split * DUAL + d) * a.M + m) * a.Np + n) = v[d];
            } else {
                epilogue<DT, EPI>(a, 0, m, n, v[0], v[1]);
            }
        }
    }
}
