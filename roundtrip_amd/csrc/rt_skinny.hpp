// rt_skinny.hpp — the feed-forward block's products for few rows (one token, a small serving batch): the weights are read
// once, straight into registers, and that is what bounds it.
//
//   C[m][n] = sum over k of X[m][k] W[k][n],     W [K][N] with n contiguous
//
// Two kernels.  Both give a workgroup of 8 waves a slab of columns and all of K (or a split of it, where columns alone leave
// the chip idle); lanes load four neighbouring columns of eight rows at a time, so that 64 lanes x eight loads are under way
// before the first is needed; rows of X that do not exist repeat the last and are dropped, like columns that do not exist.  The waves' sums
// meet in LDS in a fixed order, the splits' in gemm_join_kernel.
//
// Measured: one row, 4096 x 16384 bf16: 80 us for 403 MB (the gated product 51 us = 5.3 TB/s, as fast as a large copy; the other
// 27, its join 5); 24 rows, 4096 x 8192 bf16: 54 us for 201 MB; one row, 512 x 1024 float32: 8 us, two launches.
#pragma once
#include "rt_gemm.hpp"

// What a step brings of W and X: rows k0 + 8 g + j of the lane's four columns, and the same k's of XR rows of X.
// LO: of X and of what its rounding left off.
template <int DT, int DUAL, int XR, int KS, bool LO>
struct SkinnyStep {
    typedef typename Elem<DT>::T T;
    struct Four { T t[4]; };
    typedef unsigned Words __attribute__((ext_vector_type(ES<DT>)));
    struct __attribute__((packed, aligned(2))) Loose { Words v; };       // four elements at the alignment of one
    Four w[DUAL][8];
    u32x4 x[XR][8 / EPC<DT>], lo[LO ? XR : 1];

    // at: where the lane's columns and its first row lie from a row that is the same for the whole wave.  Row t of x is
    // m0 + t * mstep of X; rows behind M repeat the last (their sums are dropped).
    __device__ __forceinline__ void load(const GemmArgs& a, int k0, int K, int g, unsigned at, int m0, int mstep) {
        const long long ld = a.ldw[0];
        const int k = k0 + 8 * g, last = (int)a.M - 1;
        const bool whole = k0 + KS <= K;
#pragma unroll
        for (int d = 0; d < DUAL; ++d)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const Loose* p = (const Loose*)((a.w[d] + (k0 + j) * ld) + at);
                if (whole) {
                    w[d][j] = __builtin_bit_cast(Four, p->v);
                } else {
                    w[d][j] = Four{};
                    if (k + j < K) w[d][j] = __builtin_bit_cast(Four, p->v);
                }
            }
#pragma unroll
        for (int t = 0; t < XR; ++t) {
            const int m = m0 + t * mstep < last ? m0 + t * mstep : last;
            const char* p = a.x[0] + m * a.ldx[0] + (long long)k * ES<DT>;
#pragma unroll
            for (int h = 0; h < 8 / EPC<DT>; ++h) {
                if (whole) {
                    x[t][h] = ((const Chunk16*)(p + 16 * h))->v;
                } else {
                    x[t][h] = u32x4{0, 0, 0, 0};
                    if (k + h * EPC<DT> < K) x[t][h] = load_chunk<DT, false>(p + 16 * h, K - k - h * EPC<DT>);
                }
            }
            if (LO) {
                const char* q = a.x[1] + m * a.ldx[0] + (long long)k * ES<DT>;
                if (whole) {
                    lo[t] = ((const Chunk16*)q)->v;
                } else {
                    lo[t] = u32x4{0, 0, 0, 0};
                    if (k < K) lo[t] = load_chunk<DT, false>(q, K - k);
                }
            }
        }
    }
};

// Walks this wave's steps t, t + stride .. < steps with STAGES of them loaded ahead of their use.
template <int STAGES, class Step, class Load, class Use>
__device__ __forceinline__ void skinny_walk(int t, int steps, int stride, Load load, Use use) {
    Step s[STAGES];
#pragma unroll
    for (int u = 0; u < STAGES; ++u)
        if (t + u * stride < steps) load(s[u], t + u * stride);
    for (; t < steps; t += STAGES * stride) {
#pragma unroll
        for (int u = 0; u < STAGES; ++u) {
            const int at = t + u * stride;
            if (at < steps) use(s[u]);
            if (at + STAGES * stride < steps) load(s[u], at + STAGES * stride);
        }
    }
}

// Where a quad of columns begins: the last one, if it is not whole, at N - 4 (its first columns are made twice, alike).
__device__ __forceinline__ int quad_start(int n, int N) { return n < N - 4 ? n : N - 4; }

// Four sums of row m, columns n ..: to the split's partial sums, or on to what becomes of them.
template <int DT, int EPI>
__device__ __forceinline__ void finish(const GemmArgs& a, int split, long long m, int n, const f32x4 (&v)[2]) {
    constexpr int DUAL = EPI == EPI_GATED ? 2 : 1;
    if (gridDim.y > 1) {
#pragma unroll
        for (int d = 0; d < DUAL; ++d)
            ((Chunk16*)(a.part + (((long long)split * DUAL + d) * a.M + m) * a.Np + n))->v = __builtin_bit_cast(u32x4, v[d]);
    } else {
        epilogue_way<DT, EPI>(a, [&](auto way) __attribute__((always_inline)) {
            epilogue<DT, EPI, decltype(way)::act, decltype(way)::quads, decltype(way)::kept>(a, 0, m, n, v[0], v[1]);
        });
    }
}

// Up to 16 MT rows, 64 columns a workgroup, on the matrix cores.  In a step of 32 k's lane (g = lane / 16, i = lane % 16)
// holds columns 4 i .. of rows 8 g ..: for one of the four columns the eight rows are an operand of one 16x16x32 instruction
// as they are (16-bit: after one v_perm for every two values), so nothing passes through LDS.
template <int DT, int EPI, int MT, bool LO>
__global__ __launch_bounds__(64 * SK_WAVES) void skinny_kernel(GemmArgs a) {
    constexpr int DUAL = EPI == EPI_GATED ? 2 : 1, NW = SK_WAVES, TILES = MT;
    typedef SkinnyStep<DT, DUAL, TILES, 32, LO> Step;
    __shared__ float sm[NW][DUAL][SK_COLS / 4][16][4];         // [wave][..][quad of columns][row][column]: one row tile
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * SK_COLS, split = blockIdx.y, K = (int)a.K, steps = (K + 31) >> 5;
    const int stride = gridDim.y * NW;
    const unsigned at = (unsigned)(8 * g * a.ldw[0]) + (unsigned)quad_start(n0 + 4 * i, a.N) * ES<DT>;

    f32x4 acc[TILES][DUAL][4];
#pragma unroll
    for (int t = 0; t < TILES; ++t)
#pragma unroll
        for (int d = 0; d < DUAL; ++d)
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[t][d][c] = f32x4{0, 0, 0, 0};

    auto use = [&](const Step& s) __attribute__((always_inline)) {
#pragma unroll
        for (int d = 0; d < DUAL; ++d)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                if constexpr (ES<DT> == 4) {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
#pragma unroll
                        for (int t = 0; t < TILES; ++t) {
                            const f32x4 xf = __builtin_bit_cast(f32x4, s.x[t][j >> 2]);
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
                    for (int t = 0; t < TILES; ++t) {
                        acc[t][d][c] = mfma_step<DT>(w, s.x[t][0], acc[t][d][c]);
                        if constexpr (LO) acc[t][d][c] = mfma_step<DT>(w, s.lo[t], acc[t][d][c]);
                    }
                }
            }
    };

    // two waves a SIMD share its registers: as many steps ahead as they hold
    constexpr int STAGES = ES<DT> == 2 ? (DUAL == 2 ? (MT == 1 ? 3 : 2) : 4) : DUAL * MT == 4 ? 1 : 2;
    skinny_walk<STAGES, Step>(
        split * NW + wave, steps, stride, [&](Step& s, int t) __attribute__((always_inline)) { s.load(a, t * 32, K, g, at, i, 16); }, use);

    // acc[t][d][c][j] is row 16 t + i, column 4 (4 g + j) + c
#pragma unroll
    for (int t16 = 0; t16 < TILES; ++t16) {
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
                for (int w = 0; w < NW; ++w) v[d] += *(const f32x4*)sm[w][d][q][r];
            finish<DT, EPI>(a, split, m, quad_start(n, a.N), v);
        }
    }
}

// Up to MR <= 4 rows on the vector unit, 4 LI columns a workgroup.  With one row the chip is kept busy by many narrow slabs (a
// CU alone draws some 60 GB/s of weights), and a matrix instruction would be used for a sixteenth of its rows; float32's takes
// 32 cycles for four k's whatever they are.  Lane (g, i), i < LI, holds columns 4 i .. of rows 8 g .. of a step of 512 / LI k's.
template <int DT, int EPI, int MR, int LI, bool LO>
__global__ __launch_bounds__(64 * SK_WAVES) void gemv_kernel(GemmArgs a) {
    constexpr int DUAL = EPI == EPI_GATED ? 2 : 1, G = 64 / LI, KS = 8 * G;
    typedef SkinnyStep<DT, DUAL, MR, KS, LO> Step;
    __shared__ float sm[SK_WAVES][DUAL][MR][LI][4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane % LI, g = lane / LI;
    // neighbouring slabs share cache lines where they are narrow: give them to one XCD
    const int tiles = gridDim.x, b = blockIdx.x, xcd = b & 7, r8 = tiles & 7;
    const int n0 = (xcd * (tiles >> 3) + (xcd < r8 ? xcd : r8) + (b >> 3)) * 4 * LI, split = blockIdx.y;
    const int K = (int)a.K, steps = (K + KS - 1) / KS, stride = gridDim.y * SK_WAVES;
    const unsigned at = (unsigned)(8 * g * a.ldw[0]) + (unsigned)quad_start(n0 + 4 * i, a.N) * ES<DT>;

    float acc[DUAL][MR][4];
#pragma unroll
    for (int d = 0; d < DUAL; ++d)
#pragma unroll
        for (int m = 0; m < MR; ++m)
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[d][m][c] = 0.0f;

    auto use = [&](const Step& s) __attribute__((always_inline)) {
        float x[MR][8];
#pragma unroll
        for (int m = 0; m < MR; ++m)
#pragma unroll
            for (int h = 0; h < 8 / EPC<DT>; ++h) {
                float f[EPC<DT>];
                chunk_to_f32<DT>(s.x[m][h], f);
#pragma unroll
                for (int e = 0; e < EPC<DT>; ++e) x[m][h * EPC<DT> + e] = f[e];
                if constexpr (LO) {
                    chunk_to_f32<DT>(s.lo[m], f);
#pragma unroll
                    for (int e = 0; e < EPC<DT>; ++e) x[m][e] += f[e];
                }
            }
#pragma unroll
        for (int d = 0; d < DUAL; ++d)
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const float w = (float)s.w[d][j].t[c];
#pragma unroll
                    for (int m = 0; m < MR; ++m) acc[d][m][c] = fmaf(w, x[m][j], acc[d][m][c]);
                }
    };
    skinny_walk<ES<DT> == 2 ? 2 : 1, Step>(
        split * SK_WAVES + wave, steps, stride, [&](Step& s, int t) __attribute__((always_inline)) { s.load(a, t * KS, K, g, at, 0, 1); }, use);
#pragma unroll
    for (int d = 0; d < DUAL; ++d)
#pragma unroll
        for (int m = 0; m < MR; ++m) {
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int o = 32; o >= LI; o >>= 1) acc[d][m][c] += __shfl_xor(acc[d][m][c], o, 64);
            if (g == 0) *(f32x4*)sm[wave][d][m][i] = f32x4{acc[d][m][0], acc[d][m][1], acc[d][m][2], acc[d][m][3]};
        }
    __syncthreads();
    const int q = threadIdx.x % LI, m = threadIdx.x / LI, n = n0 + 4 * q;
    if (m < MR && m < a.M && n < a.N) {
        f32x4 v[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
        for (int d = 0; d < DUAL; ++d)
#pragma unroll
            for (int w = 0; w < SK_WAVES; ++w) v[d] += *(const f32x4*)sm[w][d][m][q];
        finish<DT, EPI>(a, split, m, quad_start(n, a.N), v);
    }
}
