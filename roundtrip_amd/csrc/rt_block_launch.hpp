// rt_block_launch.hpp — the kernels of the network-block operators and their launches, for the element type RT_BLOCK_DT.
#include "rt_block.hpp"

namespace rt_block {
namespace {

#include "rt_gemm.hpp"
#include "rt_skinny.hpp"
#include "rt_norm.hpp"

// One row for each kernel that a product can run on.
typedef void (*GemmFn)(GemmArgs);
template <int DT, int LX, int LW, int EPI>
GemmFn gemm_fn(bool al, int bm) {
    if constexpr (DT != RT_F32) {
        if (bm == 256) return gemm_big_kernel<DT, LX, LW, EPI>;
    }
    constexpr int SMALL_N = EPI == EPI_GATED ? 128 : 64;          // 64 columns of C
    if (bm == 64) return al ? gemm_kernel<DT, LX, LW, EPI, 64, SMALL_N, 2, 2, true> : gemm_kernel<DT, LX, LW, EPI, 64, SMALL_N, 2, 2, false>;
    return al ? gemm_kernel<DT, LX, LW, EPI, 128, 128, 2, 2, true> : gemm_kernel<DT, LX, LW, EPI, 128, 128, 2, 2, false>;
}

// Copies of matrices whose rows are no whole chunks, with zeros behind the rows (memory: 1777 x 1001 and twice 1001 x 2731 f16, 28 MB
// moved, about 10 us).  One matrix a blockIdx.y, one 16-byte chunk of the copy a thread.
template <int DT>
__global__ __launch_bounds__(256) void pad_kernel(PadArgs a) {
    const PadArgs::One& m = blockIdx.y == 0 ? a.m[0] : blockIdx.y == 1 ? a.m[1] : blockIdx.y == 2 ? a.m[2] : blockIdx.y == 3 ? a.m[3] : a.m[4];
    const int chunks = (int)(m.ldd / 16);
    const long long total = m.rows * chunks;
    for (long long p = (long long)blockIdx.x * 256 + threadIdx.x; p < total; p += (long long)gridDim.x * 256) {
        const long long r = p / chunks;
        const int c = (int)(p - r * chunks);
        *(u32x4*)(m.dst + r * m.ldd + c * 16) = load_chunk<DT, false>(m.src + r * m.ld + c * 16, m.width - c * EPC<DT>);
    }
}

hipError_t launch_join(hipStream_t st, GemmFn join, int64_t M, int Np, int nbatch, const GemmArgs& a) {
    // small joins: one wave a workgroup, so that they spread over the CUs
    const int64_t quads = M * (Np / 4);
    const int threads = quads < 65536 ? 64 : 256;
    const int64_t n = (quads + threads - 1) / threads;
    hipLaunchKernelGGL(join, dim3((unsigned)(n < 8192 ? n : 8192), 1, nbatch), dim3(threads), 0, st, a);
    return hipGetLastError();
}

template <int DT, bool AL, int TPR, int NV>
void launch_norm_fwd(hipStream_t st, const NormArgs& a) {
    constexpr int B = norm_block(TPR), RPB = B / TPR;
    // a launch holds less than 2^32 threads in x: more rows go on in y
    const int64_t n = (a.T + RPB - 1) / RPB, x = n < (1 << 21) ? n : 1 << 21;
    hipLaunchKernelGGL((norm_kernel<DT, TPR, NV, AL>), dim3((unsigned)x, (unsigned)((n + x - 1) / x)), dim3(B), 0, st, a);
}

template <int DT, bool AL, int TPR, int NV>
void launch_norm_back(hipStream_t st, const NormArgs& a) {
    hipLaunchKernelGGL((norm_back_kernel<DT, TPR, NV, AL>), dim3((unsigned)a.units), dim3(norm_block(TPR)), 0, st, a);
}

template <int DT, bool AL>
void pick_norm(hipStream_t st, const NormArgs& a, int tpr, bool back) {
    const int nv = ((a.d + EPC<DT> - 1) / EPC<DT> + tpr - 1) / tpr;
    if (back) {
        constexpr int PER = DT == RT_F32 ? 2 : 1;
        if (tpr == 64) nv <= 1 ? launch_norm_back<DT, AL, 64, 1>(st, a) : launch_norm_back<DT, AL, 64, PER>(st, a);
        else if (tpr == 256) nv <= 1 ? launch_norm_back<DT, AL, 256, 1>(st, a) : launch_norm_back<DT, AL, 256, PER>(st, a);
        else if (tpr == 512) nv <= PER ? launch_norm_back<DT, AL, 512, PER>(st, a) : launch_norm_back<DT, AL, 512, 2>(st, a);
        else if (nv <= 2) launch_norm_back<DT, AL, 1024, 2>(st, a);
        else launch_norm_back<DT, AL, 1024, 4>(st, a);
    } else if (tpr == 64) {
        if (nv <= 1) launch_norm_fwd<DT, AL, 64, 1>(st, a);
        else if (nv <= 2) launch_norm_fwd<DT, AL, 64, 2>(st, a);
        else launch_norm_fwd<DT, AL, 64, 4>(st, a);
    } else if (tpr == 256) {
        if (nv <= 1) launch_norm_fwd<DT, AL, 256, 1>(st, a);
        else if (nv <= 2) launch_norm_fwd<DT, AL, 256, 2>(st, a);
        else launch_norm_fwd<DT, AL, 256, 4>(st, a);
    } else {
        nv <= 2 ? launch_norm_fwd<DT, AL, 1024, 2>(st, a) : launch_norm_fwd<DT, AL, 1024, 4>(st, a);
    }
}

}  // namespace

template <int DT>
hipError_t launch_product(hipStream_t st, const Product& p, const Plan& pl, GemmArgs& a, bool al) {
    a.M = p.M; a.N = p.N; a.K = p.K; a.nseg = p.nseg; a.nk = pl.nk;
    a.tiles_m = pl.tiles_m; a.tiles_n = pl.tiles_n;
    a.splits = pl.splits; a.per_split = pl.per_split; a.Np = pl.Np; a.nslot = pl.nslot;
    a.No = p.No > p.N ? p.No : p.N;
    GemmFn fn, join;
    if (p.epi == EPI_GATED) {
        fn = gemm_fn<DT, LK, LI, EPI_GATED>(al, pl.bm);
        join = gemm_join_kernel<DT, EPI_GATED>;
    } else if (p.epi == EPI_GATED_BWD) {
        fn = gemm_fn<DT, LK, LK, EPI_GATED_BWD>(al, pl.bm);
        join = gemm_join_kernel<DT, EPI_GATED_BWD>;
    } else {
        fn = p.lx == LI ? gemm_fn<DT, LI, LI, EPI_STORE>(al, pl.bm)
                        : p.lw == LI ? gemm_fn<DT, LK, LI, EPI_STORE>(al, pl.bm) : gemm_fn<DT, LK, LK, EPI_STORE>(al, pl.bm);
        join = gemm_join_kernel<DT, EPI_STORE>;
    }
    hipLaunchKernelGGL(fn, dim3(pl.tiles_m * pl.tiles_n, pl.splits, p.nrun), dim3(pl.bm == 256 ? 512 : 256), 0, st, a);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess && pl.splits > 1 ? launch_join(st, join, p.M, pl.Np, p.nrun, a) : e;
}

template <int DT, int EPI, int MR, bool LO>
GemmFn gemv_fn(int li) {
    return li == 16 ? gemv_kernel<DT, EPI, MR, 16, LO> : li == 8 ? gemv_kernel<DT, EPI, MR, 8, LO> : gemv_kernel<DT, EPI, MR, 4, LO>;
}

template <int DT, int EPI, bool LO>
GemmFn skinny_fn(int64_t M, int li) {
    if (M == 1) return gemv_fn<DT, EPI, 1, LO>(li);
    if (M == 2) return gemv_fn<DT, EPI, 2, LO>(li);
    if (M <= GEMV_ROWS) return gemv_fn<DT, EPI, GEMV_ROWS, LO>(li);
    return M <= 16 ? skinny_kernel<DT, EPI, 1, LO> : skinny_kernel<DT, EPI, 2, LO>;
}

template <int DT>
hipError_t launch_skinny(hipStream_t st, const Product& p, const Plan& pl, GemmArgs& a) {
    a.M = p.M; a.N = a.No = p.N; a.K = p.K;
    a.splits = pl.splits; a.Np = pl.Np; a.nslot = pl.nslot;
    const bool gated = p.epi == EPI_GATED;
    GemmFn fn = gated ? skinny_fn<DT, EPI_GATED, false>(p.M, pl.li) : skinny_fn<DT, EPI_STORE, false>(p.M, pl.li);
    if constexpr (DT != RT_F32) {
        if (gated && p.nseg == 2) fn = skinny_fn<DT, EPI_GATED, true>(p.M, pl.li);
    }
    const GemmFn join = gated ? gemm_join_kernel<DT, EPI_GATED> : gemm_join_kernel<DT, EPI_STORE>;
    hipLaunchKernelGGL(fn, dim3(pl.tiles_n, pl.splits), dim3(64 * SK_WAVES), 0, st, a);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess && pl.splits > 1 ? launch_join(st, join, p.M, pl.Np, 1, a) : e;
}

template <int DT>
hipError_t launch_pad(hipStream_t st, const PadArgs& a) {
    hipLaunchKernelGGL(pad_kernel<DT>, dim3(2048, a.n), dim3(256), 0, st, a);
    return hipGetLastError();
}

template <int DT>
hipError_t launch_norm(hipStream_t st, const NormArgs& a, int tpr, bool back, bool al) {
    al ? pick_norm<DT, true>(st, a, tpr, back) : pick_norm<DT, false>(st, a, tpr, back);
    return hipGetLastError();
}

template <int DT>
hipError_t launch_norm_join(hipStream_t st, const NormArgs& a, int first, int last) {
    hipLaunchKernelGGL(norm_join_kernel<DT>, dim3((a.d + 31) / 32, last - first), dim3(1024), 0, st, a, first);
    return hipGetLastError();
}

template hipError_t launch_product<RT_BLOCK_DT>(hipStream_t, const Product&, const Plan&, GemmArgs&, bool);
template hipError_t launch_skinny<RT_BLOCK_DT>(hipStream_t, const Product&, const Plan&, GemmArgs&);
template hipError_t launch_pad<RT_BLOCK_DT>(hipStream_t, const PadArgs&);
template hipError_t launch_norm<RT_BLOCK_DT>(hipStream_t, const NormArgs&, int, bool, bool);
template hipError_t launch_norm_join<RT_BLOCK_DT>(hipStream_t, const NormArgs&, int, int);

}  // namespace rt_block
