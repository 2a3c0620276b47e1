// rt_block.hpp — what the host side of the network-block operators (rt_block.hip) and the translation units of their kernels
// (rt_block_f32 / bf16 / f16.hip, one for each element type, compiled side by side) share.
#pragma once
#include "rt_internal.hpp"

namespace rt_block {

enum { LK = 0, LI = 1 };
enum { EPI_STORE = 0, EPI_GATED = 1, EPI_GATED_BWD = 2 };

struct GemmArgs {
    const char* x[2];              // two K segments (nseg = 2), or one operand for each blockIdx.z
    const char* w[2];              // ... EPI_GATED: gate and up
    long long ldx[2], ldw[2];      // bytes
    long long M, K;
    int N;
    int nseg;                      // K segments: C = x[0] w[0] + x[1] w[1]
    int nk;                        // K tiles of a segment
    int tiles_m, tiles_n;
    int splits, per_split;         // K tiles are dealt to blockIdx.y, per_split each
    float* part;                   // splits > 1: [split][slot][M][Np] partial sums, joined by gemm_join_kernel
    int Np, nslot;
    int No;                        // columns written: N, or more of the workspace's own rows, zeros that the next product may read
    char* o[3];                    // EPI_STORE: o[blockIdx.z].  EPI_GATED: h, gate, up (the last two kept, or NULL).
    long long ldo[3];              // (EPI_STORE: ldo[0] for both)  EPI_GATED_BWD: dgate, dup, h
    const char* e[2];              // EPI_GATED_BWD: the gate and up that the forward pass kept
    long long lde;
    int kept_narrow;               // what is kept has the call's type, not float32
    int act;
    float alpha;
    int quads;                     // N and every output's (and e's) place are multiples of four elements
};

struct NormArgs {
    long long T;
    int d, kind;
    float eps, rs, bs, w_off;
    long long rpg;                                   // rows of x that share a row of gate
    const char *x, *b, *gate, *w_post, *w_pre, *yin; // yin: backward: y, or x where there is no branch
    char *y, *n, *n_lo;
    long long ldx, ldb, ldy, ldn, ldg;               // bytes
    // backward
    const char *dy, *dn;
    char *dx, *db, *dgate;
    long long lddy, lddn, lddx, lddb, lddg;
    float yin_scale;                                 // y = yin_scale * yin
    int want_post, want_pre;
    long long rows_per_unit;                         // consecutive rows of one workgroup
    int units;
    int together;                                    // the waves of a workgroup share its rows' gate sums
    float *p_post, *p_pre, *p_gate;                  // [units][d], [units][d], [units][2][d] partial sums
    char *dw_post, *dw_pre;
};

// ---- matrix products ----------------------------------------------------------------------------------------------
struct Product {                // C [M x N] = X W over K, nseg segments, nbatch products side by side
    int lx, lw, epi;
    int64_t M, K;
    int N = 0, nseg = 1, nbatch = 1;
    int No = 0;                 // columns to write, if more than N
    bool xpad = false, wpad = false;   // the operand's rows are padded with zeros to whole 16-byte chunks
    int nrun = nbatch;          // of the products side by side, how many are wanted: the plan, and so the bits, are the same
};

struct Plan {
    bool skinny;                // rt_skinny.hpp
    int li;
    int bm, splits, per_split, nk, tiles_m, tiles_n, nslot, Np;
    size_t part_bytes;
};

constexpr int SKINNY_ROWS = 32, GEMV_ROWS = 4;    // rt_skinny.hpp: most rows; most of them on the vector unit
constexpr int SK_WAVES = 8, SK_COLS = 64;

// Copies of matrices whose rows are no whole number of 16-byte chunks, with zeros behind each row.
struct PadArgs {
    int n;
    struct One {
        const char* src;
        char* dst;
        long long ld, ldd, rows;   // bytes
        int width;                 // elements
    } m[5];
};

// Launches on the element type DT.  Each returns the launches' first error.
template <int DT> RT_HIDDEN hipError_t launch_product(hipStream_t st, const Product& p, const Plan& pl, GemmArgs& a, bool al);
template <int DT> RT_HIDDEN hipError_t launch_skinny(hipStream_t st, const Product& p, const Plan& pl, GemmArgs& a);
template <int DT> RT_HIDDEN hipError_t launch_pad(hipStream_t st, const PadArgs& a);
template <int DT> RT_HIDDEN hipError_t launch_norm(hipStream_t st, const NormArgs& a, int tpr, bool back, bool al);
template <int DT> RT_HIDDEN hipError_t launch_norm_join(hipStream_t st, const NormArgs& a, int first, int last);

}  // namespace rt_block
