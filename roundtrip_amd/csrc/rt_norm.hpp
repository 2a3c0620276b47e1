// rt_norm.hpp — the norms before and after a network block, with the block's gate and the residual, and their backward pass.
//
//   y = rs x + bs gate N(branch; w_post)          n = N(y; w_pre)
//   N(v; w) = v' / sqrt(mean(v'^2) + eps) * (w + w_offset),   v' = v (rms) or v - mean(v) (layer)
//
// Bound by memory: a row is read once and held in registers (TPR threads a row, NV 16-byte chunks a thread) while its
// sums are made in float32, and every output is written once.
#pragma once
#include "rt_elem.hpp"

struct NormArgs {
    long long T;
    int d, kind;
    float eps, rs, bs, w_off;
    long long rpg;                                   // rows of x that share a row of gate
    const char *x, *b, *gate, *w_post, *w_pre, *yin; // yin: backward: y, or x where there is no branch
    char *y, *n;
    long long ldx, ldb, ldy, ldn, ldg;               // bytes
    // backward
    const char *dy, *dn;
    char *dx, *db, *dgate;
    long long lddy, lddn, lddx, lddb, lddg;
    float yin_scale;                                 // y = yin_scale * yin
    int want_post, want_pre;
    long long rows_per_unit;                         // consecutive rows of one unit (TPR threads)
    int units;
    float *p_post, *p_pre, *p_gate;                  // [units][d], [units][d], [units][2][d] partial sums
    char *dw_post, *dw_pre;
};

// Sum over the TPR threads of a row, the same value in all of them.  sm: one float a wave, two sets used in turn.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* sm, int& turn) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    if (TPR > 64) {
        constexpr int W = TPR / 64;
        float* s = sm + (turn & 1) * W;
        turn++;
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) s[wave] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) v += s[w];
    }
    return v;
}

// A row in registers, in float32.  hat(): v -> (v - mean) r, returns r.
template <int DT, int TPR, int NV, bool AL>
struct Row {
    static constexpr int E = EPC<DT>;
    float v[NV][E];

    __device__ __forceinline__ void load(const char* p, int d, int t) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * TPR + t) * E;
            u32x4 q = {0, 0, 0, 0};
            if (c < d) q = load_chunk<DT, AL>(p + (long long)c * ES<DT>, d - c);
            chunk_to_f32<DT>(q, v[k]);
        }
    }
    __device__ __forceinline__ void store(char* p, int d, int t) const {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * TPR + t) * E;
            if (c < d) store_chunk<DT, AL>(p + (long long)c * ES<DT>, v[k], d - c);
        }
    }
    __device__ __forceinline__ float hat(int d, int t, int kind, float eps, float* sm, int& turn) {
        const float inv = 1.0f / (float)d;
        if (kind == RT_NORM_LAYER) {
            float s = 0.0f;
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int e = 0; e < E; ++e) s += v[k][e];
            const float mean = row_sum<TPR>(s, sm, turn) * inv;
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int e = 0; e < E; ++e) v[k][e] = (k * TPR + t) * E + e < d ? v[k][e] - mean : 0.0f;
        }
        float q = 0.0f;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int e = 0; e < E; ++e) q += v[k][e] * v[k][e];
        const float r = 1.0f / sqrtf(row_sum<TPR>(q, sm, turn) * inv + eps);
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int e = 0; e < E; ++e) v[k][e] *= r;
        return r;
    }
    // the gradient through hat: this holds the hatted row, z the gradient of it, r its factor; z becomes the result
    __device__ __forceinline__ void back(Row& z, int d, int t, int kind, float r, float* sm, int& turn) const {
        const float inv = 1.0f / (float)d;
        float p = 0.0f, s = 0.0f;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const bool in = (k * TPR + t) * E + (AL ? 0 : e) < d;        // nothing behind the row's end counts
                p += in ? z.v[k][e] * v[k][e] : 0.0f;
                s += in ? z.v[k][e] : 0.0f;
            }
        p = row_sum<TPR>(p, sm, turn) * inv;
        s = kind == RT_NORM_LAYER ? row_sum<TPR>(s, sm, turn) * inv : 0.0f;      // the hatted row sums to 0
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int e = 0; e < E; ++e) z.v[k][e] = (z.v[k][e] - v[k][e] * p - s) * r;
    }
};

template <int DT, int TPR, int NV, bool AL>
__device__ __forceinline__ void load_weight(Row<DT, TPR, NV, AL>& w, const char* p, float off, int d, int t) {
    if (p) {
        w.load(p, d, t);
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int e = 0; e < EPC<DT>; ++e) w.v[k][e] += off;
    } else {
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int e = 0; e < EPC<DT>; ++e) w.v[k][e] = 1.0f;
    }
}

constexpr int norm_block(int TPR) { return TPR > 256 ? TPR : 256; }

template <int DT, int TPR, int NV, bool AL>
__global__ __launch_bounds__(norm_block(TPR)) void norm_kernel(NormArgs a) {
    typedef Row<DT, TPR, NV, AL> R;
    constexpr int E = EPC<DT>;
    __shared__ float sm[2 * (TPR > 64 ? TPR / 64 : 1)];
    int turn = 0;
    const int t = threadIdx.x % TPR;
    const long long row = (long long)blockIdx.x * (norm_block(TPR) / TPR) + threadIdx.x / TPR;
    if (row >= a.T) return;                     // TPR > 64: the whole workgroup (one row); else the whole wave
    R v;
    v.load(a.x + row * a.ldx, a.d, t);
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int e = 0; e < E; ++e) v.v[k][e] *= a.rs;
    if (a.b) {
        R b, w;
        b.load(a.b + row * a.ldb, a.d, t);
        b.hat(a.d, t, a.kind, a.eps, sm, turn);
        load_weight(w, a.w_post, a.w_off, a.d, t);
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int e = 0; e < E; ++e) b.v[k][e] *= w.v[k][e] * a.bs;
        if (a.gate) {
            w.load(a.gate + (row / a.rpg) * a.ldg, a.d, t);
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int e = 0; e < E; ++e) b.v[k][e] *= w.v[k][e];
        }
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int e = 0; e < E; ++e) v.v[k][e] += b.v[k][e];
    }
    if (a.y) v.store(a.y + row * a.ldy, a.d, t);
    if (a.n) {
        R w;
        v.hat(a.d, t, a.kind, a.eps, sm, turn);
        load_weight(w, a.w_pre, a.w_off, a.d, t);
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int e = 0; e < E; ++e) v.v[k][e] *= w.v[k][e];
        v.store(a.n + row * a.ldn, a.d, t);
    }
}

// Which slot of a unit's two gate sums a group's rows go to: 0 if the group is the unit's first.
__device__ __forceinline__ int gate_slot(long long group, long long unit_row0, long long rpg) {
    return group * rpg <= unit_row0 ? 0 : 1;
}

// A unit (TPR threads) walks rows_per_unit consecutive rows and holds its column sums in registers; a gate's sum is
// written when its rows end: to dgate if the unit saw all of them, else to one of the unit's two partial slots.
template <int DT, int TPR, int NV, bool AL>
__global__ __launch_bounds__(norm_block(TPR)) void norm_back_kernel(NormArgs a) {
    typedef Row<DT, TPR, NV, AL> R;
    constexpr int E = EPC<DT>;
    __shared__ float sm[2 * (TPR > 64 ? TPR / 64 : 1)];
    int turn = 0;
    const int t = threadIdx.x % TPR, unit = blockIdx.x * (norm_block(TPR) / TPR) + threadIdx.x / TPR;
    const long long r0 = unit * a.rows_per_unit, r1 = r0 + a.rows_per_unit < a.T ? r0 + a.rows_per_unit : a.T;
    if (r0 >= r1) return;
    float s_post[NV][E], s_pre[NV][E], s_gate[NV][E];
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int e = 0; e < E; ++e) s_post[k][e] = s_pre[k][e] = s_gate[k][e] = 0.0f;

    auto put = [&](float* p, float (&s)[NV][E]) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * TPR + t) * E;
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (c + e < a.d) p[c + e] = s[k][e];
        }
    };

    for (long long row = r0; row < r1; ++row) {
        R z, h;
        // t = dy + the gradient through n = N(y)
        if (a.dn) {
            R y, w;
            y.load(a.yin + row * a.ldy, a.d, t);
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int e = 0; e < E; ++e) y.v[k][e] *= a.yin_scale;
            const float r = y.hat(a.d, t, a.kind, a.eps, sm, turn);
            z.load(a.dn + row * a.lddn, a.d, t);
            load_weight(w, a.w_pre, a.w_off, a.d, t);
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    s_pre[k][e] += z.v[k][e] * y.v[k][e];
                    z.v[k][e] *= w.v[k][e];
                }
            y.back(z, a.d, t, a.kind, r, sm, turn);
            if (a.dy) {
                h.load(a.dy + row * a.lddy, a.d, t);
#pragma unroll
                for (int k = 0; k < NV; ++k)
#pragma unroll
                    for (int e = 0; e < E; ++e) z.v[k][e] += h.v[k][e];
            }
        } else {
            z.load(a.dy + row * a.lddy, a.d, t);
        }
        if (a.dx) {
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int e = 0; e < E; ++e) h.v[k][e] = z.v[k][e] * a.rs;
            h.store(a.dx + row * a.lddx, a.d, t);
        }
        if (!a.b) continue;
        R w, gt;
        h.load(a.b + row * a.ldb, a.d, t);
        const float r = h.hat(a.d, t, a.kind, a.eps, sm, turn);
        load_weight(w, a.w_post, a.w_off, a.d, t);
        const long long group = row / a.rpg;
        if (a.gate) {
            gt.load(a.gate + group * a.ldg, a.d, t);
        } else {
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int e = 0; e < E; ++e) gt.v[k][e] = 1.0f;
        }
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float q = z.v[k][e] * a.bs;
                s_gate[k][e] += q * h.v[k][e] * w.v[k][e];
                s_post[k][e] += q * gt.v[k][e] * h.v[k][e];
                z.v[k][e] = q * gt.v[k][e] * w.v[k][e];
            }
        if (a.db) {
            h.back(z, a.d, t, a.kind, r, sm, turn);
            z.store(a.db + row * a.lddb, a.d, t);
        }
        if (a.dgate && (row + 1 == r1 || (row + 1) % a.rpg == 0)) {
            const long long g0 = group * a.rpg, g1 = g0 + a.rpg < a.T ? g0 + a.rpg : a.T;
            if (g0 >= r0 && g1 <= r1) {
#pragma unroll
                for (int k = 0; k < NV; ++k) {
                    const int c = (k * TPR + t) * E;
                    if (c < a.d) store_chunk<DT, AL>(a.dgate + group * a.lddg + (long long)c * ES<DT>, s_gate[k], a.d - c);
                }
            } else {
                put(a.p_gate + ((long long)unit * 2 + gate_slot(group, r0, a.rpg)) * a.d, s_gate);
            }
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int e = 0; e < E; ++e) s_gate[k][e] = 0.0f;
        }
    }
    if (a.want_post) put(a.p_post + (long long)unit * a.d, s_post);
    if (a.want_pre) put(a.p_pre + (long long)unit * a.d, s_pre);
}

// Column sums of the units' partial sums, in a fixed order: 32 columns x 8 row classes a workgroup.
// blockIdx.y + first: 0 post, 1 pre, 2 + g: gate group g (of those, only what more than one unit saw).
template <int DT>
__global__ __launch_bounds__(256) void norm_join_kernel(NormArgs a, int first) {
    typedef typename Elem<DT>::T T;
    __shared__ float sm[8][33];
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), rc = threadIdx.x >> 5, what = blockIdx.y + first;
    const float* p;
    char* out;
    long long u0 = 0, u1 = a.units;
    if (what < 2) {
        p = what == 0 ? a.p_post : a.p_pre;
        out = what == 0 ? a.dw_post : a.dw_pre;
        if (!out) return;
    } else {
        const long long g = what - 2, g0 = g * a.rpg, g1 = g0 + a.rpg < a.T ? g0 + a.rpg : a.T;
        u0 = g0 / a.rows_per_unit;
        u1 = (g1 - 1) / a.rows_per_unit + 1;
        if (u1 - u0 == 1) return;
        p = nullptr;
        out = a.dgate + g * a.lddg;
    }
    float s = 0.0f;
    if (c < a.d)
        for (long long u = u0 + rc; u < u1; u += 8)
            s += what < 2 ? p[u * a.d + c]
                          : a.p_gate[(u * 2 + gate_slot(what - 2, u * a.rows_per_unit, a.rpg)) * a.d + c];
    sm[rc][threadIdx.x & 31] = s;
    __syncthreads();
    if (rc == 0 && c < a.d) {
        float v = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) v += sm[k][threadIdx.x & 31];
        ((T*)out)[c] = (T)v;
    }
}
