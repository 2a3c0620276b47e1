// rt_norm.hpp — the norms before and after a network block, with the block's gate and the residual, and their backward pass.
//
//   y = rs x + bs gate N(branch; w_post)          n = N(y; w_pre)
//   N(v; w) = v' / sqrt(mean(v'^2) + eps) * (w + w_offset),   v' = v (rms) or v - mean(v) (layer)
//
// Bound by memory: a row is read once and held in registers (TPR threads a row, NV 16-byte chunks a thread) while its
// sums are made in float32, and every output is written once.  What limits short calls is the chain load - sum - load: all
// of a row's arrays are asked for before the first is used, and sums that do not wait for each other share one exchange.
//
// The backward pass of wide rows (16-bit d > 8192, float32 d > 4096) does not fit its registers, 128 a thread: two rows' arrays,
// three column sums and two weights go to scratch memory and back (16384 bf16: 1.5 ms a training step of 64 M values, 0.7 TB/s;
// 8192: 283 us, 3.8 TB/s).
//
// Measured: 16384 x 4096 bf16 with branch and gate 97 us = 5.5 TB/s (a large copy: 5.2); one row 4.1 us, of which about 4 are
// the launch.  A wave a row up to 256 chunks, where there are rows enough: no barrier in the chain.
#pragma once
#include "rt_elem.hpp"


// A wave's sum in all its lanes, the same bits in each: within sixteen lanes by data-parallel moves, then across the rows of
// sixteen.  (ds_bpermute takes ten times as long a step, and a row waits for three such sums.)
__device__ __forceinline__ float wave_sum(float v) {
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0xb1, 0xf, 0xf, true));     // lane ^ 1
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x4e, 0xf, 0xf, true));     // lane ^ 2
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x141, 0xf, 0xf, true));    // 7 - lane
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x140, 0xf, 0xf, true));    // 15 - lane
    auto a = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
    const unsigned a0 = a[0], a1 = a[1];
    v = __builtin_bit_cast(float, a0) + __builtin_bit_cast(float, a1);
    auto b = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
    const unsigned b0 = b[0], b1 = b[1];
    return __builtin_bit_cast(float, b0) + __builtin_bit_cast(float, b1);
}

// K sums over the TPR threads of a row, the same values in all of them.  sm: K floats a wave, two sets used in turn, so that
// one barrier a call is enough.
template <int TPR, int K>
__device__ __forceinline__ void row_sums(float (&v)[K], float (*sm)[4], int& turn) {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = wave_sum(v[k]);
    if (TPR > 64) {
        constexpr int W = TPR / 64;
        float(*s)[4] = sm + (turn & 1) * W;
        turn++;
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int k = 0; k < K; ++k) s[wave][k] = v[k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w)
#pragma unroll
            for (int k = 0; k < K; ++k) v[k] += s[w][k];
    }
}

#define FOR_ROW(k, e)                        \
    _Pragma("unroll") for (int k = 0; k < NV; ++k) _Pragma("unroll") for (int e = 0; e < E; ++e)

// The buffer of one row: a row that is not there has no bytes, reads as zeros and drops what is written, so that loads and
// stores need no branches around them and the compiler can count them.
typedef __amdgpu_buffer_rsrc_t RowBuf;
__device__ __forceinline__ RowBuf row_buf(const char* p, bool there, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, p && there ? bytes : 0, 0x00020000);
}

// A row as it lies in memory.
template <int DT, int TPR, int NV, bool AL>
struct Raw {
    static constexpr int E = EPC<DT>;
    u32x4 c[NV];
    __device__ __forceinline__ void load(const char* p, int d, int t, bool there = true) {
        const RowBuf r = row_buf(p, there, d * ES<DT>);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int at = (k * TPR + t) * E;
            if (AL) {
                c[k] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, at * ES<DT>, 0, 0));
            } else {
                c[k] = u32x4{0, 0, 0, 0};
                if (p && there && at < d) c[k] = load_chunk<DT, AL>(p + (unsigned)at * (unsigned)ES<DT>, d - at);
            }
        }
    }
};

// A row in registers, in float32.
template <int DT, int TPR, int NV, bool AL>
struct Row {
    static constexpr int E = EPC<DT>;
    float v[NV][E];

    __device__ __forceinline__ Row() {}
    __device__ __forceinline__ explicit Row(const Raw<DT, TPR, NV, AL>& r) {
#pragma unroll
        for (int k = 0; k < NV; ++k) chunk_to_f32<DT>(r.c[k], v[k]);
    }
    // a weight: ones where there is none
    __device__ __forceinline__ void weight(const char* p, float off, int d, int t) {
        if (p) {
            Raw<DT, TPR, NV, AL> r;
            r.load(p, d, t);
            *this = Row(r);
            FOR_ROW(k, e) v[k][e] += off;
        } else {
            FOR_ROW(k, e) v[k][e] = 1.0f;
        }
    }
    __device__ __forceinline__ void store(char* p, int d, int t) const {
        typedef typename Elem<DT>::T T;
        const RowBuf r = row_buf(p, true, d * ES<DT>);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int at = (k * TPR + t) * E;
            if (AL) {
                union { T t[E]; u32x4 c; } u;
#pragma unroll
                for (int e = 0; e < E; ++e) u.t[e] = to_elem<DT>(v[k][e]);
                __builtin_amdgcn_raw_buffer_store_b128(u.c, r, at * ES<DT>, 0, 0);
            } else if (p && at < d) {
                store_chunk<DT, AL>(p + (unsigned)at * (unsigned)ES<DT>, v[k], d - at);
            }
        }
    }
    __device__ __forceinline__ void put(float* p, int d, int t) const {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int at = (k * TPR + t) * E;
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (at + e < d) p[at + e] = v[k][e];
        }
    }
    __device__ __forceinline__ void zero() { FOR_ROW(k, e) v[k][e] = 0.0f; }
    __device__ __forceinline__ float sum() const {
        float s = 0.0f;
        FOR_ROW(k, e) s += v[k][e];
        return s;
    }
    __device__ __forceinline__ float dot(const Row& o) const {
        float s = 0.0f;
        FOR_ROW(k, e) s += v[k][e] * o.v[k][e];
        return s;
    }
    // v - mean, and zeros behind the row's end
    __device__ __forceinline__ void centre(float mean, int d, int t) {
        FOR_ROW(k, e) v[k][e] = (k * TPR + t) * E + (AL ? 0 : e) < d ? v[k][e] - mean : 0.0f;
    }
    __device__ __forceinline__ void times(const Row& o, float off) { FOR_ROW(k, e) v[k][e] *= o.v[k][e] + off; }
    __device__ __forceinline__ void scale(float f) { FOR_ROW(k, e) v[k][e] *= f; }
};

constexpr int norm_block(int TPR) { return TPR > 256 ? TPR : 256; }

template <int DT, int TPR, int NV, bool AL>
__global__ __launch_bounds__(norm_block(TPR)) void norm_kernel(NormArgs a) {
    typedef Row<DT, TPR, NV, AL> R;
    typedef Raw<DT, TPR, NV, AL> M;
    constexpr int E = EPC<DT>;
    __shared__ float sm[2 * (TPR > 64 ? TPR / 64 : 1)][4];
    int turn = 0;
    const int t = threadIdx.x % TPR;
    constexpr int WAVES = norm_block(TPR) / TPR;
    const int w = WAVES == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / TPR);
    const long long row = ((long long)blockIdx.y * gridDim.x + blockIdx.x) * WAVES + w;
    if (row >= a.T) return;                     // TPR > 64: the whole workgroup (one row); else the whole wave
    const float inv = 1.0f / (float)a.d;
    M mx, mb, mg, mpost, mpre;
    mx.load(a.x + row * a.ldx, a.d, t);
    mb.load(a.b + row * a.ldb, a.d, t, a.b);
    mg.load(a.gate + (long long)((unsigned)row / (unsigned)a.rpg) * a.ldg, a.d, t, a.gate);      // T < 2^31
    mpost.load(a.w_post, a.d, t, a.b);
    mpre.load(a.w_pre, a.d, t, a.n);
    R v(mx);
    v.scale(a.rs);
    if (a.b) {
        R b(mb);
        float s[1];
        if (a.kind == RT_NORM_LAYER) {
            s[0] = b.sum();
            row_sums<TPR>(s, sm, turn);
            b.centre(s[0] * inv, a.d, t);
        }
        s[0] = b.dot(b);
        row_sums<TPR>(s, sm, turn);
        const float f = 1.0f / sqrtf(s[0] * inv + a.eps) * a.bs;
        b.scale(f);
        if (a.w_post) b.times(R(mpost), a.w_off);
        if (a.gate) b.times(R(mg), 0.0f);
        FOR_ROW(k, e) v.v[k][e] += b.v[k][e];
    }
    if (a.y) v.store(a.y + row * a.ldy, a.d, t);
    if (a.n) {
        float s[1];
        if (a.kind == RT_NORM_LAYER) {
            s[0] = v.sum();
            row_sums<TPR>(s, sm, turn);
            v.centre(s[0] * inv, a.d, t);
        }
        s[0] = v.dot(v);
        row_sums<TPR>(s, sm, turn);
        const float f = 1.0f / sqrtf(s[0] * inv + a.eps);
        v.scale(f);
        if (a.w_pre) v.times(R(mpre), a.w_off);
        v.store(a.n + row * a.ldn, a.d, t);
        if (a.n_lo) {                            // what the rounding left off: nothing of what it made infinite
            FOR_ROW(k, e) {
                const float r = (float)to_elem<DT>(v.v[k][e]);
                v.v[k][e] = __builtin_isinf(r) ? 0.0f : v.v[k][e] - r;
            }
            v.store(a.n_lo + row * a.ldn, a.d, t);
        }
    }
}

// Which slot of a unit's two gate sums a group's rows go to: 0 if the group is the unit's first.
__device__ __forceinline__ int gate_slot(long long group, long long unit_row0, long long rpg) {
    return group * rpg <= unit_row0 ? 0 : 1;
}

// Backward.  A unit is a workgroup: it walks rows_per_unit consecutive rows, all its threads one row at a time (TPR > 64) or a
// row for each of its four waves (TPR = 64), and its threads hold the column sums; a row's arrays are loaded while the row
// before is worked on.  The rows of one gate are a segment.  Where segments are long, the waves take its rows in turn
// (`together`) and their sums meet in LDS at its end; where short, a wave takes whole segments.  A segment's sum goes to
// dgate if the unit saw all of the gate's rows, else to one of the unit's two partial slots.
//
// Measured: 8191 x 4096 bf16, gates of 1000 rows, 97 us for 403 MB = 4.1 TB/s and the join 9; 10000 x 512 float32 28 us = 4.4
// TB/s and 5.  Two arrays of loads in turn (even, odd) with rows' bounds in the buffers instead of branches: 186 -> 52 us for
// the float32 training step, 239 -> 145 for the bf16 one, of which the forward pass has 20 and 51.
//
//   t = dy + dN(dn w_pre at y);  dx = rs t;  q = bs t;  db = dN(q gate w_post at b)
//   dN(z at v) = r (z - vh mean(z vh) [- mean z]),  vh = r v',  r = 1 / sqrt(mean(v'^2) + eps)
template <int DT, int TPR, int NV, bool AL>
__global__ __launch_bounds__(norm_block(TPR)) void norm_back_kernel(NormArgs a) {
    typedef Row<DT, TPR, NV, AL> R;
    typedef Raw<DT, TPR, NV, AL> M;
    constexpr int E = EPC<DT>, WAVES = norm_block(TPR) / TPR, COLS = TPR * NV * E;
    __shared__ float sm[2 * (TPR > 64 ? TPR / 64 : 1)][4];
    __shared__ float meet[WAVES > 1 ? WAVES * COLS : 1];
    int turn = 0;
    const int t = threadIdx.x % TPR, unit = blockIdx.x;
    const int w = WAVES == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / TPR);      // rows are the same for a whole wave
    const long long r0 = unit * a.rows_per_unit, r1 = r0 + a.rows_per_unit < a.T ? r0 + a.rows_per_unit : a.T;
    const float inv = 1.0f / (float)a.d;
    const bool layer = a.kind == RT_NORM_LAYER;
    R w_post, w_pre;
    w_post.weight(a.w_post, a.w_off, a.d, t);
    w_pre.weight(a.w_pre, a.w_off, a.d, t);

    R s_post, s_pre, s_gate;
    s_post.zero();
    s_pre.zero();
    s_gate.zero();

    // the waves' sums, added in wave order, in wave 0
    auto join = [&](R& s) __attribute__((always_inline)) {
        if (WAVES > 1) {
            __syncthreads();
            if (w) s.put(meet + w * COLS, a.d, t);
            __syncthreads();
            if (w == 0) {
#pragma unroll
                for (int k = 0; k < NV; ++k) {
                    const int at = (k * TPR + t) * E;
#pragma unroll
                    for (int e = 0; e < E; ++e)
                        if (at + e < a.d)
#pragma unroll
                            for (int o = 1; o < WAVES; ++o) s.v[k][e] += meet[o * COLS + at + e];
                }
            }
        }
    };
    auto flush = [&](long long group) __attribute__((always_inline)) {       // the segment of this gate is done
        const long long g0 = group * a.rpg, g1 = g0 + a.rpg < a.T ? g0 + a.rpg : a.T;
        if (g0 >= r0 && g1 <= r1) s_gate.store(a.dgate + group * a.lddg, a.d, t);
        else s_gate.put(a.p_gate + ((long long)unit * 2 + gate_slot(group, r0, a.rpg)) * a.d, a.d, t);
    };

    struct Arrays {
        M y, dn, dy, b, g;
    } even, odd;
    auto fetch = [&](Arrays& m, long long row, long long group, bool there) __attribute__((always_inline)) {
        m.y.load(a.yin + row * a.ldy, a.d, t, there && a.dn);
        m.dn.load(a.dn + row * a.lddn, a.d, t, there && a.dn);
        m.dy.load(a.dy + row * a.lddy, a.d, t, there && a.dy);
        m.b.load(a.b + row * a.ldb, a.d, t, there && a.b);
        m.g.load(a.gate + group * a.ldg, a.d, t, there && a.gate);
    };
    auto work = [&](const Arrays& m, long long row) __attribute__((always_inline)) {
        R y(m.y), dn(m.dn), b(m.b), z;
        float sums[4] = {0, 0, 0, 0};              // of y^2, z y, z and b^2
        if (a.yin_scale != 1.0f) y.scale(a.yin_scale);
        if (layer) {
            float mean[2] = {y.sum(), b.sum()};
            row_sums<TPR>(mean, sm, turn);
            y.centre(mean[0] * inv, a.d, t);
            b.centre(mean[1] * inv, a.d, t);
        }
        if (a.dn) {
            FOR_ROW(k, e) z.v[k][e] = dn.v[k][e] * w_pre.v[k][e];
            sums[0] = y.dot(y);
            sums[1] = z.dot(y);
            if (layer) sums[2] = z.sum();          // nothing lies behind the row's end: dn is 0 there
        }
        if (a.b) sums[3] = b.dot(b);
        row_sums<TPR>(sums, sm, turn);
        if (a.dn) {
            const float r = 1.0f / sqrtf(sums[0] * inv + a.eps), p = r * sums[1] * inv, q = sums[2] * inv;
            FOR_ROW(k, e) {
                const float h = y.v[k][e] * r;
                s_pre.v[k][e] += dn.v[k][e] * h;
                z.v[k][e] = (z.v[k][e] - h * p - q) * r;
            }
            if (a.dy) {
                const R dy(m.dy);
                FOR_ROW(k, e) z.v[k][e] += dy.v[k][e];
            }
        } else {
            z = R(m.dy);
        }
        if (a.dx) {
            R dx;
            FOR_ROW(k, e) dx.v[k][e] = z.v[k][e] * a.rs;
            dx.store(a.dx + row * a.lddx, a.d, t);
        }
        if (!a.b) return;
        const float r = 1.0f / sqrtf(sums[3] * inv + a.eps);
        b.scale(r);
        z.scale(a.bs);
        if (a.gate) {
            const R g(m.g);
            FOR_ROW(k, e) {
                const float u = z.v[k][e] * b.v[k][e];
                s_gate.v[k][e] += u * w_post.v[k][e];
                s_post.v[k][e] += u * g.v[k][e];
                z.v[k][e] *= g.v[k][e];
            }
        } else {
            FOR_ROW(k, e) s_post.v[k][e] += z.v[k][e] * b.v[k][e];
        }
        if (!a.db) return;
        FOR_ROW(k, e) z.v[k][e] *= w_post.v[k][e];
        float last[2] = {z.dot(b), 0.0f};
        if (layer) {
            z.centre(0.0f, a.d, t);
            last[1] = z.sum();
        }
        row_sums<TPR>(last, sm, turn);
        FOR_ROW(k, e) z.v[k][e] = (z.v[k][e] - b.v[k][e] * (last[0] * inv) - last[1] * inv) * r;
        z.store(a.db + row * a.lddb, a.d, t);
    };

    // One segment after another (by the gate, not by whether its gradient is wanted: the other sums keep their order).
    const bool own = a.gate && (WAVES == 1 || !a.together);         // a wave's rows are whole segments, in a row
    for (long long s0 = r0; s0 < r1;) {
        long long s1 = r1, row = s0 + w, end, step = WAVES;
        if (WAVES > 1 && own) {
            const unsigned n = ((unsigned)a.rows_per_unit / (unsigned)a.rpg + WAVES - 1) / WAVES * (unsigned)a.rpg;
            row = r0 + (long long)w * n;
            end = row + n < r1 ? row + n : r1;
            step = 1;
        }
        // the row's gate and the row behind that gate's last: rows only go up, so it takes one division a segment (T < 2^31)
        long long group = a.gate ? (unsigned)row / (unsigned)a.rpg : 0, g1 = (group + 1) * a.rpg;
        if (!(WAVES > 1 && own)) {
            if (a.gate && !own) {
                const long long first = (long long)((unsigned)s0 / (unsigned)a.rpg) * a.rpg + a.rpg;
                if (first < r1) s1 = first;
            }
            end = s1;
        }
        const long long seg_group = group;
        fetch(even, row, group, row < end);
        auto one = [&](const Arrays& now, Arrays& next) __attribute__((always_inline)) {
            const bool ends = row + step >= end || row + step >= g1;      // of this gate's rows here
            const long long here = group;
            if (row + step >= g1) {
                group++;
                g1 += a.rpg;
            }
            fetch(next, row + step, group, row + step < end);
            work(now, row);
            if (own && a.dgate && ends) {
                flush(here);
                s_gate.zero();
            }
            row += step;
        };
        while (row < end) {
            one(even, odd);
            if (row >= end) break;
            one(odd, even);
        }
        if (a.gate && !own && a.dgate) {
            join(s_gate);
            if (w == 0) flush(seg_group);
            s_gate.zero();
        }
        s0 = s1;
    }
    if (a.want_post) {
        join(s_post);
        if (w == 0) s_post.put(a.p_post + (long long)unit * a.d, a.d, t);
    }
    if (a.want_pre) {
        join(s_pre);
        if (w == 0) s_pre.put(a.p_pre + (long long)unit * a.d, a.d, t);
    }
}

// Column sums of the units' partial sums, in a fixed order: 32 columns x 32 row classes a workgroup, eight rows of a class under
// way at a time.  Latency: 5 us for 500 units of 512 columns, 9 for 256 of 4096.
// blockIdx.y + first: 0 post, 1 pre, 2 + g: gate group g (of those, only what more than one unit saw).
template <int DT>
__global__ __launch_bounds__(1024) void norm_join_kernel(NormArgs a, int first) {
    typedef typename Elem<DT>::T T;
    constexpr int RC = 32, B = 8;
    __shared__ float sm[RC][33];
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), rc = threadIdx.x >> 5, what = blockIdx.y + first;
    const long long group = what - 2;
    const float* p = what == 0 ? a.p_post : a.p_pre;
    char* out = what == 0 ? a.dw_post : a.dw_pre;
    long long u0 = 0, u1 = a.units;
    if (what >= 2) {
        const long long g0 = group * a.rpg, g1 = g0 + a.rpg < a.T ? g0 + a.rpg : a.T;
        u0 = g0 / a.rows_per_unit;
        u1 = (g1 - 1) / a.rows_per_unit + 1;
        if (u1 - u0 == 1) return;
        out = a.dgate + group * a.lddg;
    }
    if (!out) return;
    float s = 0.0f;
    if (c < a.d)
        for (long long u = u0 + rc; u < u1; u += RC * B) {
            float v[B];
#pragma unroll
            for (int b = 0; b < B; ++b) {
                const long long at = u + b * RC;
                v[b] = 0.0f;
                if (at < u1)
                    v[b] = what < 2 ? p[at * a.d + c] : a.p_gate[(at * 2 + gate_slot(group, at * a.rows_per_unit, a.rpg)) * a.d + c];
            }
#pragma unroll
            for (int b = 0; b < B; ++b) s += v[b];
        }
    sm[rc][threadIdx.x & 31] = s;
    __syncthreads();
    if (rc == 0 && c < a.d) {
        float v = 0.0f;
#pragma unroll
        for (int k = 0; k < RC; ++k) v += sm[k][threadIdx.x & 31];
        ((T*)out)[c] = to_elem<DT>(v);
    }
}
