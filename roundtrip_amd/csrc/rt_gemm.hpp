// rt_gemm.hpp — the matrix products of the gated feed-forward block, on the matrix cores, with their epilogues.
//
//   C[m][n] = sum over k of X[m][k] W[k][n]           X: rows (tokens, or the rows of a weight gradient), W: columns
//
// Each operand lies in memory with k contiguous (LK) or with its own index contiguous (LI): weights are [in, out], so the
// forward products read W as LI, the products with a transposed weight as LK, and a weight gradient (k = tokens) reads
// both as LI.  Tiles of 128 bytes of k go through LDS, two in turn; the matrix instruction is 16x16x32 (16-bit types) or
// 16x16x4 (float32) with W as its rows and X as its columns, so that a lane holds four neighbouring n of one m.
//
// Bound by the matrix cores.  Measured, all launches of a call: 8192 rows of a 4096 x 16384 bf16 block 2.6 ms = 1.27 PF/s (a
// library product of those sizes alone: 1.15 to 1.34); a training step at 4096 x 2048 x 8192 bf16 1.29 ms = 0.96 PF/s; 10000 x
// 512 x 1024 float32 268 us = 117 TF/s (matrix cores busy 74 % and 65 % of the two products).
#pragma once
#include "rt_elem.hpp"


// ---- the gate's activation ----------------------------------------------------------------------------------------
// s(t) = 1 / (1 + exp(-t)).  16-bit results: hardware exp2 and reciprocal (each <= 1 ulp of float32, far below the
// rounding of the result).
template <int DT>
__device__ __forceinline__ float sigmoid_f(float t) {
    if (ES<DT> == 4) return 1.0f / (1.0f + expf(-t));
    return __builtin_amdgcn_rcpf(1.0f + __expf(-t));
}

// a = act(g), d = act'(g).  gelu: the tanh form, 0.5 g (1 + tanh z) = g s(2z), which loses nothing where tanh z is near -1.
template <int DT, int ACT>
__device__ __forceinline__ void act_f(float alpha, float g, float& a, float& d) {
    if (ACT == RT_ACT_LRELU) {
        d = g > 0.0f ? 1.0f : alpha;
        a = g * d;
    } else if (ACT == RT_ACT_GELU_TANH) {
        const float c2 = 1.5957691216057308f, c3 = 0.044715f;      // 2 sqrt(2 / pi)
        const float s = sigmoid_f<DT>(c2 * (g + c3 * g * g * g));
        a = g * s;
        // from |g| = 64 on s (1 - s) is 0, and g^2 would not be finite for all g
        const float b = __builtin_amdgcn_fmed3f(g, -64.0f, 64.0f);
        d = s + b * s * (1.0f - s) * c2 * (1.0f + 3.0f * c3 * b * b);
    } else {
        const float s = sigmoid_f<DT>(g);
        a = ACT == RT_ACT_SILU ? g * s : s;
        d = ACT == RT_ACT_SILU ? s * (1.0f + g * (1.0f - s)) : s * (1.0f - s);
    }
}

// Four values at p, of which `valid` exist; QUADS: all four do, and p is aligned to them.
template <int DT, bool QUADS>
__device__ __forceinline__ void put4(char* p, f32x4 v, int valid) {
    typedef typename Elem<DT>::T T;
    typedef T T4 __attribute__((ext_vector_type(4)));
    if (QUADS) *(T4*)p = T4{to_elem<DT>(v[0]), to_elem<DT>(v[1]), to_elem<DT>(v[2]), to_elem<DT>(v[3])};
    else store4<DT>(p, v, valid);
}

// Four kept values as they lie in memory, of type KT.
template <int KT> using Kept = typename Elem<KT>::Quad;
template <int KT, bool QUADS>
__device__ __forceinline__ Kept<KT> load_kept(const char* p, int valid) {
    if (QUADS) return *(const Kept<KT>*)p;
    return __builtin_convertvector(load4<KT>(p, valid), Kept<KT>);       // of that type, so exact
}

// The kept gate and up at four places (columns behind N: zeros).
template <int KT, bool QUADS>
__device__ __forceinline__ void kept4(const GemmArgs& a, long long m, int n, Kept<KT>& g, Kept<KT>& u) {
    const int valid = a.N - n;
    g = u = Kept<KT>{0, 0, 0, 0};
    if (valid <= 0) return;
    const char *pg = a.e[0] + m * a.lde + (long long)n * ES<KT>, *pu = a.e[1] + m * a.lde + (long long)n * ES<KT>;
    g = load_kept<KT, QUADS>(pg, valid);
    u = load_kept<KT, QUADS>(pu, valid);
}

// EPI_GATED_BWD: v is dh.
template <int DT, int ACT, bool QUADS, int KT>
__device__ __forceinline__ void epilogue_bwd(const GemmArgs& a, long long m, int n, f32x4 v, Kept<KT> g, Kept<KT> u) {
    const int room = a.No - n, valid = a.N - n;
    if (room <= 0) return;
    const long long c = (long long)n * ES<DT>;
    f32x4 dg, du, h;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float t, d;
        act_f<DT, ACT>(a.alpha, (float)g[j], t, d);
        const float w = j < valid ? v[j] : 0.0f;         // zeros behind the row's end, whatever the sum there was of
        dg[j] = w * (float)u[j] * d;
        du[j] = w * t;
        h[j] = t * (float)u[j];
    }
    put4<DT, QUADS>(a.o[0] + m * a.ldo[0] + c, dg, room);
    put4<DT, QUADS>(a.o[1] + m * a.ldo[1] + c, du, room);
    put4<DT, QUADS>(a.o[2] + m * a.ldo[2] + c, h, room);
}

// What becomes of four neighbouring sums of row m, columns n .. n+3 (v1: the second of EPI_GATED).
template <int DT, int EPI, int ACT, bool QUADS, int KT>
__device__ __forceinline__ void epilogue(const GemmArgs& a, int z, long long m, int n, f32x4 v0, f32x4 v1) {
    const int valid = a.N - n, room = a.No - n;
    if (room <= 0) return;
    const long long c = (long long)n * ES<DT>, ck = (long long)n * ES<KT>;
    if (EPI == EPI_STORE) {
        put4<DT, QUADS>((z ? a.o[1] : a.o[0]) + m * a.ldo[0] + c, v0, valid);
    } else if (EPI == EPI_GATED) {
        f32x4 h;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float t, d;
            act_f<DT, ACT>(a.alpha, v0[j], t, d);
            h[j] = j < valid ? t * v1[j] : 0.0f;          // behind the row's end zeros, where an infinite x left NaN too
        }
        put4<DT, QUADS>(a.o[0] + m * a.ldo[0] + c, h, room);
        if (a.o[1] && valid > 0) {
            put4<KT, QUADS>(a.o[1] + m * a.ldo[1] + ck, v0, valid);
            put4<KT, QUADS>(a.o[2] + m * a.ldo[2] + ck, v1, valid);
        }
    } else {
        Kept<KT> g, u;
        kept4<KT, QUADS>(a, m, n, g, u);
        epilogue_bwd<DT, ACT, QUADS, KT>(a, m, n, v0, g, u);
    }
}

// body(ACT, QUADS, KT: the type of what is kept) with all as constants: the choice is made once, outside the loops over a tile.
template <int ACT, bool QUADS, int KT> struct EpiWay {
    static constexpr int act = ACT, kept = KT;
    static constexpr bool quads = QUADS;
};
template <bool QUADS, int KT, class Body>
__device__ __forceinline__ void epilogue_act(const GemmArgs& a, Body body) {
    if (a.act == RT_ACT_SILU) body(EpiWay<RT_ACT_SILU, QUADS, KT>());
    else if (a.act == RT_ACT_GELU_TANH) body(EpiWay<RT_ACT_GELU_TANH, QUADS, KT>());
    else if (a.act == RT_ACT_LRELU) body(EpiWay<RT_ACT_LRELU, QUADS, KT>());
    else body(EpiWay<RT_ACT_SIGMOID, QUADS, KT>());
}
template <int DT, int EPI, class Body>
__device__ __forceinline__ void epilogue_way(const GemmArgs& a, Body body) {
    if (EPI == EPI_STORE) {
        if (a.quads) body(EpiWay<0, true, RT_F32>());
        else body(EpiWay<0, false, RT_F32>());
    } else if (DT == RT_F32 || !a.kept_narrow) {
        if (a.quads) epilogue_act<true, RT_F32>(a, body);
        else epilogue_act<false, RT_F32>(a, body);
    } else {
        if (a.quads) epilogue_act<true, DT>(a, body);
        else epilogue_act<false, DT>(a, body);
    }
}

// ---- tiles --------------------------------------------------------------------------------------------------------
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// A buffer of `span` bytes from p on: what lies behind it reads as zeros.
__device__ __forceinline__ u32x4 buffer_of(const char* p, int span) {
    const unsigned long long at = (unsigned long long)p;
    return u32x4{(unsigned)__builtin_amdgcn_readfirstlane((int)at), (unsigned)__builtin_amdgcn_readfirstlane((int)(at >> 32) & 0xffff),
                 (unsigned)__builtin_amdgcn_readfirstlane(span), 0x00020000u};
}

// Sixteen bytes a lane straight to LDS, lane after lane from sm on (the same for the whole wave).  Written out because the
// compiler, where it loses track of which of the two tiles a read of LDS belongs to, waits for all such loads before it;
// whoever reads the tile waits for vmcnt(0) and a barrier.  (s_nop: m0 is set one wait state before its use.)
__device__ __forceinline__ void load_to_lds(u32x4 r, char* sm, int off) {
    const unsigned at = (unsigned)(uintptr_t)(lds_void*)sm;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" : : "s"(at), "v"(off), "s"(r) : "memory", "m0");
}

constexpr int OOB = 0x7fffff00;            // an offset that every buffer below ends before

// One operand's tile in LDS: R of its rows (or columns) x 128 bytes of k, as 16-byte chunks.
//   LK: [row][8 chunks], chunk c of row r at c ^ ((r >> 1) & 7): sixteen rows' reads of one chunk fall into sixteen
//       different 16-byte slots of the 256 bytes that LDS serves at once.
//   LI: [k][row], NSUB sub-tiles of R / NSUB rows one behind the other.  16-bit types are read with ds_read_b64_tr_b16
//       (sixteen lanes read a 4 x 16 block, each gets a column): its 32-byte units are xored with (k & 3) | (k >> 3 & 1) << 2
//       (rows of 128 bytes, two of which lie in those 256: (k >> 1 & 1) | (k >> 3 & 1) << 1); float32 is read four bytes a
//       lane, 64 a row: its 64-byte units are xored with (k >> 2) & 3.
template <int DT, int L, int R, int NSUB, int NT>
struct Tile {
    static constexpr int KE = 128 / ES<DT>;                 // k's of a tile
    static constexpr int BYTES = R * 128;
    static constexpr int SR = R / NSUB;
    static constexpr int PITCH = L == LK ? 128 : SR * ES<DT>;
    static constexpr int PC = PITCH / 16;
    static constexpr int ITER = BYTES / 16 / NT;            // chunks a thread brings
    static constexpr int SUB_CHUNKS = KE * PC;              // LI: chunks of a sub-tile
    static_assert(BYTES % (16 * NT) == 0, "every thread brings whole chunks");
    static_assert(L == LK ? NSUB == 1 : SR >= 64, "the xor needs that many units");

    static __device__ __forceinline__ int unit_xor(int k) {       // LI, 16-bit types
        return SR == 64 ? (k >> 1 & 1) | (k >> 3 & 1) << 1 : (k & 3) | (k >> 3 & 1) << 2;
    }

    // chunk it of thread tid: which row / k (idx), which chunk of it (c), which sub-tile
    static __device__ __forceinline__ void place(int tid, int it, int& sub, int& idx, int& c) {
        const int q = it * NT + tid;
        if (L == LK) {
            sub = 0;
            idx = q >> 3;
            c = (q & 7) ^ ((idx >> 1) & 7);
        } else {
            sub = q / SUB_CHUNKS;
            const int p = q % PC;
            idx = (q % SUB_CHUNKS) / PC;
            c = ES<DT> == 4 ? ((((p >> 2) ^ ((idx >> 2) & 3)) << 2) | (p & 3))
                            : ((((p >> 1) ^ unit_xor(idx)) << 1) | (p & 1));
        }
    }
};

// v as a number of 128 bits, shifted down by so many bytes.
__device__ __forceinline__ u32x4 shift_down(u32x4 v, int bytes) {
    const int d = bytes >> 2;
    unsigned w[8] = {v[0], v[1], v[2], v[3], 0, 0, 0, 0}, x[5];
#pragma unroll
    for (int i = 0; i < 5; ++i) x[i] = d == 0 ? w[i] : d == 1 ? w[i + 1] : d == 2 ? w[i + 2] : d == 3 ? w[i + 3] : 0;
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __builtin_amdgcn_alignbyte(x[i + 1], x[i], bytes & 3);
    return r;
}

template <int DT, int L, int R, int NSUB, int NT, bool AL>
struct Loader {
    typedef Tile<DT, L, R, NSUB, NT> T;
    int voff[T::ITER];                // byte offset from the tile's start.  AL: OOB where the row or column does not exist
    // !AL: chunks go through registers.  A chunk that is not whole is loaded so that it ends where its row does, from earlier
    // columns on, and shifted into place (zeros follow); rows that do not exist repeat the last.  So loads have no branches.
    bool ragged, tiny;                // the last chunk of columns is not whole; a row is shorter than a chunk
    bool on_way, fix;                 // the tile's chunks are in reg; some have to be shifted
    int had;                          // the k's it has
    u32x4 reg[AL ? 1 : T::ITER];

    // Elements that chunk it lacks at its end, of `rows` columns (LI) or `ke` k's (LK, LI).
    static __device__ __forceinline__ int lacks(int tid, int it, int rows, int ke) {
        int sub, idx, c;
        T::place(tid, it, sub, idx, c);
        if (L == LI && idx >= ke) return EPC<DT>;
        const int n = (c + 1) * EPC<DT> - (L == LK ? ke : rows);
        return n > 0 ? n : 0;
    }

    // rows: how many of the tile's rows (LI: columns) exist, counted in a sub-tile; all: how many elements a row of the operand has
    __device__ __forceinline__ void init(int tid, long long ld, int rows, long long all) {
        ragged = L == LI && rows % (T::SR) != 0;
        tiny = all < EPC<DT>;
#pragma unroll
        for (int it = 0; it < T::ITER; ++it) {
            int sub, idx, c;
            T::place(tid, it, sub, idx, c);
            if (AL) {
                const int row = L == LK ? idx : c * EPC<DT>;
                voff[it] = row < rows ? (int)(idx * ld) + c * 16 : OOB;
            } else if (L == LK) {
                voff[it] = (int)((idx < rows ? idx : rows - 1) * ld) + c * 16;
            } else {
                voff[it] = (int)(idx * ld) + c * 16 - lacks(tid, it, rows, T::KE) * ES<DT>;
            }
        }
    }

    // Brings the tile that starts at element k0 of K.  base: the operand's first row (LK) or column (LI) of this tile,
    // base2: the second sub-tile's.
    __device__ __forceinline__ void fetch(char* sm, const char* base, const char* base2, long long ld, long long k0, long long K,
                                          int rows, int tid) {
        const long long left = K - k0;
        const int ke = left < T::KE ? (int)left : T::KE;
        const long long adv = L == LK ? k0 * ES<DT> : k0 * ld;
        if (AL) {
            // a tile spans less than 2^31 bytes (the host bounds ld), whatever the whole operand spans
            // (a row's last chunk is whole: it ends with the row, or with the zeros behind it)
            const int whole = ((L == LK ? ke : rows) + EPC<DT> - 1) / EPC<DT> * 16;
            const int span = (int)(((L == LK ? rows : ke) - 1) * ld) + whole;
            const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
#pragma unroll
            for (int it = 0; it < T::ITER; ++it) {
                const bool second = L == LI && NSUB == 2 && it >= T::ITER / 2;
                const u32x4 r = buffer_of((second ? base2 : base) + adv, span);
                int v = voff[it];
                if (L == LK && ke < T::KE) {            // the last tile: chunks behind K are zeros
                    int sub, idx, c;
                    T::place(tid, it, sub, idx, c);
                    if (c * EPC<DT> >= ke) v = OOB;
                }
                if (L == LI && ke < T::KE) {            // k's behind K: behind the span, or before it ends in a short last row
                    int sub, idx, c;
                    T::place(tid, it, sub, idx, c);
                    if (idx >= ke) v = OOB;
                }
                load_to_lds(r, sm + (it * NT + wave * 64) * 16, v);
            }
        } else if (!tiny) {
            on_way = true;
            had = ke;
            fix = ragged || ke < T::KE;
            const char *b0 = base + adv, *b1 = (NSUB == 2 ? base2 : base) + adv;
            if (ke == T::KE) {
#pragma unroll
                for (int it = 0; it < T::ITER; ++it) reg[it] = ((const Chunk16*)((NSUB == 2 && it >= T::ITER / 2 ? b1 : b0) + voff[it]))->v;
            } else {
                asm volatile("" : "+v"(tid));
#pragma unroll
                for (int it = 0; it < T::ITER; ++it) {
                    int sub, idx, c;
                    T::place(tid, it, sub, idx, c);
                    const long long less = L == LK ? lacks(tid, it, rows, ke) * ES<DT> : idx >= ke ? (idx - ke + 1) * ld : 0;
                    reg[it] = ((const Chunk16*)((NSUB == 2 && it >= T::ITER / 2 ? b1 : b0) + (voff[it] - less)))->v;
                }
            }
        } else {
            on_way = false;
#pragma unroll 1
            for (int it = 0; it < T::ITER; ++it) {
                int sub, idx, c;
                T::place(tid, it, sub, idx, c);
                const char* b = (L == LI && NSUB == 2 && sub ? base2 : base) + adv;
                const int have = L == LK ? (idx < rows ? ke - c * EPC<DT> : 0) : (idx < ke ? rows - c * EPC<DT> : 0);
                u32x4 r = {0, 0, 0, 0};
                if (have > 0) r = load_chunk<DT, false>(b + idx * ld + c * 16, have);
                *(u32x4*)(sm + (it * NT + tid) * 16) = r;
            }
        }
    }

    __device__ __forceinline__ void land(char* sm, int tid, int rows) {
        if (AL || !on_way) return;
        if (fix) {
            asm volatile("" : "+v"(tid));                // worked out here when it is needed, not held in registers all the time
#pragma unroll
            for (int it = 0; it < T::ITER; ++it) reg[it] = shift_down(reg[it], lacks(tid, it, rows, had) * ES<DT>);
        }
#pragma unroll
        for (int it = 0; it < T::ITER; ++it) *(u32x4*)(sm + (it * NT + tid) * 16) = reg[it];
    }
};

// Reads the fragment of sixteen rows (or columns) starting at 16 t of sub-tile `sub`, k step s (of two): lane (g = lane / 16, i = lane % 16)
// gets row i, k = 32 s + 8 g .. + 7 (16-bit), 16 s + 4 g .. + 3 (float32).  The same k's for both operands is all that
// the sum needs.
template <int DT, int L, int R, int NSUB, int NT>
__device__ __forceinline__ u32x4 read_frag(const char* sm, int lane, int sub, int t, int s) {
    typedef Tile<DT, L, R, NSUB, NT> T;
    const int i = lane & 15, g = lane >> 4;
    if (L == LK) {
        return *(const u32x4*)(sm + (16 * t + i) * 128 + (((4 * s + g) ^ (i >> 1)) << 4));
    } else {
        sm += sub * (T::SUB_CHUNKS * 16);
        if (ES<DT> == 4) {
            u32x4 r;
#pragma unroll
            for (int j = 0; j < 4; ++j) r[j] = *(const unsigned*)(sm + (16 * s + 4 * g + j) * T::PITCH + ((t ^ g) << 6) + i * 4);
            return r;
        }
        union { s16x4 h[2]; u32x4 v; } u;
#pragma unroll
        for (int h = 0; h < 2; ++h)
            u.h[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (lds_s16x4*)(sm + (32 * s + 8 * g + 4 * h + (i >> 2)) * T::PITCH + ((t ^ T::unit_xor(8 * g + (i >> 2))) << 5) + (i & 3) * 8));
        return u.v;
    }
}

template <int DT>
__device__ __forceinline__ f32x4 mfma_step(u32x4 w, u32x4 x, f32x4 c) {
    if constexpr (DT == RT_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w), __builtin_bit_cast(bf16x8, x), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, w), __builtin_bit_cast(f16x8, x), c, 0, 0, 0);
}

// acc[i][j] += W fragment j times X fragment i.  float32 takes four instructions a fragment; the same sums' come as far apart
// as can be, so that none waits for the one before it.
template <int DT, int MT, int NTL>
__device__ __forceinline__ void mfma_tile(const u32x4 (&fw)[NTL], const u32x4 (&fx)[MT], f32x4 (&acc)[MT][NTL]) {
    if constexpr (DT == RT_F32) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NTL; ++j) {
                    const f32x4 w = __builtin_bit_cast(f32x4, fw[j]), x = __builtin_bit_cast(f32x4, fx[i]);
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[q], x[q], acc[i][j], 0, 0, 0);
                }
    } else {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NTL; ++j) acc[i][j] = mfma_step<DT>(fw[j], fx[i], acc[i][j]);
    }
}

// Workgroup -> tile.  Workgroups go to the eight XCDs in turn: each XCD gets a run of tiles, walked in bands of GM tile rows,
// so that the tiles it works on at a time share their operands in its L2.
__device__ __forceinline__ void tile_of(int b, int tiles_m, int tiles_n, int& tm, int& tn) {
    const int n = tiles_m * tiles_n, q = n >> 3, r = n & 7, xcd = b & 7;
    const int id = xcd * q + (xcd < r ? xcd : r) + (b >> 3);
    constexpr int GM = 8;
    const int band = id / (GM * tiles_n), first = band * GM;
    const int h = tiles_m - first < GM ? tiles_m - first : GM;
    const int in = id - band * GM * tiles_n;
    tm = first + in % h;
    tn = in / h;
}

// A wave's MT x NTL sums of 16 x 16, from row m0 and column n0 of C on: finished, or written as a split's partial sums.
template <int DT, int EPI, int MT, int NTL>
__device__ __forceinline__ void finish_tile(const GemmArgs& a, int z, int split, long long m0, int n0, const f32x4 (&acc)[MT][NTL]) {
    constexpr int DUAL = EPI == EPI_GATED ? 2 : 1, H = NTL / DUAL;
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    if (a.splits > 1) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            const long long m = m0 + mt * 16 + i;
            if (m >= a.M) continue;
#pragma unroll
            for (int j = 0; j < H; ++j) {
                const int n = n0 + j * 16 + 4 * g;
                if (n < a.Np) {
#pragma unroll
                    for (int d = 0; d < DUAL; ++d)
                        *(f32x4*)(a.part + (((long long)split * a.nslot + (DUAL == 2 ? d : z)) * a.M + m) * a.Np + n) = acc[mt][j + d * H];
                }
            }
        }
        return;
    }
    epilogue_way<DT, EPI>(a, [&](auto way) __attribute__((always_inline)) {
        constexpr int ACT = decltype(way)::act, KT = decltype(way)::kept;
        constexpr bool QUADS = decltype(way)::quads;
        if constexpr (EPI == EPI_GATED_BWD) {            // what it reads is asked for a row of tiles ahead
            Kept<KT> gate[2][H], up[2][H];
            auto ask = [&](int mt) __attribute__((always_inline)) {
                const long long m = m0 + mt * 16 + i;
#pragma unroll
                for (int j = 0; j < H; ++j)
                    if (m < a.M) kept4<KT, QUADS>(a, m, n0 + j * 16 + 4 * g, gate[mt & 1][j], up[mt & 1][j]);
            };
            ask(0);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                if (mt + 1 < MT) ask(mt + 1);
                const long long m = m0 + mt * 16 + i;
                if (m >= a.M) continue;
#pragma unroll
                for (int j = 0; j < H; ++j)
                    epilogue_bwd<DT, ACT, QUADS, KT>(a, m, n0 + j * 16 + 4 * g, acc[mt][j], gate[mt & 1][j], up[mt & 1][j]);
            }
        } else {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                const long long m = m0 + mt * 16 + i;
                if (m >= a.M) continue;
#pragma unroll
                for (int j = 0; j < H; ++j)
                    epilogue<DT, EPI, ACT, QUADS, KT>(a, z, m, n0 + j * 16 + 4 * g, acc[mt][j], acc[mt][DUAL == 2 ? j + H : j]);
            }
        }
    });
}

// BM x BN sums a workgroup of WM x WN waves.  EPI_GATED: the BN columns are BN / 2 of the gate's and the same of up's, and
// every wave holds both of its columns, so the product needs no exchange.  128 x 128: two workgroups a CU (64 KB of LDS each) hide each
// other's waits; 64 x 64 for products with too few tiles of 128 to fill the chip, and for float32, whose step of 128 x 128
// leaves CUs idle at the end (10000 x 512 x 1024: 334 us before, 268 with both to choose from and mfma_tile's order).
template <int DT, int LX, int LW, int EPI, int BM, int BN, int WM, int WN, bool AL>
__global__ __launch_bounds__(64 * WM * WN, 2) void gemm_kernel(GemmArgs a) {
    constexpr int NT = 64 * WM * WN, DUAL = EPI == EPI_GATED ? 2 : 1;
    typedef Tile<DT, LX, BM, 1, NT> TX;
    typedef Tile<DT, LW, BN, DUAL, NT> TW;
    constexpr int MT = BM / WM / 16, NTL = BN / WN / 16, CN = BN / DUAL;      // CN: columns of C a tile covers
    __shared__ __attribute__((aligned(1024))) char sx0[TX::BYTES], sw0[TW::BYTES], sx1[TX::BYTES], sw1[TW::BYTES];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WN, wn = wave % WN, z = blockIdx.z, split = blockIdx.y;
    int tm, tn;
    tile_of(blockIdx.x, a.tiles_m, a.tiles_n, tm, tn);
    const long long m0 = (long long)tm * BM;
    const int n0 = tn * CN;
    const int mrows = a.M - m0 < BM ? (int)(a.M - m0) : BM, nrows = a.N - n0 < CN ? a.N - n0 : CN;
    const int t0 = split * a.per_split, t_all = a.nk * a.nseg, t1 = t0 + a.per_split < t_all ? t0 + a.per_split : t_all;

    Loader<DT, LX, BM, 1, NT, AL> lx;
    Loader<DT, LW, BN, DUAL, NT, AL> lw;
    lx.init(tid, a.ldx[0], mrows, LX == LK ? a.K : a.M);
    lw.init(tid, a.ldw[0], nrows, LW == LK ? a.K : a.N);
    f32x4 acc[MT][NTL];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NTL; ++j) acc[i][j] = f32x4{0, 0, 0, 0};

    auto fetch = [&](char* sx, char* sw, int t) __attribute__((always_inline)) {
        const int seg = t >= a.nk ? 1 : 0;
        const long long k0 = (long long)(t - (seg ? a.nk : 0)) * TX::KE;
        const bool second = seg | z;                     // never a variable index: the arguments would be copied to scratch memory
        const char* bx = (second ? a.x[1] : a.x[0]) + (LX == LK ? m0 * a.ldx[0] : m0 * ES<DT>);
        const long long nw = LW == LK ? n0 * a.ldw[0] : (long long)n0 * ES<DT>;
        lx.fetch(sx, bx, nullptr, a.ldx[0], k0, a.K, mrows, tid);
        lw.fetch(sw, (EPI != EPI_GATED && second ? a.w[1] : a.w[0]) + nw, EPI == EPI_GATED ? a.w[1] + nw : nullptr, a.ldw[0], k0, a.K, nrows, tid);
    };
    auto land = [&](char* sx, char* sw) __attribute__((always_inline)) {
        lx.land(sx, tid, mrows);
        lw.land(sw, tid, nrows);
        __builtin_amdgcn_s_waitcnt(0x0f70);          // vmcnt(0): the chunks on their way to LDS have arrived
        __syncthreads();
    };
    auto compute = [&](const char* sx, const char* sw) __attribute__((always_inline)) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            if (!AL && s) __builtin_amdgcn_sched_barrier(0);      // the chunks on their way need the registers of a second set
            u32x4 fx[MT], fw[NTL];
#pragma unroll
            for (int i = 0; i < MT; ++i) fx[i] = read_frag<DT, LX, BM, 1, NT>(sx, lane, 0, wm * MT + i, s);
#pragma unroll
            for (int j = 0; j < NTL; ++j) {
                constexpr int H = NTL / DUAL;
                fw[j] = read_frag<DT, LW, BN, DUAL, NT>(sw, lane, j / H, wn * H + j % H, s);
            }
            mfma_tile<DT>(fw, fx, acc);
        }
    };

    fetch(sx0, sw0, t0);
    land(sx0, sw0);
    for (int t = t0; t < t1; t += 2) {
        if (t + 1 < t1) fetch(sx1, sw1, t + 1);
        compute(sx0, sw0);
        if (t + 1 >= t1) break;
        land(sx1, sw1);
        if (t + 2 < t1) fetch(sx0, sw0, t + 2);
        compute(sx1, sw1);
        if (t + 2 < t1) land(sx0, sw0);
    }

    finish_tile<DT, EPI>(a, z, split, m0 + wm * (BM / WM), n0 + wn * (CN / WN), acc);
}

// The same product in 256 x 256 tiles by eight waves of 128 x 64, for operands large enough to give every CU a tile: half the
// bytes from memory and three quarters from LDS of 128 x 128 a sum (8192 x 4096 x 16384 bf16: 3765 -> 2600 us; 4096 x 2048 x 8192
// training 1740 -> 1290).  Its matrix cores are busy 57 to 62 % of the time at 2.07 GHz; LDS is read without bank conflicts for
// about as long as the matrix cores work, and that bounds it.  (256 x 128 tiles: 1.25 us a step, chosen for no sizes.)
//
// Two waves share a SIMD.  The lower four and the upper four run half a step apart: while the one half's 32 matrix
// instructions of a k half have the matrix core, the other half reads its next fragments from LDS and sends for the next
// tile, and a barrier hands over.  Reads are complete before the barrier, so that when a half starts a tile, the buffer of the
// tile before it is free for the one after it.
template <int DT, int LX, int LW, int EPI>
__global__ __launch_bounds__(512, 2) void gemm_big_kernel(GemmArgs a) {
    constexpr int BM = 256, BN = 256, WM = 2, WN = 4, NT = 512, DUAL = EPI == EPI_GATED ? 2 : 1;
    typedef Tile<DT, LX, BM, 1, NT> TX;
    typedef Tile<DT, LW, BN, DUAL, NT> TW;
    constexpr int MT = BM / WM / 16, NTL = BN / WN / 16, CN = BN / DUAL, H = NTL / DUAL;
    __shared__ __attribute__((aligned(1024))) char sx0[TX::BYTES], sw0[TW::BYTES], sx1[TX::BYTES], sw1[TW::BYTES];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WN, wn = wave % WN, z = blockIdx.z, split = blockIdx.y;
    int tm, tn;
    tile_of(blockIdx.x, a.tiles_m, a.tiles_n, tm, tn);
    const long long m0 = (long long)tm * BM;
    const int n0 = tn * CN;
    const int mrows = a.M - m0 < BM ? (int)(a.M - m0) : BM, nrows = a.N - n0 < CN ? a.N - n0 : CN;
    const int t0 = split * a.per_split, t_all = a.nk * a.nseg, t1 = t0 + a.per_split < t_all ? t0 + a.per_split : t_all;

    Loader<DT, LX, BM, 1, NT, true> lx;
    Loader<DT, LW, BN, DUAL, NT, true> lw;
    lx.init(tid, a.ldx[0], mrows, LX == LK ? a.K : a.M);
    lw.init(tid, a.ldw[0], nrows, LW == LK ? a.K : a.N);
    f32x4 acc[MT][NTL];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NTL; ++j) acc[i][j] = f32x4{0, 0, 0, 0};

    auto fetch = [&](char* sx, char* sw, int t) __attribute__((always_inline)) {
        const int seg = t >= a.nk ? 1 : 0;
        const long long k0 = (long long)(t - (seg ? a.nk : 0)) * TX::KE;
        const bool second = seg | z;                     // never a variable index: the arguments would be copied to scratch memory
        const char* bx = (second ? a.x[1] : a.x[0]) + (LX == LK ? m0 * a.ldx[0] : m0 * ES<DT>);
        const long long nw = LW == LK ? n0 * a.ldw[0] : (long long)n0 * ES<DT>;
        lx.fetch(sx, bx, nullptr, a.ldx[0], k0, a.K, mrows, tid);
        lw.fetch(sw, (EPI != EPI_GATED && second ? a.w[1] : a.w[0]) + nw, EPI == EPI_GATED ? a.w[1] + nw : nullptr, a.ldw[0], k0, a.K, nrows, tid);
    };
    u32x4 fx[MT], fw[NTL];
    auto read = [&](const char* sx, const char* sw, int s) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < NTL; ++j) {
            fw[j] = read_frag<DT, LW, BN, DUAL, NT>(sw, lane, j / H, wn * H + j % H, s);
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) fx[i] = read_frag<DT, LX, BM, 1, NT>(sx, lane, 0, wm * MT + i, s);
    };
    auto turn = [&]() __attribute__((always_inline)) {
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
    };
    auto multiply = [&]() __attribute__((always_inline)) {
        __builtin_amdgcn_s_setprio(1);
        mfma_tile<DT>(fw, fx, acc);
        __builtin_amdgcn_s_setprio(0);
    };
    // one tile: s*: where it lies, n*: where the next one goes
    auto tile = [&](char* sx, char* sw, char* nx, char* nw, int t) __attribute__((always_inline)) {
        if (t + 1 < t1) fetch(nx, nw, t + 1);
        read(sx, sw, 0);
        __builtin_amdgcn_s_waitcnt(0xc07f);              // lgkmcnt(0)
        turn();
        multiply();
        turn();
        read(sx, sw, 1);
        __builtin_amdgcn_s_waitcnt(0x0070);              // vmcnt(0), lgkmcnt(0): the next tile is there
        turn();
        multiply();
        turn();
    };

    fetch(sx0, sw0, t0);
    __builtin_amdgcn_s_waitcnt(0x0070);
    turn();
    if (wave >= 4) turn();                               // half a step behind
    for (int t = t0; t < t1; t += 2) {
        tile(sx0, sw0, sx1, sw1, t);
        if (t + 1 < t1) tile(sx1, sw1, sx0, sw0, t + 1);
    }
    if (wave < 4) turn();                                // every wave has passed as many barriers

    finish_tile<DT, EPI>(a, z, split, m0 + wm * (BM / WM), n0 + wn * (CN / WN), acc);
}

// Joins the partial sums of the K splits, in their order, and finishes them.  Eight splits' loads are under way at a time:
// they come from other XCDs' writes, about a microsecond each.  4 to 5 us a launch at the sizes of a few rows: latency.
template <int DT, int EPI>
__global__ __launch_bounds__(256) void gemm_join_kernel(GemmArgs a) {
    constexpr int DUAL = EPI == EPI_GATED ? 2 : 1, B = 8 / DUAL;
    const int quads = a.Np >> 2, z = blockIdx.z;
    const long long total = a.M * quads, slot = a.M * a.Np;
    for (long long p = (long long)blockIdx.x * blockDim.x + threadIdx.x; p < total; p += (long long)gridDim.x * blockDim.x) {
        const long long m = p / quads;
        const int n = (int)(p - m * quads) * 4;
        const float* q = a.part + (long long)z * slot + m * a.Np + n;
        f32x4 v[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
        for (int s = 0; s < a.splits; s += B) {
            f32x4 t[B][DUAL];
#pragma unroll
            for (int b = 0; b < B; ++b)
#pragma unroll
                for (int d = 0; d < DUAL; ++d)
                    t[b][d] = *(const f32x4*)(q + ((long long)(s + b < a.splits ? s + b : s) * a.nslot + d) * slot);
#pragma unroll
            for (int b = 0; b < B; ++b)
#pragma unroll
                for (int d = 0; d < DUAL; ++d)
                    if (s + b < a.splits) v[d] += t[b][d];
        }
        epilogue_way<DT, EPI>(a, [&](auto way) __attribute__((always_inline)) {
            epilogue<DT, EPI, decltype(way)::act, decltype(way)::quads, decltype(way)::kept>(a, z, m, n, v[0], v[1]);
        });
    }
}
