// rt_block.hip — the network-block operators of the C ABI: the gated feed-forward block and the norms around it, forward and
// backward (include/rt_is.h): checks, plans and launches.  Kernels: rt_gemm.hpp, rt_skinny.hpp (matrix products), rt_norm.hpp.
//
// Every call is a few launches on the context's stream, allocates nothing and keeps nothing: what it needs beyond its
// arguments is the caller's workspace.  So a call can be captured into a graph, and two graphs do not meet unless their
// caller gives them the same workspace.

#include "rt_block.hpp"
#include <math.h>
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

using namespace rt_block;

namespace {

int failf(rt_ctx* ctx, int code, const char* fmt, ...) {
    char msg[320];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(msg, sizeof msg, fmt, ap);
    va_end(ap);
    return rt_ctx_fail(ctx, code, msg);
}

#define HIPCHK(ctx, call)                                                                          \
    do {                                                                                           \
        const hipError_t e_ = (call);                                                              \
        if (e_ != hipSuccess) return failf(ctx, RT_EHIP, "%s: %s", #call, hipGetErrorString(e_));  \
    } while (0)

// Makes the context's device current for the duration of a call, and what was current again behind it.
struct DeviceScope {
    int before = -1;
    hipError_t err;
    explicit DeviceScope(int device) {
        err = hipGetDevice(&before);
        if (err == hipSuccess && before != device) err = hipSetDevice(device);
        else before = -1;
    }
    ~DeviceScope() { if (before >= 0) (void)hipSetDevice(before); }
};

constexpr int64_t MAX_DIM = 1 << 20;              // elements of a row, and of its stride: a tile then spans < 2^31 bytes
constexpr int64_t MAX_ROWS = 1ll << 40;
constexpr int64_t MAX_TILES = (1 << 23) - 1;      // of up to 512 threads: a launch holds less than 2^32

int elem_size(int dtype) { return dtype == RT_F32 ? 4 : 2; }
int64_t up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

// A strided matrix in device memory, as the checks see it.
struct Mat {
    const char* name;
    const void* p;
    int64_t rows, width, ld;      // ld in elements
    int es;                       // bytes of an element
};

// Whether two matrices share an element.  Columns of one buffer (equal strides, disjoint column ranges) do not.
bool overlap(const Mat& a, const Mat& b) {
    if (!a.p || !b.p || a.rows == 0 || b.rows == 0) return false;
    const uintptr_t a0 = (uintptr_t)a.p, a1 = a0 + ((a.rows - 1) * a.ld + a.width) * a.es;
    const uintptr_t b0 = (uintptr_t)b.p, b1 = b0 + ((b.rows - 1) * b.ld + b.width) * b.es;
    if (a1 <= b0 || b1 <= a0) return false;
    const int64_t pitch = a.ld * a.es;
    if (pitch != b.ld * b.es) return true;
    const int64_t d = (int64_t)(b0 - a0) % pitch, off = d < 0 ? d + pitch : d;
    return !(off >= a.width * a.es && off + b.width * b.es <= pitch);
}

bool same_place(const Mat& a, const Mat& b) { return a.p == b.p && (a.ld == b.ld || a.rows <= 1); }

int check_mat(rt_ctx* ctx, const char* fn, const Mat& m, bool required) {
    if (!m.p) return required && m.rows > 0 ? failf(ctx, RT_EINVAL, "%s: %s is NULL", fn, m.name) : RT_OK;
    if ((uintptr_t)m.p % m.es) return failf(ctx, RT_EINVAL, "%s: %s is not aligned to its %d-byte elements", fn, m.name, m.es);
    if (m.ld < m.width)
        return failf(ctx, RT_EINVAL, "%s: the row stride of %s (%lld) is less than its width (%lld)", fn, m.name, (long long)m.ld,
                     (long long)m.width);
    if (m.ld > MAX_DIM)
        return failf(ctx, RT_EUNSUPPORTED, "%s: the row stride of %s (%lld) exceeds %lld", fn, m.name, (long long)m.ld,
                     (long long)MAX_DIM);
    return RT_OK;
}

// No output may share memory with an input or another output.
int check_disjoint(rt_ctx* ctx, const char* fn, const Mat* in, int nin, const Mat* out, int nout) {
    for (int i = 0; i < nout; ++i) {
        for (int j = 0; j < nin; ++j)
            if (overlap(out[i], in[j])) return failf(ctx, RT_EINVAL, "%s: %s and %s overlap", fn, out[i].name, in[j].name);
        for (int j = 0; j < i; ++j)
            if (overlap(out[i], out[j])) return failf(ctx, RT_EINVAL, "%s: %s and %s overlap", fn, out[i].name, out[j].name);
    }
    return RT_OK;
}

int check_ws(rt_ctx* ctx, const char* fn, const void* ws, size_t have, size_t need) {
    if (need == 0) return RT_OK;
    if (!ws) return failf(ctx, RT_EINVAL, "%s: workspace is NULL (%zu bytes needed)", fn, need);
    if ((uintptr_t)ws % 16) return failf(ctx, RT_EINVAL, "%s: workspace is not aligned to 16 bytes", fn);
    if (have < need) return failf(ctx, RT_EINVAL, "%s: workspace of %zu bytes, %zu needed", fn, have, need);
    return RT_OK;
}

// ---- matrix products ----------------------------------------------------------------------------------------------


// Few rows against weights as they lie in memory: the weights' bytes are all the time there is.
bool skinny_sizes(const Product& p) { return p.M <= SKINNY_ROWS && p.lx == LK && p.lw == LI && p.N >= 4; }

void plan_skinny(int cus, int dtype, const Product& p, Plan& pl) {
    const int es = elem_size(dtype);
    pl.skinny = true;
    pl.nslot = p.epi == EPI_GATED ? 2 : 1;
    pl.Np = (int)up(p.N, 4);
    // Lanes of a row (gemv_kernel): 16 where that gives every CU a slab, or where there is so much to read that lines should
    // be read whole by one workgroup (32 MB: 6 us of the chip); else as few as give more workgroups.
    const int64_t all = p.K * p.N * es * pl.nslot;
    pl.li = 16;
    if (p.M <= GEMV_ROWS && all < (32 << 20))
        while (pl.li > 4 && p.N / (4 * pl.li) < cus) pl.li /= 2;
    const int cols = 4 * pl.li;
    pl.tiles_n = (p.N + cols - 1) / cols;
    // K is split where columns alone leave CUs idle.  A second launch to join the splits costs about 4 us, in which one CU reads
    // some 256 KB: workgroups that read less than twice that are not split.
    const int64_t steps = (p.K + 31) / 32, bytes = p.K * cols * es * pl.nslot;
    int64_t s = bytes >= (512 << 10) ? cus / pl.tiles_n : 1;
    if (s > steps / SK_WAVES) s = steps / SK_WAVES;
    pl.splits = s < 1 ? 1 : (int)s;
    pl.part_bytes = pl.splits > 1 ? (size_t)pl.splits * pl.nslot * p.M * pl.Np * sizeof(float) : 0;
}

int plan_product(rt_ctx* ctx, int cus, int dtype, const Product& p, bool al, Plan& pl) {
    pl.skinny = false;
    const int ke = 128 / elem_size(dtype);
    // Three tiles: 256 x 256, 128 x 128, 64 x 64 columns of C (the gate's and up's count as one: 128, 64, 64), and K split over s
    // workgroups.  With L workgroups side by side on a CU (at most `fit`, what its LDS holds) a step (128 bytes of k) takes the
    // larger of `least`, what one workgroup waits for memory and barriers, and L * `each`, what the matrix core (16-bit tiles
    // below 256: LDS) needs; splits are joined by another launch, which reads what they wrote.  By measurement, in us:
    // (of long sums; the epilogue's bytes are not in it: where those count, products take up to twice what this says)
    //   16-bit: 256 x 256 1.65 / 1.65;  128 x 128 0.7 / 0.5;  64 x 64 0.7 / 0.25        float32: 128 x 128 2.2 / 1.9;  64 x 64 0.8 / 0.5
    struct Size { int bm, cn, fit; double least, each; };
    const int half = p.epi == EPI_GATED ? 2 : 1;
    const bool f32 = dtype == RT_F32;
    const Size sizes[3] = {{64, 64, half == 2 ? 3 : 5, f32 ? 0.8 : 0.7, (f32 ? 0.5 : 0.25) * half},
                           {128, 128 / half, 2, f32 ? 2.2 : 0.7, f32 ? 1.9 : 0.5}, {256, 256 / half, 1, 1.65, 1.65}};
    pl.nslot = p.epi == EPI_GATED ? 2 : p.nbatch;
    pl.Np = (int)up(p.No > p.N ? p.No : p.N, 4);
    const int64_t nk = (p.K + ke - 1) / ke, steps = nk * p.nseg;
    double best = 1e300;
    int64_t tm = 0, tn = 0;
    for (int i = 0; i < (al && !f32 ? 3 : 2); ++i) {
        const Size& z = sizes[i];
        const int64_t m = (p.M + z.bm - 1) / z.bm, n = (p.N + z.cn - 1) / z.cn, tiles = m * n * p.nbatch;
        if (m * n > MAX_TILES) continue;
        for (int64_t k = 1; k <= 32 && (k == 1 || (k * 2 <= steps && tiles * k <= 2 * cus)); k *= 2) {
            const int64_t per = (steps + k - 1) / k, load = (tiles * k + cus - 1) / cus;
            const double join = k > 1 ? 5.0 + (double)k * pl.nslot * p.M * pl.Np * 8 / 4.5e6 : 0.0;
            auto together = [&](int64_t n) { return n * z.each > z.least ? n * z.each : n ? z.least : 0.0; };
            const double t = per * (load / z.fit * together(z.fit) + together(load % z.fit)) + join;
            if (t >= best) continue;
            best = t;
            pl.bm = z.bm;
            pl.per_split = (int)per;
            pl.splits = (int)((steps + per - 1) / per);
            tm = m;
            tn = n;
        }
    }
    if (tm == 0 || steps > 0x7fffffff)
        return failf(ctx, RT_EUNSUPPORTED, "a product of %lld x %d over %lld is larger than one launch covers", (long long)p.M, p.N,
                     (long long)p.K);
    pl.tiles_m = (int)tm;
    pl.tiles_n = (int)tn;
    pl.nk = (int)nk;
    pl.part_bytes = pl.splits > 1 ? (size_t)pl.splits * pl.nslot * p.M * pl.Np * sizeof(float) : 0;
    return RT_OK;
}

int run_product(rt_ctx* ctx, const RtCtxView& v, int dtype, const Product& p, GemmArgs& a) {
    Plan pl;
    const int es = elem_size(dtype), epc = 16 / es, kept = a.kept_narrow ? es : 4;
    a.quads = p.N % 4 == 0;
    for (int i = 0; i < 3; ++i) {
        const int os = p.epi == EPI_GATED && i ? kept : es;
        if (p.epi == EPI_STORE && i >= p.nrun) break;
        a.quads = a.quads && (uintptr_t)a.o[i] % (4 * os) == 0 && a.ldo[i] % (4 * os) == 0;
    }
    if (p.epi == EPI_GATED_BWD) a.quads = a.quads && (uintptr_t)a.e[0] % (4 * kept) == 0 && (uintptr_t)a.e[1] % (4 * kept) == 0 && a.lde % (4 * kept) == 0;
    if (skinny_sizes(p)) {
        plan_skinny(v.cu_count, dtype, p, pl);
        HIPCHK(ctx, dtype == RT_F32 ? launch_skinny<RT_F32>(v.stream, p, pl, a)
                    : dtype == RT_BF16 ? launch_skinny<RT_BF16>(v.stream, p, pl, a) : launch_skinny<RT_F16>(v.stream, p, pl, a));
        return RT_OK;
    }
    bool al = (p.xpad || (p.lx == LK ? p.K : p.M) % epc == 0) && (p.wpad || (p.lw == LK ? p.K : p.N) % epc == 0) && a.ldx[0] % 16 == 0 && a.ldw[0] % 16 == 0;
    for (int i = 0; i < 2; ++i) al = al && (uintptr_t)a.x[i] % 16 == 0 && (uintptr_t)a.w[i] % 16 == 0;
    const int rc = plan_product(ctx, v.cu_count, dtype, p, al, pl);
    if (rc) return rc;
    HIPCHK(ctx, dtype == RT_F32 ? launch_product<RT_F32>(v.stream, p, pl, a, al)
                : dtype == RT_BF16 ? launch_product<RT_BF16>(v.stream, p, pl, a, al) : launch_product<RT_F16>(v.stream, p, pl, a, al));
    return RT_OK;
}

// rows x bytes of zeros: a weight gradient of no tokens.
__global__ void zero_rows_kernel(char* p, long long ld, long long rows, long long width) {
    for (long long r = blockIdx.x; r < rows; r += gridDim.x)
        for (long long c = threadIdx.x * 2; c < width; c += blockDim.x * 2) *(unsigned short*)(p + r * ld + c) = 0;
}

int zero_rows(rt_ctx* ctx, hipStream_t st, void* p, int64_t ld, int64_t rows, int64_t width) {
    if (!p) return RT_OK;
    hipLaunchKernelGGL(zero_rows_kernel, dim3((unsigned)(rows < 1024 ? rows : 1024)), dim3(256), 0, st, (char*)p, ld, rows, width);
    HIPCHK(ctx, hipGetLastError());
    return RT_OK;
}

// ---- the gated feed-forward block ---------------------------------------------------------------------------------
struct Ffn {
    rt_gated_ffn a;                // with its strides filled in
    int es, kept;                  // bytes of an element; of the kept gate's and up's
    int64_t ldh;                   // elements; h, dgate and dup lie in the workspace
    size_t h_bytes;
    bool pad;                      // many rows: operands of odd widths are copied, padded
    size_t pad_x, pad_in, pad_down, pad_dout;      // bytes of a copy, 0: none is needed
    Product gated, down;           // forward
    Product dh, dx, dw_in, dw_down;
    size_t ws, part;               // bytes of the workspace, and of partial sums in it
};

constexpr int PAD_ROWS = 1024;

// Raises `most` to the bytes of partial sums this product can need.
int most_part_bytes(rt_ctx* ctx, int cus, int dtype, const Product& p, size_t& most) {
    Plan pl;
    if (skinny_sizes(p)) {
        plan_skinny(cus, dtype, p, pl);
        if (pl.part_bytes > most) most = pl.part_bytes;
        return RT_OK;
    }
    for (int al = 0; al < 2; ++al) {
        const int rc = plan_product(ctx, cus, dtype, p, al, pl);
        if (rc) return rc;
        if (pl.part_bytes > most) most = pl.part_bytes;
    }
    return RT_OK;
}

// The sizes, and the products and workspace of the forward or the backward pass.
int ffn_make(rt_ctx* ctx, const char* fn, const rt_gated_ffn* in, int cus, bool backward, Ffn& f) {
    if (!in) return failf(ctx, RT_EINVAL, "%s: the arguments are NULL", fn);
    f.a = *in;
    rt_gated_ffn& a = f.a;
    if (a.dtype != RT_F32 && a.dtype != RT_BF16 && a.dtype != RT_F16) return failf(ctx, RT_EINVAL, "%s: unknown dtype %d", fn, a.dtype);
    if (a.pre_dtype != RT_F32 && a.pre_dtype != a.dtype)
        return failf(ctx, RT_EINVAL, "%s: pre_dtype %d is neither RT_F32 nor the arrays' type", fn, a.pre_dtype);
    if (a.act < RT_ACT_SILU || a.act > RT_ACT_SIGMOID) return failf(ctx, RT_EINVAL, "%s: unknown activation %d", fn, a.act);
    if (a.x_lo && a.dtype == RT_F32) return failf(ctx, RT_EINVAL, "%s: x_lo is for 16-bit types", fn);
    if (!isfinite(a.alpha)) return failf(ctx, RT_EINVAL, "%s: alpha is not finite", fn);
    if (a.T < 0 || a.T > MAX_ROWS) return failf(ctx, RT_EINVAL, "%s: T = %lld", fn, (long long)a.T);
    if (a.d_in < 1 || a.d_ff < 1 || a.d_out < 1 || a.d_in > MAX_DIM || a.d_ff > MAX_DIM || a.d_out > MAX_DIM)
        return failf(ctx, RT_EINVAL, "%s: widths %d, %d, %d: each must be in [1, %lld]", fn, a.d_in, a.d_ff, a.d_out, (long long)MAX_DIM);
    f.es = elem_size(a.dtype);
    f.kept = elem_size(a.pre_dtype);
    if (!a.ldx) a.ldx = a.d_in;
    if (!a.ld_in) a.ld_in = a.d_ff;
    if (!a.ld_down) a.ld_down = a.d_out;
    if (!a.ld_out) a.ld_out = a.d_out;
    if (!a.ld_pre) a.ld_pre = a.d_ff;
    f.ldh = up(a.d_ff, 16 / f.es);
    f.h_bytes = (size_t)up(a.T * f.ldh * f.es, 256);
    // Odd widths make every product read its operands unaligned, at half the speed of the kernels for whole chunks (1777 x 1001 x
    // 2731 f16 training step 449 us, with copies 270 us); one pass over the weights before costs as much as a few hundred rows
    // gain.  (x and dout cost as much as some 130 columns of d_ff gain: at 14912 x 3890 x 47 it is the same with and without.)
    f.pad = a.T >= PAD_ROWS;
    const int epc = 16 / f.es;
    auto copy = [&](int64_t rows, int64_t width) { return f.pad && width % epc ? (size_t)up(rows * up(width, epc) * f.es, 256) : (size_t)0; };
    f.pad_x = copy(a.T, a.d_in);
    f.pad_in = copy(a.d_in, a.d_ff);
    f.pad_down = copy(a.d_ff, a.d_out);
    f.pad_dout = copy(a.T, a.d_out);
    f.gated = {LK, LI, EPI_GATED, a.T, a.d_in, a.d_ff, a.x_lo ? 2 : 1, 1};      // x_lo: another run of k's, of the same weights
    f.down = {LK, LI, EPI_STORE, a.T, a.d_ff, a.d_out, 1, 1};
    f.dh = {LK, LK, EPI_GATED_BWD, a.T, a.d_out, a.d_ff, 1, 1};
    f.dx = {LK, LK, EPI_STORE, a.T, a.d_ff, a.d_in, 2, 1};
    f.dw_in = {LI, LI, EPI_STORE, a.d_in, a.T, a.d_ff, 1, 2};
    f.dw_down = {LI, LI, EPI_STORE, a.d_ff, a.T, a.d_out, 1, 1};
    if (f.pad) {
        // h, dgate and dup are written with zeros behind their rows, and count as padded where they are read
        f.gated.No = f.dh.No = (int)f.ldh;
        f.down.xpad = f.dx.xpad = f.dw_down.xpad = f.dw_in.wpad = true;
        f.gated.xpad = f.dw_in.xpad = f.pad_x;
        f.gated.wpad = f.dx.wpad = f.pad_in;
        f.down.wpad = f.dh.wpad = f.pad_down;
        f.dh.xpad = f.dw_down.wpad = f.pad_dout;
    }
    f.ws = f.part = 0;
    if (a.T == 0) return RT_OK;
    // whichever kernels the call's alignment lets it use, with and without x_lo
    Product other = f.gated;
    other.nseg = 3 - other.nseg;
    const Product* forward[] = {&f.gated, &other, &f.down};
    const Product* back[] = {&f.dh, &f.dx, &f.dw_in, &f.dw_down};
    for (int i = 0; i < (backward ? 4 : 3); ++i) {
        const int rc = most_part_bytes(ctx, cus, a.dtype, backward ? *back[i] : *forward[i], f.part);
        if (rc) return rc;
    }
    const size_t copies = 2 * f.pad_x + 2 * f.pad_in + f.pad_down;      // (x_lo too)
    f.ws = (backward ? 3 : 1) * f.h_bytes + up(f.part, 256) + copies + (backward ? f.pad_dout : 0);
    return RT_OK;
}

void set_x(GemmArgs& g, const void* p0, const void* p1, int64_t ld) {
    g.x[0] = (const char*)p0;
    g.x[1] = (const char*)p1;
    g.ldx[0] = g.ldx[1] = ld;
}
void set_w(GemmArgs& g, const void* p0, const void* p1, int64_t ld) {
    g.w[0] = (const char*)p0;
    g.w[1] = (const char*)p1;
    g.ldw[0] = g.ldw[1] = ld;
}
void set_o(GemmArgs& g, int i, void* p, int64_t ld) {
    g.o[i] = (char*)p;
    g.ldo[i] = ld;
}

// Operands as the products read them: the caller's, or padded copies of them at `at` in the workspace.
struct Operands {
    const void *x, *x_lo, *w_gate, *w_up, *w_down, *dout;
    int64_t ldx, ld_in, ld_down, ld_dout;      // bytes
};

int ffn_operands(rt_ctx* ctx, const RtCtxView& v, const Ffn& f, const void* dout, int64_t ld_dout, char* at, Operands& o) {
    const rt_gated_ffn& a = f.a;
    const int64_t es = f.es, epc = 16 / es;
    o = {a.x, a.x_lo, a.w_gate, a.w_up, a.w_down, dout, a.ldx * es, a.ld_in * es, a.ld_down * es, ld_dout * es};
    PadArgs p;
    p.n = 0;
    auto copy = [&](const void*& src, int64_t ld, int64_t rows, int64_t width, size_t bytes) {
        if (!bytes || !src) return;
        p.m[p.n++] = {(const char*)src, at, ld, up(width, epc) * es, rows, (int)width};
        src = at;
        at += bytes;
    };
    copy(o.x, o.ldx, a.T, a.d_in, f.pad_x);
    if (!dout) copy(o.x_lo, o.ldx, a.T, a.d_in, f.pad_x);
    copy(o.w_gate, o.ld_in, a.d_in, a.d_ff, f.pad_in);
    copy(o.w_up, o.ld_in, a.d_in, a.d_ff, f.pad_in);
    copy(o.w_down, o.ld_down, a.d_ff, a.d_out, f.pad_down);
    copy(o.dout, o.ld_dout, a.T, a.d_out, f.pad_dout);
    if (f.pad_x) o.ldx = up(a.d_in, epc) * es;
    if (f.pad_in) o.ld_in = up(a.d_ff, epc) * es;
    if (f.pad_down) o.ld_down = up(a.d_out, epc) * es;
    if (f.pad_dout) o.ld_dout = up(a.d_out, epc) * es;
    if (p.n)
        HIPCHK(ctx, a.dtype == RT_F32 ? launch_pad<RT_F32>(v.stream, p) : a.dtype == RT_BF16 ? launch_pad<RT_BF16>(v.stream, p)
                                                                                              : launch_pad<RT_F16>(v.stream, p));
    return RT_OK;
}

int ffn_forward(rt_ctx* ctx, const RtCtxView& v, const Ffn& f, char* ws) {
    const rt_gated_ffn& a = f.a;
    const int64_t es = f.es;
    char* h = ws;
    Operands o;
    int rc = ffn_operands(ctx, v, f, nullptr, 0, ws + f.h_bytes + up(f.part, 256), o);
    if (rc) return rc;
    GemmArgs g;
    memset(&g, 0, sizeof g);
    g.part = (float*)(ws + f.h_bytes);
    g.act = a.act;
    g.alpha = a.alpha;
    set_x(g, o.x, a.x_lo ? o.x_lo : o.x, o.ldx);
    set_w(g, o.w_gate, o.w_up, o.ld_in);
    set_o(g, 0, h, f.ldh * es);
    set_o(g, 1, a.pre_gate, a.ld_pre * f.kept);
    set_o(g, 2, a.pre_up, a.ld_pre * f.kept);
    g.kept_narrow = f.kept < 4;
    if ((rc = run_product(ctx, v, a.dtype, f.gated, g))) return rc;
    set_x(g, h, h, f.ldh * es);
    set_w(g, o.w_down, o.w_down, o.ld_down);
    set_o(g, 0, a.out, a.ld_out * es);
    return run_product(ctx, v, a.dtype, f.down, g);
}

int ffn_backward(rt_ctx* ctx, const RtCtxView& v, const Ffn& f, const rt_gated_ffn_grads& r, char* ws) {
    const rt_gated_ffn& a = f.a;
    const int64_t es = f.es, ldh = f.ldh * es;
    char *dg = ws, *du = ws + f.h_bytes, *h = ws + 2 * f.h_bytes;
    GemmArgs g;
    memset(&g, 0, sizeof g);
    g.part = (float*)(ws + 3 * f.h_bytes);
    g.act = a.act;
    g.alpha = a.alpha;
    Operands o;
    int rc = ffn_operands(ctx, v, f, r.dout, r.ld_dout, ws + 3 * f.h_bytes + up(f.part, 256), o);
    if (rc) return rc;
    // dh = dout Wd^T, and from it what the gate's and up's sums get, and h again
    set_x(g, o.dout, o.dout, o.ld_dout);
    set_w(g, o.w_down, o.w_down, o.ld_down);
    set_o(g, 0, dg, ldh);
    set_o(g, 1, du, ldh);
    set_o(g, 2, h, ldh);
    g.e[0] = (const char*)a.pre_gate;
    g.e[1] = (const char*)a.pre_up;
    g.lde = a.ld_pre * f.kept;
    g.kept_narrow = f.kept < 4;
    if ((rc = run_product(ctx, v, a.dtype, f.dh, g))) return rc;
    if (r.dx) {                      // dx = dgate Wg^T + dup Wu^T: one sum over both
        set_x(g, dg, du, ldh);
        set_w(g, o.w_gate, o.w_up, o.ld_in);
        set_o(g, 0, r.dx, r.ld_dx * es);
        if ((rc = run_product(ctx, v, a.dtype, f.dx, g))) return rc;
    }
    if (r.dw_gate || r.dw_up) {      // x^T dgate and x^T dup side by side
        Product p = f.dw_in;
        set_x(g, o.x, o.x, o.ldx);
        set_w(g, r.dw_gate ? dg : du, r.dw_up ? du : dg, ldh);
        set_o(g, 0, r.dw_gate ? r.dw_gate : r.dw_up, r.ld_dw_in * es);
        set_o(g, 1, r.dw_up, r.ld_dw_in * es);
        p.nrun = r.dw_gate && r.dw_up ? 2 : 1;
        if ((rc = run_product(ctx, v, a.dtype, p, g))) return rc;
    }
    if (r.dw_down) {
        set_x(g, h, h, ldh);
        set_w(g, o.dout, o.dout, o.ld_dout);
        set_o(g, 0, r.dw_down, r.ld_dw_down * es);
        if ((rc = run_product(ctx, v, a.dtype, f.dw_down, g))) return rc;
    }
    return RT_OK;
}

// ---- the norms ----------------------------------------------------------------------------------------------------
struct Norm {
    rt_block_norm a;
    int es;
    int tpr, tpr_back;               // threads of a row
    int together;
    int units;
    int64_t rows_per_unit;
    size_t part, ws;                 // bytes of one [units][d] array; of the workspace
};

int norm_make(rt_ctx* ctx, const char* fn, const rt_block_norm* in, int cus, Norm& m) {
    if (!in) return failf(ctx, RT_EINVAL, "%s: the arguments are NULL", fn);
    m.a = *in;
    rt_block_norm& a = m.a;
    if (a.dtype != RT_F32 && a.dtype != RT_BF16 && a.dtype != RT_F16) return failf(ctx, RT_EINVAL, "%s: unknown dtype %d", fn, a.dtype);
    if (a.kind != RT_NORM_RMS && a.kind != RT_NORM_LAYER) return failf(ctx, RT_EINVAL, "%s: unknown kind of norm %d", fn, a.kind);
    m.es = elem_size(a.dtype);
    const int d_max = a.dtype == RT_F32 ? 16384 : 32768;
    if (a.T < 0 || a.T > MAX_ROWS) return failf(ctx, RT_EINVAL, "%s: T = %lld", fn, (long long)a.T);
    if (a.d < 1) return failf(ctx, RT_EINVAL, "%s: d = %d", fn, a.d);
    if (a.d > d_max) return failf(ctx, RT_EUNSUPPORTED, "%s: d = %d: at most %d of this type fit a workgroup's registers", fn, a.d, d_max);
    if (!(a.eps >= 0.0f) || !isfinite(a.eps) || !isfinite(a.res_scale) || !isfinite(a.branch_scale) || !isfinite(a.w_offset))
        return failf(ctx, RT_EINVAL, "%s: eps must be >= 0, and it and the scales finite", fn);
    if (a.gate && a.rows_per_gate < 1) return failf(ctx, RT_EINVAL, "%s: rows_per_gate = %lld", fn, (long long)a.rows_per_gate);
    if (!a.gate || a.rows_per_gate > (a.T > 0 ? a.T : 1)) a.rows_per_gate = a.T > 0 ? a.T : 1;
    if (!a.ldx) a.ldx = a.d;
    if (!a.ld_branch) a.ld_branch = a.d;
    if (!a.ldy) a.ldy = a.d;
    if (!a.ldn) a.ldn = a.d;
    if (!a.ld_gate) a.ld_gate = a.d;
    if (a.T > 0x7fffffffll)
        return failf(ctx, RT_EUNSUPPORTED, "%s: T = %lld rows are more than one launch covers", fn, (long long)a.T);
    const int chunks = (a.d + 16 / m.es - 1) / (16 / m.es);
    // A row to a wave where it is short; with fewer rows than CUs, to a workgroup sooner (a chunk a thread: what counts is
    // how long one row takes)
    const bool few = a.T < cus;
    m.tpr = chunks <= (few ? 64 : 256) ? 64 : chunks <= 1024 ? 256 : 1024;
    // backward: five arrays and three sums of a chunk of eight values are about what a thread's registers hold; two chunks of
    // four float32 values
    const int per = a.dtype == RT_F32 ? 2 : 1;
    m.tpr_back = chunks <= 64 * (few ? 1 : per) ? 64 : chunks <= 256 * per ? 256 : chunks <= 1024 ? 512 : 1024;
    // units: as many workgroups a CU as their registers allow, consecutive rows each; whole gates where a unit can hold some
    const int64_t fill = (int64_t)cus * (m.tpr_back >= 512 ? 1 : 2);
    int64_t r = (a.T + fill - 1) / fill;
    const int waves = m.tpr_back == 64 ? 4 : 1;
    if (m.tpr_back == 64 && r < waves) r = waves;
    // a wave walks four gates at least before a segment's end is worth an exchange between waves
    m.together = a.rows_per_gate >= 16;
    if (a.gate && waves > 1 && !m.together) r = up(r, waves * a.rows_per_gate);
    else if (a.gate && a.rows_per_gate <= r) r = r / a.rows_per_gate * a.rows_per_gate;
    if (r < 1) r = 1;
    m.rows_per_unit = r;
    m.units = (int)((a.T + r - 1) / r);
    m.part = (size_t)m.units * a.d * sizeof(float);
    m.ws = m.part * 2 + (a.gate && a.rows_per_gate > r ? 2 * m.part : 0);
    return RT_OK;
}

int run_norm(rt_ctx* ctx, hipStream_t st, int dtype, const NormArgs& a, int tpr, bool back, bool al) {
    HIPCHK(ctx, dtype == RT_F32 ? launch_norm<RT_F32>(st, a, tpr, back, al)
                : dtype == RT_BF16 ? launch_norm<RT_BF16>(st, a, tpr, back, al) : launch_norm<RT_F16>(st, a, tpr, back, al));
    return RT_OK;
}

struct Aligned {                     // whether every row of every matrix starts on 16 bytes and ends on a whole chunk
    bool ok = true;
    int es;
    void operator()(const void* p, int64_t ld, int64_t width) {
        if (p) ok = ok && (uintptr_t)p % 16 == 0 && ld * es % 16 == 0 && width * es % 16 == 0;
    }
};

void norm_args(const Norm& m, NormArgs& k) {
    const rt_block_norm& a = m.a;
    const int64_t es = m.es;
    memset(&k, 0, sizeof k);
    k.T = a.T; k.d = a.d; k.kind = a.kind;
    k.eps = a.eps; k.rs = a.res_scale; k.bs = a.branch_scale; k.w_off = a.w_offset; k.rpg = a.rows_per_gate;
    k.x = (const char*)a.x; k.b = (const char*)a.branch; k.gate = (const char*)a.gate;
    k.w_post = (const char*)a.w_post; k.w_pre = (const char*)a.w_pre;
    k.y = (char*)a.y; k.n = (char*)a.n; k.n_lo = (char*)a.n_lo;
    k.ldx = a.ldx * es; k.ldb = a.ld_branch * es; k.ldy = a.ldy * es; k.ldn = a.ldn * es; k.ldg = a.ld_gate * es;
}

}  // namespace

extern "C" {

int rt_ctx_stream(rt_ctx* ctx, void** stream) {
    if (!ctx) return RT_EINVAL;
    if (!stream) return failf(ctx, RT_EINVAL, "rt_ctx_stream: stream is NULL");
    RtCtxView v;
    rt_ctx_view(ctx, &v);
    *stream = (void*)v.stream;
    return RT_OK;
}

int rt_gated_ffn_workspace(rt_ctx* ctx, const rt_gated_ffn* a, int backward, size_t* bytes) {
    if (!ctx) return RT_EINVAL;
    if (!bytes) return failf(ctx, RT_EINVAL, "rt_gated_ffn_workspace: bytes is NULL");
    RtCtxView v;
    rt_ctx_view(ctx, &v);
    Ffn f;
    const int rc = ffn_make(ctx, "rt_gated_ffn_workspace", a, v.cu_count, backward != 0, f);
    if (rc) return rc;
    *bytes = f.ws;
    return RT_OK;
}

int rt_gated_ffn_dev(rt_ctx* ctx, const rt_gated_ffn* args, void* ws, size_t ws_bytes) {
    static const char fn[] = "rt_gated_ffn_dev";
    if (!ctx) return RT_EINVAL;
    RtCtxView v;
    rt_ctx_view(ctx, &v);
    Ffn f;
    int rc = ffn_make(ctx, fn, args, v.cu_count, false, f);
    if (rc) return rc;
    const rt_gated_ffn& a = f.a;
    const Mat in[] = {{"x", a.x, a.T, a.d_in, a.ldx, f.es}, {"w_gate", a.w_gate, a.d_in, a.d_ff, a.ld_in, f.es}, {"w_up", a.w_up, a.d_in, a.d_ff, a.ld_in, f.es},
                      {"w_down", a.w_down, a.d_ff, a.d_out, a.ld_down, f.es}, {"x_lo", a.x_lo, a.T, a.d_in, a.ldx, f.es}};
    const Mat out[] = {{"out", a.out, a.T, a.d_out, a.ld_out, f.es}, {"pre_gate", a.pre_gate, a.T, a.d_ff, a.ld_pre, f.kept},
                       {"pre_up", a.pre_up, a.T, a.d_ff, a.ld_pre, f.kept}, {"the workspace", ws, 1, (int64_t)f.ws, (int64_t)f.ws, 1}};
    for (int i = 0; i < 5; ++i)
        if ((rc = check_mat(ctx, fn, in[i], i < 4))) return rc;
    for (int i = 0; i < 3; ++i)
        if ((rc = check_mat(ctx, fn, out[i], i == 0))) return rc;
    if (!a.pre_gate != !a.pre_up) return failf(ctx, RT_EINVAL, "%s: give both of pre_gate and pre_up, or neither", fn);
    if (a.T == 0) return RT_OK;
    if ((rc = check_ws(ctx, fn, ws, ws_bytes, f.ws)) || (rc = check_disjoint(ctx, fn, in, 5, out, 4))) return rc;
    DeviceScope dev(v.device);
    HIPCHK(ctx, dev.err);
    return ffn_forward(ctx, v, f, (char*)ws);
}

int rt_gated_ffn_backward_dev(rt_ctx* ctx, const rt_gated_ffn* args, const rt_gated_ffn_grads* grads, void* ws, size_t ws_bytes) {
    static const char fn[] = "rt_gated_ffn_backward_dev";
    if (!ctx) return RT_EINVAL;
    if (!grads) return failf(ctx, RT_EINVAL, "%s: the gradients are NULL", fn);
    RtCtxView v;
    rt_ctx_view(ctx, &v);
    Ffn f;
    int rc = ffn_make(ctx, fn, args, v.cu_count, true, f);
    if (rc) return rc;
    const rt_gated_ffn& a = f.a;
    rt_gated_ffn_grads r = *grads;
    if (!r.ld_dout) r.ld_dout = a.d_out;
    if (!r.ld_dx) r.ld_dx = a.d_in;
    if (!r.ld_dw_in) r.ld_dw_in = a.d_ff;
    if (!r.ld_dw_down) r.ld_dw_down = a.d_out;
    const Mat in[] = {{"x", a.x, a.T, a.d_in, a.ldx, f.es}, {"w_gate", a.w_gate, a.d_in, a.d_ff, a.ld_in, f.es}, {"w_up", a.w_up, a.d_in, a.d_ff, a.ld_in, f.es},
                      {"w_down", a.w_down, a.d_ff, a.d_out, a.ld_down, f.es}, {"pre_gate", a.pre_gate, a.T, a.d_ff, a.ld_pre, f.kept},
                      {"pre_up", a.pre_up, a.T, a.d_ff, a.ld_pre, f.kept}, {"dout", r.dout, a.T, a.d_out, r.ld_dout, f.es}};
    const Mat out[] = {{"dx", r.dx, a.T, a.d_in, r.ld_dx, f.es}, {"dw_gate", r.dw_gate, a.d_in, a.d_ff, r.ld_dw_in, f.es},
                       {"dw_up", r.dw_up, a.d_in, a.d_ff, r.ld_dw_in, f.es}, {"dw_down", r.dw_down, a.d_ff, a.d_out, r.ld_dw_down, f.es},
                       {"the workspace", ws, 1, (int64_t)f.ws, (int64_t)f.ws, 1}};
    for (const Mat& m : in)
        if ((rc = check_mat(ctx, fn, m, true))) return rc;
    for (int i = 0; i < 4; ++i)
        if ((rc = check_mat(ctx, fn, out[i], false))) return rc;
    if (a.T > 0 && ((rc = check_ws(ctx, fn, ws, ws_bytes, f.ws)))) return rc;
    if ((rc = check_disjoint(ctx, fn, in, 7, out, a.T > 0 ? 5 : 4))) return rc;
    DeviceScope dev(v.device);
    HIPCHK(ctx, dev.err);
    if (a.T == 0) {
        if ((rc = zero_rows(ctx, v.stream, r.dw_gate, r.ld_dw_in * f.es, a.d_in, (int64_t)a.d_ff * f.es)) ||
            (rc = zero_rows(ctx, v.stream, r.dw_up, r.ld_dw_in * f.es, a.d_in, (int64_t)a.d_ff * f.es)))
            return rc;
        return zero_rows(ctx, v.stream, r.dw_down, r.ld_dw_down * f.es, a.d_ff, (int64_t)a.d_out * f.es);
    }
    return ffn_backward(ctx, v, f, r, (char*)ws);
}

int rt_block_norm_workspace(rt_ctx* ctx, const rt_block_norm* a, size_t* bytes) {
    if (!ctx) return RT_EINVAL;
    if (!bytes) return failf(ctx, RT_EINVAL, "rt_block_norm_workspace: bytes is NULL");
    RtCtxView v;
    rt_ctx_view(ctx, &v);
    Norm m;
    const int rc = norm_make(ctx, "rt_block_norm_workspace", a, v.cu_count, m);
    if (rc) return rc;
    *bytes = m.ws;
    return RT_OK;
}

int rt_block_norm_dev(rt_ctx* ctx, const rt_block_norm* args) {
    static const char fn[] = "rt_block_norm_dev";
    if (!ctx) return RT_EINVAL;
    RtCtxView v;
    rt_ctx_view(ctx, &v);
    Norm m;
    int rc = norm_make(ctx, fn, args, v.cu_count, m);
    if (rc) return rc;
    const rt_block_norm& a = m.a;
    const int64_t gates = (a.T + a.rows_per_gate - 1) / a.rows_per_gate;
    const Mat in[] = {{"x", a.x, a.T, a.d, a.ldx, m.es}, {"branch", a.branch, a.T, a.d, a.ld_branch, m.es}, {"gate", a.gate, gates, a.d, a.ld_gate, m.es},
                      {"w_post", a.w_post, 1, a.d, a.d, m.es}, {"w_pre", a.w_pre, 1, a.d, a.d, m.es}};
    const Mat out[] = {{"y", a.y, a.T, a.d, a.ldy, m.es}, {"n", a.n, a.T, a.d, a.ldn, m.es}, {"n_lo", a.n_lo, a.T, a.d, a.ldn, m.es}};
    for (int i = 0; i < 5; ++i)
        if ((rc = check_mat(ctx, fn, in[i], i == 0))) return rc;
    for (const Mat& o : out)
        if ((rc = check_mat(ctx, fn, o, false))) return rc;
    if (a.gate && !a.branch) return failf(ctx, RT_EINVAL, "%s: a gate without a branch", fn);
    if (a.n_lo && (a.dtype == RT_F32 || !a.n)) return failf(ctx, RT_EINVAL, "%s: n_lo is for 16-bit types, beside n", fn);
    if (a.T == 0) return RT_OK;
    if (!a.y && !a.n) return failf(ctx, RT_EINVAL, "%s: y and n are both NULL", fn);
    // rows are read before they are written: an output may take the place of x or of branch, whole
    for (const Mat& o : out)
        for (int i = 0; i < 5; ++i)
            if (overlap(o, in[i]) && !(i < 2 && &o != &out[2] && same_place(o, in[i])))
                return failf(ctx, RT_EINVAL, "%s: %s and %s overlap", fn, o.name, in[i].name);
    if (overlap(out[0], out[1])) return failf(ctx, RT_EINVAL, "%s: y and n overlap", fn);
    for (int i = 0; i < 2; ++i)
        if (overlap(out[2], out[i])) return failf(ctx, RT_EINVAL, "%s: n_lo and %s overlap", fn, out[i].name);
    DeviceScope dev(v.device);
    HIPCHK(ctx, dev.err);
    NormArgs k;
    norm_args(m, k);
    Aligned al;
    al.es = m.es;
    for (const Mat& x : in) al(x.p, x.ld, x.width);
    for (const Mat& x : out) al(x.p, x.ld, x.width);
    return run_norm(ctx, v.stream, a.dtype, k, m.tpr, false, al.ok);
}

int rt_block_norm_backward_dev(rt_ctx* ctx, const rt_block_norm* args, const rt_block_norm_grads* grads, void* ws, size_t ws_bytes) {
    static const char fn[] = "rt_block_norm_backward_dev";
    if (!ctx) return RT_EINVAL;
    if (!grads) return failf(ctx, RT_EINVAL, "%s: the gradients are NULL", fn);
    RtCtxView v;
    rt_ctx_view(ctx, &v);
    Norm m;
    int rc = norm_make(ctx, fn, args, v.cu_count, m);
    if (rc) return rc;
    const rt_block_norm& a = m.a;
    rt_block_norm_grads r = *grads;
    if (!r.ld_dy) r.ld_dy = a.d;
    if (!r.ld_dn) r.ld_dn = a.d;
    if (!r.ld_dx) r.ld_dx = a.d;
    if (!r.ld_dbranch) r.ld_dbranch = a.d;
    if (!r.ld_dgate) r.ld_dgate = a.d;
    const int64_t gates = (a.T + a.rows_per_gate - 1) / a.rows_per_gate;
    // without a branch y is res_scale * x, and x stands in for a y that was not written
    const bool from_x = !a.y && !a.branch;
    const Mat yin = from_x ? Mat{"x", a.x, a.T, a.d, a.ldx, m.es} : Mat{"y", a.y, a.T, a.d, a.ldy, m.es};
    const Mat in[] = {yin, {"branch", a.branch, a.T, a.d, a.ld_branch, m.es}, {"dy", r.dy, a.T, a.d, r.ld_dy, m.es}, {"dn", r.dn, a.T, a.d, r.ld_dn, m.es},
                      {"gate", a.gate, gates, a.d, a.ld_gate, m.es}, {"w_post", a.w_post, 1, a.d, a.d, m.es}, {"w_pre", a.w_pre, 1, a.d, a.d, m.es}};
    const Mat out[] = {{"dx", r.dx, a.T, a.d, r.ld_dx, m.es}, {"dbranch", r.dbranch, a.T, a.d, r.ld_dbranch, m.es}, {"dgate", r.dgate, gates, a.d, r.ld_dgate, m.es},
                       {"dw_post", r.dw_post, 1, a.d, a.d, m.es}, {"dw_pre", r.dw_pre, 1, a.d, a.d, m.es},
                       {"the workspace", ws, 1, (int64_t)m.ws, (int64_t)m.ws, 1}};
    for (int i = 0; i < 7; ++i)
        if ((rc = check_mat(ctx, fn, in[i], i == 0 && r.dn))) return rc;
    for (int i = 0; i < 5; ++i)
        if ((rc = check_mat(ctx, fn, out[i], false))) return rc;
    if (a.T > 0 && !r.dy && !r.dn) return failf(ctx, RT_EINVAL, "%s: dy and dn are both NULL", fn);
    if (a.gate && !a.branch) return failf(ctx, RT_EINVAL, "%s: a gate without a branch", fn);
    if (!a.branch && (r.dbranch || r.dgate || r.dw_post)) return failf(ctx, RT_EINVAL, "%s: dbranch, dgate or dw_post without a branch", fn);
    if (!a.gate && r.dgate) return failf(ctx, RT_EINVAL, "%s: dgate without a gate", fn);
    if (a.T > 0 && (rc = check_ws(ctx, fn, ws, ws_bytes, m.ws))) return rc;
    // a row's dx is written when its y, dy and dn have been read, its dbranch when all of it has
    for (int i = 0; i < (a.T > 0 ? 6 : 5); ++i) {
        for (int j = 0; j < 7; ++j) {
            const bool fine = same_place(out[i], in[j]) && ((i == 0 && (j == 0 || j == 2 || j == 3)) || (i == 1 && j < 4));
            if (overlap(out[i], in[j]) && !fine) return failf(ctx, RT_EINVAL, "%s: %s and %s overlap", fn, out[i].name, in[j].name);
        }
        for (int j = 0; j < i; ++j)
            if (overlap(out[i], out[j])) return failf(ctx, RT_EINVAL, "%s: %s and %s overlap", fn, out[i].name, out[j].name);
    }
    DeviceScope dev(v.device);
    HIPCHK(ctx, dev.err);
    if (a.T == 0) {
        if ((rc = zero_rows(ctx, v.stream, r.dw_post, (int64_t)a.d * m.es, 1, (int64_t)a.d * m.es))) return rc;
        return zero_rows(ctx, v.stream, r.dw_pre, (int64_t)a.d * m.es, 1, (int64_t)a.d * m.es);
    }
    NormArgs k;
    norm_args(m, k);
    const int64_t es = m.es;
    k.yin = (const char*)yin.p; k.ldy = yin.ld * es; k.yin_scale = from_x ? a.res_scale : 1.0f;
    k.dy = (const char*)r.dy; k.dn = (const char*)r.dn;
    k.dx = (char*)r.dx; k.db = (char*)r.dbranch; k.dgate = (char*)r.dgate;
    k.lddy = r.ld_dy * es; k.lddn = r.ld_dn * es; k.lddx = r.ld_dx * es; k.lddb = r.ld_dbranch * es; k.lddg = r.ld_dgate * es;
    k.want_post = r.dw_post != nullptr; k.want_pre = r.dw_pre != nullptr && r.dn != nullptr;
    k.rows_per_unit = m.rows_per_unit; k.units = m.units; k.together = m.together;
    k.p_post = (float*)ws; k.p_pre = (float*)((char*)ws + m.part); k.p_gate = (float*)((char*)ws + 2 * m.part);
    k.dw_post = (char*)r.dw_post; k.dw_pre = k.want_pre ? (char*)r.dw_pre : nullptr;
    Aligned al;
    al.es = m.es;
    for (const Mat& x : in) al(x.p, x.ld, x.width);
    for (int i = 0; i < 5; ++i) al(out[i].p, out[i].ld, out[i].width);
    if ((rc = run_norm(ctx, v.stream, a.dtype, k, m.tpr_back, true, al.ok))) return rc;
    if (r.dw_pre && !r.dn && (rc = zero_rows(ctx, v.stream, r.dw_pre, (int64_t)a.d * es, 1, (int64_t)a.d * es))) return rc;
    // what is left to join: the weights' sums, and the gates that more than one unit saw
    const bool gates_left = r.dgate && a.rows_per_gate > m.rows_per_unit;
    const int first = k.want_post || k.want_pre ? 0 : 2, last = gates_left ? 2 + (int)gates : 2;
    if (last > first) {
        HIPCHK(ctx, a.dtype == RT_F32 ? launch_norm_join<RT_F32>(v.stream, k, first, last)
                    : a.dtype == RT_BF16 ? launch_norm_join<RT_BF16>(v.stream, k, first, last)
                                         : launch_norm_join<RT_F16>(v.stream, k, first, last));
    }
    return RT_OK;
}

}  // extern "C"
