"""The network-block operators (rt_gated_ffn_*, rt_block_norm_*) against float64 with derived bounds (block_ref.py)."""
import pytest

torch = pytest.importorskip("torch")
import block_ref as ref  # noqa: E402
from roundtrip_amd import _lib  # noqa: E402

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CODE = {"f32": _lib.RT_F32, "bf16": _lib.RT_BF16, "f16": _lib.RT_F16}
ACT = {"silu": _lib.RT_ACT_SILU, "gelu": _lib.RT_ACT_GELU_TANH, "lrelu": _lib.RT_ACT_LRELU, "sigmoid": _lib.RT_ACT_SIGMOID}
KIND = {"rms": _lib.RT_NORM_RMS, "layer": _lib.RT_NORM_LAYER}
GUARD = 7.0                     # what lies around the arrays, and has to lie there afterwards


class Array(object):
    """rows x width of dtype on the GPU inside a larger buffer, `shift` elements from its start, `ld` elements a row."""

    def __init__(self, rows, width, dtype, ld=None, shift=0, value=None):
        self.ld, self.rows, self.width, self.shift = ld or width, rows, width, shift
        n = shift + rows * self.ld + 16
        self.buf = torch.full((n,), GUARD, dtype=dtype, device="cuda")
        self.view = self.buf[shift:shift + rows * self.ld].view(rows, self.ld)[:, :width]
        if value is not None:
            self.view.copy_(value)
        self.before = self.buf.clone()

    @property
    def ptr(self):
        return self.buf.data_ptr() + self.shift * self.buf.element_size()

    def untouched_outside(self):
        a, b = self.buf.clone(), self.before.clone()
        for t in (a, b):
            t[self.shift:self.shift + self.rows * self.ld].view(self.rows, self.ld)[:, :self.width] = 0
        return torch.equal(a, b)


def normal(gen, shape, dtype, scale=1.0, shift=0.0):
    """(the rounded values on the CPU, the same in float64)"""
    v = (torch.randn(shape, generator=gen, dtype=torch.float64) * scale + shift).to(dtype)
    return v, v.double()


def workspace(n):
    return torch.full((max(n, 16),), 0xA5, dtype=torch.uint8, device="cuda")


def ffn_case(engine, T, di, f, do, dt, act, lds=(0, 0, 0, 0, 0), shift=0, alpha=0.2, seed=0, lo=False):
    """Runs forward and backward and checks every output."""
    dtype, gen = DT[dt], torch.Generator().manual_seed(seed)
    x, x64 = normal(gen, (T, di), dtype)
    xl, xl64 = normal(gen, (T, di), dtype, 2.0 ** -9) if lo else (None, 0.0)
    wg, wg64 = normal(gen, (di, f), dtype, 1.5 * di ** -0.5)
    wu, wu64 = normal(gen, (di, f), dtype, di ** -0.5)
    wd, wd64 = normal(gen, (f, do), dtype, f ** -0.5)
    dout, dout64 = normal(gen, (T, do), dtype)
    ld = [w + l for w, l in zip((di, f, do, do, f), lds)]
    A = lambda r, w, l=None, v=None: Array(r, w, dtype, l, shift, v)  # noqa: E731
    ax, ag, au, ad = A(T, di, ld[0], x), A(di, f, ld[1], wg), A(di, f, ld[1], wu), A(f, do, ld[2], wd)
    ao, ado = A(T, do, ld[3]), A(T, do, ld[3], dout)
    al = A(T, di, ld[0], xl) if lo else None
    pg, pu = Array(T, f, torch.float32, ld[4], shift), Array(T, f, torch.float32, ld[4], shift)
    for keep in (False, True):
        a = engine.gated_ffn_args(T, di, f, do, CODE[dt], ACT[act], x=ax.ptr, w_gate=ag.ptr, w_up=au.ptr, w_down=ad.ptr,
                                  out=ao.ptr, pre_gate=pg.ptr if keep else None, pre_up=pu.ptr if keep else None, alpha=alpha, x_lo=al.ptr if lo else None,
                                  ldx=ld[0], ld_in=ld[1], ld_down=ld[2], ld_out=ld[3], ld_pre=ld[4])
        n = engine.gated_ffn_workspace(a)
        ws = workspace(n)
        torch.cuda.synchronize()
        engine.gated_ffn_dev(a, ws.data_ptr(), n)
        engine.sync()
        want = ref.ffn(x64 + xl64, wg64, wu64, wd64, act, alpha, dtype)
        ref.check(ao.view, want["out"], "out")
        if keep:
            ref.check(pg.view, want["pre_gate"], "pre_gate")
            ref.check(pu.view, want["pre_up"], "pre_up")
        else:
            assert torch.equal(pg.buf, pg.before)
            first = ao.view.clone()
        for arr in (ax, ag, au, ad, ao, pg, pu):
            assert arr.untouched_outside()
    assert torch.equal(first, ao.view)                   # keeping the gate and up changes nothing
    # backward, at values of pre_gate and pre_up of its own
    g, g64 = normal(gen, (T, f), torch.float32, 1.5)
    u, u64 = normal(gen, (T, f), torch.float32)
    pg.view.copy_(g)
    pu.view.copy_(u)
    dx, dg, du, dd = A(T, di, ld[0]), A(di, f, ld[1]), A(di, f, ld[1]), A(f, do, ld[2])
    r = engine.gated_ffn_grads(dout=ado.ptr, dx=dx.ptr, dw_gate=dg.ptr, dw_up=du.ptr, dw_down=dd.ptr, ld_dout=ld[3], ld_dx=ld[0],
                               ld_dw_in=ld[1], ld_dw_down=ld[2])
    n = engine.gated_ffn_workspace(a, backward=True)
    ws = workspace(n)
    torch.cuda.synchronize()
    engine.gated_ffn_backward_dev(a, r, ws.data_ptr(), n)
    engine.sync()
    want = ref.ffn_back(x64, wg64, wu64, wd64, g64, u64, dout64, act, alpha, dtype)
    got = {"dx": dx, "dw_gate": dg, "dw_up": du, "dw_down": dd}
    for k, arr in got.items():
        ref.check(arr.view, want[k], k)
        assert arr.untouched_outside(), k
    # each gradient alone is the same
    for k, arr in got.items():
        again = A(arr.rows, arr.width, arr.ld)
        one = engine.gated_ffn_grads(dout=ado.ptr, ld_dout=ld[3], ld_dx=ld[0], ld_dw_in=ld[1], ld_dw_down=ld[2], **{k: again.ptr})
        torch.cuda.synchronize()
        engine.gated_ffn_backward_dev(a, one, ws.data_ptr(), n)
        engine.sync()
        assert torch.equal(again.view, arr.view), k


SIZES = [(1, 1, 1, 1), (1, 64, 128, 64), (2, 2, 512, 3), (3, 7, 5, 9), (17, 128, 256, 128), (33, 100, 72, 40), (64, 64, 64, 64),
         (65, 130, 96, 66), (129, 72, 136, 200), (130, 33, 257, 31), (300, 512, 64, 512), (1000, 24, 48, 16)]


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_gated_ffn(engine, size, dt):
    act = list(ACT)[sum(size) % 4]
    ffn_case(engine, *size, dt, act)


@pytest.mark.parametrize("act", sorted(ACT))
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_gated_ffn_activations(engine, act, dt):
    ffn_case(engine, 40, 64, 192, 32, dt, act, alpha=0.1, seed=3)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("lds,shift", [((8, 8, 8, 8, 8), 0), ((8, 16, 24, 32, 40), 8), ((1, 3, 5, 7, 9), 0), ((0, 0, 0, 0, 0), 1),
                                       ((4, 4, 4, 4, 4), 2)])
def test_gated_ffn_strides_and_alignment(engine, dt, lds, shift):
    ffn_case(engine, 70, 64, 128, 96, dt, "silu", lds, shift, seed=5)
    ffn_case(engine, 5, 64, 128, 96, dt, "gelu", lds, shift, seed=6)


@pytest.mark.parametrize("dt", ["bf16", "f32", "f16"])
@pytest.mark.parametrize("size,lds,shift", [((1030, 101, 203, 77), (0, 0, 0, 0, 0), 0), ((1100, 36, 1001, 52), (0, 0, 0, 0, 0), 0),
                                            ((1024, 64, 132, 33), (0, 0, 0, 0, 0), 0), ((1025, 43, 64, 65), (3, 1, 2, 5, 7), 1),
                                            ((1500, 130, 66, 128), (6, 6, 0, 8, 2), 0), ((1100, 130, 211, 33), (1, 0, 0, 0, 0), 0), ((2050, 7, 5, 3), (0, 0, 0, 0, 0), 0)])
def test_gated_ffn_odd_widths_of_many_rows(engine, size, lds, shift, dt):
    """Operands that are copied with zeros behind their rows, beside ones that are not."""
    ffn_case(engine, *size, dt, "sigmoid", lds, shift, seed=15, lo=dt != "f32")


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("size", [(1, 64, 128, 64), (2, 70, 256, 8), (3, 2000, 96, 5), (16, 128, 256, 128), (31, 72, 104, 40), (100, 130, 96, 66), (300, 512, 512, 64),
                                  (7, 33, 57, 31), (4100, 72, 4104, 16)], ids=lambda s: "x".join(map(str, s)))
def test_gated_ffn_with_the_rest_of_x(engine, size, dt):
    """x_lo: the gate's and up's sums are those of x + x_lo."""
    ffn_case(engine, *size, dt, "lrelu", seed=14, lo=True)


@pytest.mark.parametrize("dt", ["bf16", "f32", "f16"])
@pytest.mark.parametrize("size", [(1, 1501, 6293, 1502), (2, 70, 4, 5), (3, 35, 67, 131), (9, 100, 1023, 66), (32, 257, 5, 4), (4, 3000, 1030, 7)],
                         ids=lambda s: "x".join(map(str, s)))
def test_gated_ffn_few_rows_of_odd_widths(engine, size, dt):
    ffn_case(engine, *size, dt, "gelu", seed=16)
    ffn_case(engine, *size, dt, "gelu", (1, 3, 5, 7, 9), 1, seed=17)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_gated_ffn_long_sums(engine, dt):
    """Few columns under long sums: products whose K is split."""
    ffn_case(engine, 2100, 64, 72, 8, dt, "silu", seed=7)
    ffn_case(engine, 4, 2000, 1600, 40, dt, "lrelu", seed=8)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("size", [(4100, 72, 4104, 72), (4100, 4104, 40, 4104), (40, 4104, 2056, 4104)], ids=lambda s: "x".join(map(str, s)))
def test_gated_ffn_many_tiles(engine, size, dt):
    """Results large enough for the largest tiles, ragged at every edge, under short sums."""
    ffn_case(engine, *size, dt, "silu", seed=13)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_gated_ffn_without_tokens(engine, dt):
    dtype = DT[dt]
    w = [Array(12, 20, dtype, value=1.0), Array(12, 20, dtype, value=1.0), Array(20, 12, dtype, value=1.0)]
    a = engine.gated_ffn_args(0, 12, 20, 12, CODE[dt], ACT["silu"], w_gate=w[0].ptr, w_up=w[1].ptr, w_down=w[2].ptr)
    assert engine.gated_ffn_workspace(a) == 0 and engine.gated_ffn_workspace(a, True) == 0
    engine.gated_ffn_dev(a)
    d = [Array(12, 20, dtype, 24), Array(12, 20, dtype, 24), Array(20, 12, dtype, 13)]
    torch.cuda.synchronize()
    engine.gated_ffn_backward_dev(a, engine.gated_ffn_grads(dw_gate=d[0].ptr, dw_up=d[1].ptr, dw_down=d[2].ptr, ld_dw_in=24, ld_dw_down=13))
    engine.sync()
    for t in d:
        assert not t.view.any() and t.untouched_outside()


def test_gated_ffn_weights_side_by_side(engine):
    """Gate and up as the two halves of one [d, 2 f] array, and their gradients likewise."""
    di, f, T, dtype = 64, 128, 20, torch.bfloat16
    gen = torch.Generator().manual_seed(9)
    x, x64 = normal(gen, (T, di), dtype)
    w, w64 = normal(gen, (di, 2 * f), dtype, 0.1)
    wd, wd64 = normal(gen, (f, di), dtype, 0.1)
    xd, wc, wdd = x.cuda(), w.cuda(), wd.cuda()
    out = torch.empty(T, di, dtype=dtype, device="cuda")
    pre = torch.empty(T, 2 * f, device="cuda")
    a = engine.gated_ffn_args(T, di, f, di, CODE["bf16"], ACT["silu"], x=xd.data_ptr(), w_gate=wc.data_ptr(), w_up=wc.data_ptr() + 2 * f,
                              w_down=wdd.data_ptr(), out=out.data_ptr(), pre_gate=pre.data_ptr(), pre_up=pre.data_ptr() + 4 * f,
                              ld_in=2 * f, ld_pre=2 * f)
    n = max(engine.gated_ffn_workspace(a), engine.gated_ffn_workspace(a, True))
    ws = workspace(n)
    dw = torch.empty_like(wc)
    r = engine.gated_ffn_grads(dout=xd.data_ptr(), dw_gate=dw.data_ptr(), dw_up=dw.data_ptr() + 2 * f, ld_dw_in=2 * f)
    torch.cuda.synchronize()
    engine.gated_ffn_dev(a, ws.data_ptr(), n)
    engine.gated_ffn_backward_dev(a, r, ws.data_ptr(), n)
    engine.sync()
    want = ref.ffn(x64, w64[:, :f], w64[:, f:], wd64, "silu", 0.2, dtype)
    ref.check(out, want["out"], "out")
    p = pre.cpu().double()
    back = ref.ffn_back(x64, w64[:, :f], w64[:, f:], wd64, p[:, :f], p[:, f:], x64, "silu", 0.2, dtype)
    ref.check(dw[:, :f], back["dw_gate"], "dw_gate")
    ref.check(dw[:, f:], back["dw_up"], "dw_up")


@pytest.mark.parametrize("act", sorted(ACT))
def test_gated_ffn_gradient_by_differences(engine, act):
    """The backward pass against differences of the forward pass, along random directions (float32)."""
    T, d, f = 6, 10, 14
    gen = torch.Generator().manual_seed(11)
    v = {"x": torch.randn(T, d, generator=gen), "w_gate": torch.randn(d, f, generator=gen) * 0.4,
         "w_up": torch.randn(d, f, generator=gen) * 0.4, "w_down": torch.randn(f, d, generator=gen) * 0.4}
    if act == "lrelu":      # away from the kink: no |gate| below the step's reach
        g = v["x"] @ v["w_gate"]
        assert float(g.abs().min()) > 1e-4
    dout = torch.randn(T, d, generator=gen)
    dev = {k: t.cuda() for k, t in v.items()}
    out, pg, pu = (torch.empty(s, device="cuda") for s in ((T, d), (T, f), (T, f)))

    def forward(t):
        a = engine.gated_ffn_args(T, d, f, d, _lib.RT_F32, ACT[act], out=out.data_ptr(), pre_gate=pg.data_ptr(), pre_up=pu.data_ptr(),
                                  **{k: x.data_ptr() for k, x in t.items()})
        n = engine.gated_ffn_workspace(a)
        ws = workspace(n)
        torch.cuda.synchronize()
        engine.gated_ffn_dev(a, ws.data_ptr(), n)
        engine.sync()
        return a, float((out.cpu().double() * dout.double()).sum())

    a, _ = forward(dev)
    grads = {k: torch.empty_like(t) for k, t in dev.items()}
    dd = dout.cuda()
    r = engine.gated_ffn_grads(dout=dd.data_ptr(), dx=grads["x"].data_ptr(), **{"d" + k: t.data_ptr() for k, t in grads.items() if k != "x"})
    n = engine.gated_ffn_workspace(a, True)
    ws = workspace(n)
    torch.cuda.synchronize()
    engine.gated_ffn_backward_dev(a, r, ws.data_ptr(), n)
    engine.sync()
    # central differences: step 2^-6 for the smooth gates; their third derivatives are below 4 along directions of length 1,
    # so the cut-off error is below 4 step^2 / 6 * |dout| |x| |w|.. < 0.01; the float32 forward pass (60 values of size < 4,
    # each off by < 2^-20) adds < 60 * 4 * 2^-20 / step = 0.015.  The leaky gate is piecewise cubic: a smaller step that
    # stays on its side.
    step = 2.0 ** -6
    for k in dev:
        way = torch.randn(v[k].shape, generator=gen)
        way /= way.norm()
        if act == "lrelu" and k in ("x", "w_gate"):
            move = (way @ v["w_gate"]) if k == "x" else (v["x"] @ way)
            g = v["x"] @ v["w_gate"]
            # directions that would cross the kink are made zero for the rows concerned by shrinking the whole direction
            while bool((move.abs() * step >= g.abs()).any()):
                way, move = way / 2, move / 2
        up, down = dict(dev), dict(dev)
        up[k], down[k] = (v[k] + step * way).cuda(), (v[k] - step * way).cuda()
        diff = (forward(up)[1] - forward(down)[1]) / (2 * step)
        got = float((grads[k].cpu().double() * way.double()).sum())
        assert abs(got - diff) < 0.03, (k, got, diff)


# ---- norms -------------------------------------------------------------------------------------------------------------------
def norm_case(engine, T, d, dt, kind, rpg, branch=True, post=True, pre=True, rs=0.9, bs=0.7, off=0.0, lds=(0, 0, 0, 0, 0), shift=0,
              eps=1e-5, seed=0, want_y=True, want_n=True, mean=0.5):
    """rpg 0: no gate."""
    dtype, gen = DT[dt], torch.Generator().manual_seed(seed)
    x, x64 = normal(gen, (T, d), dtype, 1.0, mean)
    b, b64 = normal(gen, (T, d), dtype, 2.0, mean) if branch else (None, None)
    G = -(-T // rpg) if rpg else 0
    gate, gate64 = normal(gen, (G, d), dtype, 0.7) if rpg else (None, None)
    wpo, wpo64 = normal(gen, (1, d), dtype, 0.2, 1.0 - off) if post and branch else (None, None)
    wpr, wpr64 = normal(gen, (1, d), dtype, 0.2, 1.0 - off) if pre else (None, None)
    ld = [d + k for k in lds]
    A = lambda r, l=None, v=None: Array(r, d, dtype, l, shift, v)  # noqa: E731
    ptr = lambda a: None if a is None else a.ptr  # noqa: E731
    opt = lambda r, l, v: None if v is None else A(r, l, v)  # noqa: E731
    ax, ab, ag = A(T, ld[0], x), opt(T, ld[1], b), opt(G, ld[4], gate)
    aw, av = opt(1, d, wpo), opt(1, d, wpr)
    y, n = A(T, ld[2]) if want_y else None, A(T, ld[3]) if want_n else None
    nl = A(T, ld[3]) if want_n and dt != "f32" else None
    a = engine.block_norm_args(T, d, CODE[dt], KIND[kind], x=ax.ptr, branch=ptr(ab), y=ptr(y), n=ptr(n), n_lo=ptr(nl), w_post=ptr(aw), w_pre=ptr(av),
                               gate=ptr(ag), rows_per_gate=rpg, res_scale=rs, branch_scale=bs, eps=eps, w_offset=off, ldx=ld[0],
                               ld_branch=ld[1], ldy=ld[2], ldn=ld[3], ld_gate=ld[4])
    torch.cuda.synchronize()
    engine.block_norm_dev(a)
    engine.sync()
    flat = lambda w: None if w is None else w[0]  # noqa: E731
    want = ref.norm(x64, b64, gate64, rpg, flat(wpo64), flat(wpr64), kind, eps, rs, bs, off, dtype)
    for k, arr in (("y", y), ("n", n)):
        if arr is not None:
            ref.check(arr.view, want[k], k)
            assert arr.untouched_outside(), k
    if nl is not None:
        ref.check(n.view.double() + nl.view.double(), want["n_and_lo"], "n + n_lo")
        assert nl.untouched_outside()
        plain = A(T, ld[3])                       # without it n is the same
        a.n, a.n_lo = plain.ptr, None
        if y is not None:
            a.y = None
        torch.cuda.synchronize()
        engine.block_norm_dev(a)
        engine.sync()
        assert torch.equal(plain.view, n.view)
        a.y = ptr(y)
    # backward, at a y of its own
    dy, dy64 = normal(gen, (T, d), dtype) if want_y else (None, None)
    dn, dn64 = normal(gen, (T, d), dtype) if want_n else (None, None)
    if y is not None:
        y_in, y64 = normal(gen, (T, d), dtype, 1.0, mean)
        y.view.copy_(y_in)
    else:
        y64 = rs * x64
        if branch:
            return
    ady, adn = opt(T, ld[0], dy), opt(T, ld[1], dn)
    got = {"dx": A(T, ld[2])}
    if branch:
        got.update(dbranch=A(T, ld[3]), dw_post=A(1))
        if rpg:
            got["dgate"] = A(G, ld[4])
    if want_n:
        got["dw_pre"] = A(1)
    r = engine.block_norm_grads(dy=ptr(ady), dn=ptr(adn), ld_dy=ld[0], ld_dn=ld[1], ld_dx=ld[2], ld_dbranch=ld[3], ld_dgate=ld[4],
                                **{k: v.ptr for k, v in got.items()})
    size = engine.block_norm_workspace(a)
    ws = workspace(size)
    torch.cuda.synchronize()
    engine.block_norm_backward_dev(a, r, ws.data_ptr(), size)
    engine.sync()
    want = ref.norm_back(y64, b64, gate64, rpg or T, flat(wpo64), flat(wpr64), dy64, dn64, kind, eps, rs, bs, off, dtype)
    for k, arr in got.items():
        ref.check(arr.view if arr.rows > 1 or want[k][0].dim() == 2 else arr.view[0], want[k], k)
        assert arr.untouched_outside(), k
    for k, arr in got.items():                    # each alone is the same
        again = Array(arr.rows, d, dtype, arr.ld, shift)
        one = engine.block_norm_grads(dy=ptr(ady), dn=ptr(adn), ld_dy=ld[0], ld_dn=ld[1], ld_dx=ld[2], ld_dbranch=ld[3], ld_dgate=ld[4],
                                      **{k: again.ptr})
        torch.cuda.synchronize()
        engine.block_norm_backward_dev(a, one, ws.data_ptr(), size)
        engine.sync()
        assert torch.equal(again.view, arr.view), k


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("T,d,rpg", [(1, 1, 1), (1, 8, 0), (2, 2, 1), (5, 33, 2), (7, 64, 7), (9, 512, 4), (3, 520, 1), (130, 90, 50), (11, 1000, 3),
                                     (4, 1024, 0), (6, 2047, 5), (3, 2056, 2), (3, 4096, 3), (2, 8192, 1), (2, 8200, 2), (2, 16384, 1)])
def test_block_norm(engine, T, d, rpg, kind, dt):
    norm_case(engine, T, d, dt, kind, rpg, seed=T + d)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_block_norm_widest(engine, dt):
    norm_case(engine, 2, 32768, dt, "layer", 1)
    norm_case(engine, 3, 32761, dt, "rms", 2)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("rpg", [0, 1, 3, 9, 1000, 4096, 6000, 12289])
def test_block_norm_many_rows(engine, dt, rpg):
    """Several rows for each unit of the backward pass; gates whose rows one unit sees, and gates that it shares."""
    norm_case(engine, 12289, 24, dt, "rms", rpg, seed=rpg)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("rpg", [2, 700, 2500])
def test_block_norm_many_rows_of_a_workgroup(engine, dt, rpg):
    norm_case(engine, 2500, 2200, dt, "layer", rpg, seed=rpg)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("lds,shift", [((8, 8, 8, 8, 8), 8), ((1, 2, 3, 4, 5), 0), ((0, 0, 0, 0, 0), 1), ((16, 0, 8, 24, 32), 0)])
def test_block_norm_strides_and_alignment(engine, dt, lds, shift):
    norm_case(engine, 21, 200, dt, "rms", 4, lds=lds, shift=shift)
    norm_case(engine, 4, 2304, dt, "layer", 3, lds=lds, shift=shift)


@pytest.mark.parametrize("branch,post,pre,rpg,want_y,want_n,rs,off", [
    (False, False, True, 0, False, True, 1.0, 0.0), (False, False, True, 0, False, True, 0.5, 1.0), (False, False, False, 0, True, True, 1.5, 0.0),
    (True, False, False, 0, True, True, 1.0, 0.0), (True, True, True, 3, True, False, 1.0, 1.0), (True, True, True, 2, False, True, 0.0, 0.0),
    (True, False, True, 13, True, True, -1.0, 0.5)])
def test_block_norm_parts(engine, branch, post, pre, rpg, want_y, want_n, rs, off):
    for dt in ("f32", "bf16"):
        norm_case(engine, 13, 72, dt, "rms", rpg, branch, post, pre, rs, 0.8, off, want_y=want_y, want_n=want_n, seed=2)


def test_block_norm_rows_of_zeros(engine):
    """A row of zeros is normed to zeros; its gradient has the factor 1 / sqrt(eps)."""
    T, d, eps = 4, 40, 1e-3
    x = torch.zeros(T, d, device="cuda")
    x[2] = 1.0
    n, dn, dx = torch.empty_like(x), torch.ones_like(x), torch.empty_like(x)
    a = engine.block_norm_args(T, d, _lib.RT_F32, KIND["rms"], x=x.data_ptr(), n=n.data_ptr(), eps=eps)
    size = engine.block_norm_workspace(a)
    ws = workspace(size)
    torch.cuda.synchronize()
    engine.block_norm_dev(a)
    engine.block_norm_backward_dev(a, engine.block_norm_grads(dn=dn.data_ptr(), dx=dx.data_ptr()), ws.data_ptr(), size)
    engine.sync()
    assert not n[[0, 1, 3]].any()
    assert torch.allclose(dx[[0, 1, 3]], torch.full_like(dx[:3], eps ** -0.5), rtol=1e-5)


def test_block_norm_in_place(engine):
    """y in x's memory and n in branch's; dx in dy's and dbranch in branch's: the same bits as apart."""
    T, d, dtype = 37, 264, torch.bfloat16
    gen = torch.Generator().manual_seed(4)
    t = {k: normal(gen, (T, d), dtype)[0].cuda() for k in ("x", "branch", "dy", "dn")}
    w = normal(gen, (d,), dtype, 0.1, 1.0)[0].cuda()
    o = {k: torch.empty_like(t["x"]) for k in ("y", "n", "dx", "dbranch")}
    kw = dict(w_post=w.data_ptr(), w_pre=w.data_ptr())
    a = engine.block_norm_args(T, d, CODE["bf16"], KIND["rms"], x=t["x"].data_ptr(), branch=t["branch"].data_ptr(), y=o["y"].data_ptr(),
                               n=o["n"].data_ptr(), **kw)
    size = engine.block_norm_workspace(a)
    ws = workspace(size)
    torch.cuda.synchronize()
    engine.block_norm_dev(a)
    engine.block_norm_backward_dev(a, engine.block_norm_grads(dy=t["dy"].data_ptr(), dn=t["dn"].data_ptr(), dx=o["dx"].data_ptr(),
                                                              dbranch=o["dbranch"].data_ptr()), ws.data_ptr(), size)
    engine.sync()
    x2, b2, b3 = t["x"].clone(), t["branch"].clone(), t["branch"].clone()
    a2 = engine.block_norm_args(T, d, CODE["bf16"], KIND["rms"], x=x2.data_ptr(), branch=b2.data_ptr(), y=x2.data_ptr(), n=b2.data_ptr(), **kw)
    torch.cuda.synchronize()
    engine.block_norm_dev(a2)
    engine.sync()
    assert torch.equal(x2, o["y"]) and torch.equal(b2, o["n"])
    a2.branch = b3.data_ptr()
    torch.cuda.synchronize()
    engine.block_norm_backward_dev(a2, engine.block_norm_grads(dy=t["dy"].data_ptr(), dn=t["dn"].data_ptr(), dx=t["dy"].data_ptr(),
                                                               dbranch=b3.data_ptr()), ws.data_ptr(), size)
    engine.sync()
    assert torch.equal(t["dy"], o["dx"]) and torch.equal(b3, o["dbranch"])


# ---- together ----------------------------------------------------------------------------------------------------------------
class Block(object):
    """norm - gated feed-forward - norm with gate and residual, and back, as a program keeps it."""

    def __init__(self, engine, T, d, f, dt, seed=0):
        self.eng, self.dtype = engine, DT[dt]
        gen = torch.Generator().manual_seed(seed)
        new = lambda *s: torch.empty(s, dtype=self.dtype, device="cuda")  # noqa: E731
        self.host = {"x": normal(gen, (T, d), self.dtype), "w_in": normal(gen, (d,), self.dtype, 0.1, 1.0),
                     "w_gate": normal(gen, (d, f), self.dtype, d ** -0.5), "w_up": normal(gen, (d, f), self.dtype, d ** -0.5),
                     "w_down": normal(gen, (f, d), self.dtype, f ** -0.5), "w_post": normal(gen, (d,), self.dtype, 0.1, 1.0),
                     "w_pre": normal(gen, (d,), self.dtype, 0.1, 1.0), "gate": normal(gen, (-(-T // 3), d), self.dtype, 0.5),
                     "dy": normal(gen, (T, d), self.dtype), "dn": normal(gen, (T, d), self.dtype)}
        t = self.t = {k: v[0].cuda() for k, v in self.host.items()}
        t.update(h=new(T, d), b=new(T, d), y=new(T, d), n=new(T, d), pg=torch.empty(T, f, device="cuda"), pu=torch.empty(T, f, device="cuda"), dx=new(T, d), db=new(T, d), dh=new(T, d))
        for k in ("w_in", "w_gate", "w_up", "w_down", "w_post", "w_pre", "gate"):
            t["d" + k] = torch.empty_like(t[k])
        p = {k: v.data_ptr() for k, v in t.items()}
        code = CODE[dt]
        p["lo"] = None
        if dt != "f32":
            t["lo"] = new(T, d)
            p["lo"] = t["lo"].data_ptr()
        self.before = engine.block_norm_args(T, d, code, KIND["rms"], x=p["x"], n=p["h"], n_lo=p["lo"], w_pre=p["w_in"])
        self.ffn = engine.gated_ffn_args(T, d, f, d, code, ACT["silu"], x=p["h"], x_lo=p["lo"], w_gate=p["w_gate"], w_up=p["w_up"], w_down=p["w_down"],
                                         out=p["b"], pre_gate=p["pg"], pre_up=p["pu"])
        self.after = engine.block_norm_args(T, d, code, KIND["rms"], x=p["x"], branch=p["b"], y=p["y"], n=p["n"], w_post=p["w_post"],
                                            w_pre=p["w_pre"], gate=p["gate"], rows_per_gate=3)
        self.g_after = engine.block_norm_grads(dy=p["dy"], dn=p["dn"], dx=p["dx"], dbranch=p["db"], dgate=p["dgate"], dw_post=p["dw_post"],
                                               dw_pre=p["dw_pre"])
        self.g_ffn = engine.gated_ffn_grads(dout=p["db"], dx=p["dh"], dw_gate=p["dw_gate"], dw_up=p["dw_up"], dw_down=p["dw_down"])
        self.g_before = engine.block_norm_grads(dy=p["dx"], dn=p["dh"], dx=p["dx"], dw_pre=p["dw_in"])
        self.size = max(engine.gated_ffn_workspace(self.ffn), engine.gated_ffn_workspace(self.ffn, True), engine.block_norm_workspace(self.after),
                        engine.block_norm_workspace(self.before))
        self.ws = workspace(self.size)
        torch.cuda.synchronize()

    def run(self):
        e, ws, n = self.eng, self.ws.data_ptr(), self.size
        e.block_norm_dev(self.before)
        e.gated_ffn_dev(self.ffn, ws, n)
        e.block_norm_dev(self.after)
        e.block_norm_backward_dev(self.after, self.g_after, ws, n)
        e.gated_ffn_backward_dev(self.ffn, self.g_ffn, ws, n)
        e.block_norm_backward_dev(self.before, self.g_before, ws, n)

    def outputs(self):
        return {k: self.t[k].clone() for k in ("y", "n", "dx", "dgate", "dw_in", "dw_gate", "dw_up", "dw_down", "dw_post", "dw_pre")}


def exact_block(host):
    """The block in float64, its gradients by differentiation."""
    v = {k: t[1].clone().requires_grad_(k not in ("dy", "dn")) for k, t in host.items()}
    nrm = lambda a, w: a / torch.sqrt(a.pow(2).mean(1, keepdim=True) + 1e-5) * w  # noqa: E731
    h = nrm(v["x"], v["w_in"])
    b = (torch.nn.functional.silu(h @ v["w_gate"]) * (h @ v["w_up"])) @ v["w_down"]
    T = v["x"].shape[0]
    y = v["x"] + v["gate"].repeat_interleave(3, 0)[:T] * nrm(b, v["w_post"])
    n = nrm(y, v["w_pre"])
    names = [k for k in v if k not in ("dy", "dn")]
    out = dict(zip(["dx" if k == "x" else "d" + k for k in names], torch.autograd.grad([y, n], [v[k] for k in names], [v["dy"], v["dn"]])))
    out.update(y=y.detach(), n=n.detach())
    return out


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("T,d,f", [(1, 64, 128), (50, 128, 320), (200, 90, 170)])
def test_block_together(engine, T, d, f, dt):
    """Forward and backward in a row against float64.  Between two operators a value is rounded once: nine roundings lie on
    the longest way at most (the norm's h, the product's h, b, y; then db, dg, du, dh, the result), each off by at most u of its size and
    nearly independent from element to element, so each moves a result by at most about u of its root mean square; norms and
    activations stretch a relative error by less than 2 here, hence 2 * 9 u in that measure."""
    blk = Block(engine, T, d, f, dt)
    blk.run()
    engine.sync()
    want = exact_block(blk.host)
    u = torch.finfo(DT[dt]).eps / 2
    for k, v in blk.outputs().items():
        off = float((v.cpu().double() - want[k]).norm() / want[k].norm())
        assert off < 18 * u, (k, off / u)


def test_block_captured_and_replayed(engine):
    """Two blocks' steps in two graphs on the engine's stream; replays give the eager bits, with eager work between them."""
    stream = torch.cuda.ExternalStream(engine.stream)
    blocks = [Block(engine, 33, 128, 256, "bf16", seed=1), Block(engine, 7, 96, 130, "f32", seed=2)]
    want, graphs = [], []
    for b in blocks:
        b.run()
        engine.sync()
        want.append(b.outputs())
    for b in blocks:
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=stream):
            b.run()
        graphs.append(g)
    for turn in range(4):
        for b, g, w in zip(blocks, graphs, want):
            for k in w:
                b.t[k].fill_(3.0)
            b.ws.fill_(turn)
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                g.replay()
            torch.cuda.synchronize()
            got = b.outputs()
            for k in w:
                assert torch.equal(got[k], w[k]), (turn, k)
        blocks[turn % 2].run()
        engine.sync()


def test_block_repeats_its_bits_and_two_engines_agree(engine):
    other = _lib.Engine(0)
    try:
        a, b = Block(engine, 400, 256, 512, "bf16", seed=3), Block(other, 400, 256, 512, "bf16", seed=3)
        a.run()
        b.run()                           # at the same time, on two streams
        engine.sync()
        other.sync()
        first = a.outputs()
        for k, v in b.outputs().items():
            assert torch.equal(v, first[k]), k
        a.run()
        engine.sync()
        for k, v in a.outputs().items():
            assert torch.equal(v, first[k]), k
    finally:
        other.close()


def test_block_leaves_the_current_device(engine):
    torch.cuda.set_device(0)
    Block(engine, 3, 16, 16, "f32").run()
    engine.sync()
    assert torch.cuda.current_device() == 0


def test_gated_ffn_far_offsets(engine):
    """Rows whose byte offsets pass 2^32 (a wide stride): the last ones are as right as the first."""
    T, d, f, ld, dtype = 2304, 64, 64, 1 << 20, torch.bfloat16
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GiB of free device memory")
    gen = torch.Generator().manual_seed(12)
    x, x64 = normal(gen, (T, d), dtype)
    w = [normal(gen, s, dtype, 0.125) for s in ((d, f), (d, f), (f, d))]
    big = torch.empty(T * ld, dtype=dtype, device="cuda")             # 4.8 GB: x in columns 0.., out in columns d..
    view = big.view(T, ld)
    view[:, :d].copy_(x)
    dev = [v[0].cuda() for v in w]
    a = engine.gated_ffn_args(T, d, f, d, CODE["bf16"], ACT["silu"], x=big.data_ptr(), w_gate=dev[0].data_ptr(), w_up=dev[1].data_ptr(),
                              w_down=dev[2].data_ptr(), out=big.data_ptr() + 2 * d, ldx=ld, ld_out=ld)
    n = engine.gated_ffn_workspace(a)
    ws = workspace(n)
    torch.cuda.synchronize()
    engine.gated_ffn_dev(a, ws.data_ptr(), n)
    engine.sync()
    ref.check(view[:, d:2 * d], ref.ffn(x64, w[0][1], w[1][1], w[2][1], "silu", 0.2, dtype)["out"], "out")


def test_block_norm_without_tokens(engine):
    d = 50
    w = [Array(1, d, torch.bfloat16) for _ in range(2)]
    a = engine.block_norm_args(0, d, CODE["bf16"], KIND["rms"], x=w[0].ptr, branch=w[0].ptr, y=w[0].ptr, n=w[0].ptr)
    engine.block_norm_dev(a)
    torch.cuda.synchronize()
    engine.block_norm_backward_dev(a, engine.block_norm_grads(dy=w[0].ptr, dn=w[0].ptr, dw_post=w[0].ptr, dw_pre=w[1].ptr))
    engine.sync()
    for t in w:
        assert not t.view.any() and t.untouched_outside()


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_gated_ffn_infinities_stay_in_their_rows(engine, dt):
    """Positive weights: an infinite x makes an infinite output row, with and without operands padded by zeros."""
    T, di, f, do = 1030, 13, 21, 11
    gen = torch.Generator().manual_seed(3)
    x = (torch.rand((T, di), generator=gen) + 0.5).to(DT[dt])
    x[7, 4] = float("inf")
    w = [(torch.rand(s, generator=gen) + 0.5).to(DT[dt]) for s in ((di, f), (di, f), (f, do))]
    want = ref.ffn(x.double(), w[0].double(), w[1].double(), w[2].double(), "silu", 0.0, DT[dt])
    rows = [r for r in range(T) if r != 7]
    ax, ag, au, ad = [Array(t.shape[0], t.shape[1], DT[dt], None, 0, t) for t in [x] + w]
    for n_rows in (T, 20):
        ao = Array(n_rows, do, DT[dt])
        a = engine.gated_ffn_args(n_rows, di, f, do, CODE[dt], ACT["silu"], x=ax.ptr, w_gate=ag.ptr, w_up=au.ptr, w_down=ad.ptr, out=ao.ptr)
        n = engine.gated_ffn_workspace(a)
        ws = workspace(n)
        torch.cuda.synchronize()
        engine.gated_ffn_dev(a, ws.data_ptr(), n)
        engine.sync()
        assert bool((ao.view[7] == float("inf")).all())
        keep = [r for r in rows if r < n_rows]
        out = want["out"]
        ref.check(ao.view[keep], tuple(t[keep] for t in out), "out")


@pytest.mark.parametrize("T,d", [((1 << 26) + 5, 8), ((1 << 21) * 4 + 3, 520)])
def test_block_norm_of_more_rows_than_one_row_of_workgroups(engine, T, d):
    x = torch.empty((T, d), dtype=torch.bfloat16, device="cuda")
    x.random_(-4, 5, generator=torch.Generator(device="cuda").manual_seed(2))
    n = torch.full_like(x, GUARD)
    a = engine.block_norm_args(T, d, _lib.RT_BF16, _lib.RT_NORM_RMS, x=x.data_ptr(), n=n.data_ptr(), eps=0.25)
    torch.cuda.synchronize()
    engine.block_norm_dev(a)
    engine.sync()
    for r0 in (0, (1 << 23) - 50, T // 2, T - 100):
        v = x[r0:r0 + 100].double()
        want = v / (v.square().mean(1, keepdim=True) + 0.25).sqrt()
        # half a step of bf16, and some float32 roundings
        assert bool(((n[r0:r0 + 100].double() - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -20)).all())
