"""The network-block operators at values near the ends of their types."""
import pytest

torch = pytest.importorskip("torch")
import block_ref as ref  # noqa: E402
from roundtrip_amd import _lib  # noqa: E402
from test_gpu_blocks import ACT, CODE, DT, KIND, norm_case, workspace  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("act", sorted(ACT))
def test_bits_do_not_depend_on_what_is_kept_nor_where(engine, act, dt):
    """The same out with nothing kept, with the gate and up kept, and with them kept at an odd place.  Of the 408000 values of h some 25
    would differ in float16 if one of these rounded h's product once and another twice."""
    T, d, f, dtype = 3000, 64, 136, DT[dt]
    gen = torch.Generator().manual_seed(8)
    x, wg, wu, wd = [(torch.randn(s, generator=gen) * k).to(dtype).cuda() for s, k in (((T, d), 1.0), ((d, f), 0.15), ((d, f), 0.125), ((f, d), 0.1))]
    got = []
    for shift in (None, 0, 1):
        out = torch.empty(T, d, dtype=dtype, device="cuda")
        pre = torch.empty(2, T * f + 4, device="cuda")
        at = [None if shift is None else p.data_ptr() + 4 * shift for p in pre]
        a = engine.gated_ffn_args(T, d, f, d, CODE[dt], ACT[act], x=x.data_ptr(), w_gate=wg.data_ptr(), w_up=wu.data_ptr(), w_down=wd.data_ptr(),
                                  out=out.data_ptr(), pre_gate=at[0], pre_up=at[1])
        n = engine.gated_ffn_workspace(a)
        ws = workspace(n)
        torch.cuda.synchronize()
        engine.gated_ffn_dev(a, ws.data_ptr(), n)
        engine.sync()
        got.append(out)
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("d", [512, 515])
def test_n_and_its_rest_of_many_values(engine, d, dt):
    """n + n_lo at two million values: one whose n was rounded otherwise than n_lo supposes would be off by a step of n."""
    norm_case(engine, 4096, d, dt, "rms", 0, branch=False, want_y=False, seed=d)


@pytest.mark.parametrize("act", sorted(ACT))
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_gradient_of_large_gates(engine, act, dt):
    """act'(g) for gates up to the type's end: with unit weights and ones for up and dout, dx is act'(g), rounded once in 16 bits
    (dg; the sum over k then adds zeros)."""
    dtype = DT[dt]
    g = torch.tensor([0.0, 1.0, -1.0, 6.0, -6.0, 30.0, -30.0, 70.0, -70.0, 1e4, -1e4, 8e12, -8e12, 1.9e19, -1.9e19, 3e38, -3e38])
    f = g.numel()
    T = 3
    eye, zero = torch.eye(f, dtype=dtype, device="cuda"), torch.zeros(f, f, dtype=dtype, device="cuda")
    x, dout, dx = (torch.ones(T, f, dtype=dtype, device="cuda") for _ in range(3))
    pg, pu = g.expand(T, f).contiguous().cuda(), torch.ones(T, f, device="cuda")
    a = engine.gated_ffn_args(T, f, f, f, CODE[dt], ACT[act], x=x.data_ptr(), w_gate=eye.data_ptr(), w_up=zero.data_ptr(), w_down=eye.data_ptr(),
                              out=x.data_ptr(), pre_gate=pg.data_ptr(), pre_up=pu.data_ptr(), alpha=0.25)
    n = engine.gated_ffn_workspace(a, backward=True)
    ws = workspace(n)
    torch.cuda.synchronize()
    engine.gated_ffn_backward_dev(a, engine.gated_ffn_grads(dout=dout.data_ptr(), dx=dx.data_ptr()), ws.data_ptr(), n)
    engine.sync()
    d = ref.act(act, g.double(), 0.25)[1].expand(T, f)
    # float32's: ref.ACT where exp's argument is up to 16 in size; at the tails of exp (30 and beyond) the derivative is below 1e-11 or
    # that near 1
    tail = (2 * ref.ACT[dtype] * (d.abs() + g.double().abs().clamp(max=16)) + 1e-11).expand(T, f)
    ref.check(dx, ref.rounded(d, tail, dtype), "dx")


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("dt,w", [("f16", 6e4), ("bf16", 3e38)])
def test_the_rest_of_an_infinite_value_is_zero(engine, dt, w, kind):
    """Normed rows beyond the type's range are infinite, and n_lo is zero there: n + n_lo, and a product with positive weights,
    are infinite and not NaN."""
    T, d, f = 40, 64, 72
    dtype = DT[dt]
    gen = torch.Generator().manual_seed(5)
    x = torch.randn(T, d, generator=gen).to(dtype)
    x64 = x.double()
    c = x64 - x64.mean(1, keepdim=True) if kind == "layer" else x64
    hat = c / (c.square().mean(1, keepdim=True) + 1e-5).sqrt()
    wp = torch.ones(d, dtype=dtype)
    wp[5] = w
    beyond = torch.zeros(T, d, dtype=torch.bool)
    beyond[:, 5] = hat[:, 5].abs() > 1.3                 # 1.3 w is beyond either type by more than the norm's error
    near = torch.zeros(T, d, dtype=torch.bool)
    near[:, 5] = (hat[:, 5].abs() > 1.0) & ~beyond[:, 5]
    assert 3 < int(beyond.sum()) < T - 3
    dev = [t.cuda() for t in (x, wp)]
    n, lo = torch.empty_like(dev[0]), torch.empty_like(dev[0])
    a = engine.block_norm_args(T, d, CODE[dt], KIND[kind], x=dev[0].data_ptr(), n=n.data_ptr(), n_lo=lo.data_ptr(), w_pre=dev[1].data_ptr(), eps=1e-5)
    torch.cuda.synchronize()
    engine.block_norm_dev(a)
    engine.sync()
    got, rest = n.cpu().double(), lo.cpu().double()
    assert torch.equal(got[beyond], torch.sign(hat[beyond]) * float("inf"))
    assert not rest[beyond].any()
    fine = ~beyond & ~near
    assert torch.isfinite(got[fine]).all() and torch.isfinite(rest[fine]).all()
    # the block behind it: positive weights, so that gate and up are +infinity where x is
    ones = [torch.full(s, 2.0 ** -4, dtype=dtype, device="cuda") for s in ((d, f), (d, f), (f, d))]
    out = torch.empty(T, d, dtype=dtype, device="cuda")
    b = engine.gated_ffn_args(T, d, f, d, CODE[dt], ACT["silu"], x=n.data_ptr(), x_lo=lo.data_ptr(), w_gate=ones[0].data_ptr(), w_up=ones[1].data_ptr(),
                              w_down=ones[2].data_ptr(), out=out.data_ptr())
    size = engine.gated_ffn_workspace(b)
    ws = workspace(size)
    torch.cuda.synchronize()
    engine.gated_ffn_dev(b, ws.data_ptr(), size)
    engine.sync()
    rows = beyond[:, 5] & (hat[:, 5] > 0)
    assert bool(rows.any()) and bool((out[rows.cuda()] == float("inf")).all())
