"""The gate and up kept in the call's own 16-bit type: forward they are the float32 ones rounded once, backward they count as their values."""
import pytest

torch = pytest.importorskip("torch")
from test_gpu_blocks import ACT, Array, CODE, DT, normal, workspace  # noqa: E402

pytestmark = pytest.mark.gpu

# few rows (vector and matrix units, K split), tiles of 64, 128 and 256, with K in one run and in several, odd widths, copies of them
SIZES = [(1, 64, 128, 64), (3, 2000, 96, 5), (17, 3000, 260, 128), (33, 100, 72, 40), (300, 512, 65, 31), (67, 528, 1344, 48), (1030, 101, 203, 77),
         (3397, 136, 1168, 40), (130, 3488, 2056, 456), (4033, 45, 2184, 140), (1000, 40, 2051, 1200), (931, 55, 2479, 145)]


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("more,shift", [(0, 0), (3, 1)])
def test_kept_in_sixteen_bits(engine, size, dt, more, shift):
    T, di, f, do = size
    dtype, gen, act = DT[dt], torch.Generator().manual_seed(sum(size)), list(ACT)[sum(size) % 4]
    x, wg, wu, wd, dout = [normal(gen, s, dtype, k)[0].cuda() for s, k in
                           (((T, di), 1.0), ((di, f), 1.5 * di ** -0.5), ((di, f), di ** -0.5), ((f, do), f ** -0.5), ((T, do), 1.0))]
    wide = [torch.empty(T, f, device="cuda") for _ in range(2)]
    narrow = [Array(T, f, dtype, f + more, shift) for _ in range(2)]
    outs, grads = [], []
    for kind in ("wide", "narrow"):
        out = torch.empty(T, do, dtype=dtype, device="cuda")
        kw = (dict(pre_gate=wide[0].data_ptr(), pre_up=wide[1].data_ptr()) if kind == "wide" else
              dict(pre_gate=narrow[0].ptr, pre_up=narrow[1].ptr, ld_pre=f + more, pre_dtype=CODE[dt]))
        a = engine.gated_ffn_args(T, di, f, do, CODE[dt], ACT[act], x=x.data_ptr(), w_gate=wg.data_ptr(), w_up=wu.data_ptr(), w_down=wd.data_ptr(),
                                  out=out.data_ptr(), **kw)
        n = max(engine.gated_ffn_workspace(a), engine.gated_ffn_workspace(a, backward=True))
        ws = workspace(n)
        torch.cuda.synchronize()
        engine.gated_ffn_dev(a, ws.data_ptr(), n)
        engine.sync()
        outs.append(out)
        if kind == "wide":
            rounded = [t.to(dtype) for t in wide]
            for t, r in zip(wide, rounded):
                t.copy_(r)                                # the backward passes of both read the same values
        else:
            for t, r in zip(narrow, rounded):
                assert torch.equal(t.view, r) and t.untouched_outside()
        d = {k: torch.empty(s, dtype=dtype, device="cuda") for k, s in (("dx", (T, di)), ("dw_gate", (di, f)), ("dw_up", (di, f)), ("dw_down", (f, do)))}
        torch.cuda.synchronize()
        engine.gated_ffn_backward_dev(a, engine.gated_ffn_grads(dout=dout.data_ptr(), **{k: t.data_ptr() for k, t in d.items()}), ws.data_ptr(), n)
        engine.sync()
        grads.append(d)
    assert torch.equal(*outs)
    for k in grads[0]:
        assert torch.isfinite(grads[0][k]).all() and torch.equal(grads[0][k], grads[1][k]), k
