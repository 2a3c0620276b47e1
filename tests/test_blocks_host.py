"""What the network-block entry points refuse, and what they ask for: their checks run on the host, before any GPU call, so
rt_block.hip is linked with a stand-in for the context (tests/block_double) and needs no GPU."""
import ctypes as C
import os

import pytest

from roundtrip_amd import _lib

HERE = os.path.dirname(os.path.abspath(__file__))
SO = os.path.join(HERE, "block_double", "librt_block_double.so")
OK, EINVAL, EHIP, EUNSUPPORTED = 0, 1, 2, 4


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(SO):
        pytest.skip("built by __graft_entry__.build()")
    L = C.CDLL(SO)
    L.double_ctx.restype = C.c_void_p
    L.double_error.restype = C.c_char_p
    L.double_error.argtypes = [C.c_void_p]
    real = _lib.load()
    for n in ("rt_gated_ffn_workspace", "rt_gated_ffn_dev", "rt_gated_ffn_backward_dev", "rt_block_norm_workspace", "rt_block_norm_dev",
              "rt_block_norm_backward_dev", "rt_ctx_stream"):
        getattr(L, n).argtypes = getattr(real, n).argtypes
    L.ctx = C.c_void_p(L.double_ctx())
    return L


def refused(lib, rc, code, *words):
    text = lib.double_error(lib.ctx).decode()
    assert rc == code, (rc, text)
    for w in words:
        assert w in text, text


BASE = 1 << 32        # addresses that nothing reads: every call below ends in a check


def ffn(**kw):
    a = dict(T=10, d_in=16, d_ff=32, d_out=16, dtype=_lib.RT_BF16, act=0)
    at = {k: BASE + i * (1 << 24) for i, k in enumerate(("x", "w_gate", "w_up", "w_down", "out"))}
    a.update(at)
    a.update(kw)
    return _lib.Engine.gated_ffn_args(**a)


def ffn_kept(**kw):
    return ffn(**dict(dict(pre_gate=BASE + (1 << 28), pre_up=BASE + (1 << 28) + (1 << 24)), **kw))


WS = C.c_void_p(BASE + (1 << 30))


@pytest.mark.parametrize("kw,code,words", [
    (dict(dtype=7), EINVAL, "dtype"), (dict(dtype=-1), EINVAL, "dtype"), (dict(act=4), EINVAL, "activation"), (dict(act=-1), EINVAL, "activation"),
    (dict(alpha=float("nan")), EINVAL, "alpha"), (dict(alpha=float("inf")), EINVAL, "alpha"),
    (dict(T=-1), EINVAL, "T = -1"), (dict(T=1 << 41), EINVAL, "T = "), (dict(d_in=0), EINVAL, "widths"), (dict(d_ff=-3), EINVAL, "widths"),
    (dict(d_out=(1 << 20) + 1), EINVAL, "widths"), (dict(x=None), EINVAL, "x is NULL"), (dict(w_gate=None), EINVAL, "w_gate is NULL"),
    (dict(w_up=None), EINVAL, "w_up is NULL"), (dict(w_down=None), EINVAL, "w_down is NULL"), (dict(out=None), EINVAL, "out is NULL"),
    (dict(x=BASE + 1), EINVAL, "x is not aligned"), (dict(dtype=0, w_up=BASE + (1 << 25) + 2), EINVAL, "w_up is not aligned"),
    (dict(ldx=15), EINVAL, "row stride of x"), (dict(ld_in=31), EINVAL, "row stride of w_gate"), (dict(ld_out=-16), EINVAL, "row stride of out"),
    (dict(ld_down=(1 << 20) + 8), EUNSUPPORTED, "row stride of w_down"), (dict(pre_gate=BASE + (1 << 28)), EINVAL, "both of pre_gate"),
    (dict(pre_up=BASE + (1 << 28)), EINVAL, "both of pre_gate"), (dict(out=BASE), EINVAL, "out and x overlap"),
    (dict(out=BASE + 318), EINVAL, "out and x overlap"), (dict(out=BASE + (1 << 24) + 64), EINVAL, "out and w_gate overlap"),
    (dict(pre_gate=BASE + (1 << 28), pre_up=BASE + (1 << 28) + 4), EINVAL, "overlap"), (dict(pre_gate=BASE + (1 << 28) + 2, pre_up=BASE + (1 << 27)), EINVAL, "pre_gate is not aligned"), (dict(out=WS.value), EINVAL, "workspace and out overlap"),
    (dict(dtype=0, x_lo=BASE + (1 << 26) + (1 << 25)), EINVAL, "x_lo is for 16-bit"), (dict(x_lo=BASE + (1 << 26) + (1 << 25) + 1), EINVAL, "x_lo is not aligned"),
    (dict(x_lo=BASE + 4 * (1 << 24) + 8), EINVAL, "out and x_lo overlap"),
    (dict(T=1 << 38, d_ff=1 << 20, d_in=1 << 20), EUNSUPPORTED, "one launch")])
def test_gated_ffn_refusals(lib, kw, code, words):
    a = ffn(**kw)
    refused(lib, lib.rt_gated_ffn_dev(lib.ctx, C.byref(a), WS, 1 << 62), code, words)


def test_gated_ffn_workspace_is_asked_for(lib):
    a, n = ffn(), C.c_size_t()
    assert lib.rt_gated_ffn_workspace(lib.ctx, C.byref(a), 0, C.byref(n)) == OK
    assert n.value >= 10 * 32 * 2
    need = n.value
    refused(lib, lib.rt_gated_ffn_dev(lib.ctx, C.byref(a), None, 0), EINVAL, "workspace is NULL", str(need))
    refused(lib, lib.rt_gated_ffn_dev(lib.ctx, C.byref(a), WS, need - 1), EINVAL, "%d needed" % need)
    refused(lib, lib.rt_gated_ffn_dev(lib.ctx, C.byref(a), C.c_void_p(WS.value + 8), need), EINVAL, "aligned to 16")
    refused(lib, lib.rt_gated_ffn_workspace(lib.ctx, C.byref(a), 0, None), EINVAL, "bytes is NULL")
    refused(lib, lib.rt_gated_ffn_workspace(lib.ctx, None, 0, C.byref(n)), EINVAL, "arguments are NULL")
    refused(lib, lib.rt_gated_ffn_dev(lib.ctx, None, WS, need), EINVAL, "arguments are NULL")
    assert lib.rt_gated_ffn_dev(None, C.byref(a), WS, need) == EINVAL
    assert lib.rt_gated_ffn_workspace(lib.ctx, C.byref(a), 1, C.byref(n)) == OK
    assert n.value >= 3 * 10 * 32 * 2
    zero = ffn(T=0)
    assert lib.rt_gated_ffn_dev(lib.ctx, C.byref(zero), None, 0) == OK         # nothing to do, before any GPU call


@pytest.mark.parametrize("kw,gr,words", [
    (dict(pre_gate=None, pre_up=None), {}, "pre_gate is NULL"), ({}, dict(dout=None), "dout is NULL"), ({}, dict(ld_dout=8), "row stride of dout"),
    ({}, dict(ld_dx=8), "row stride of dx"), ({}, dict(ld_dw_in=31), "row stride of dw_gate"), ({}, dict(dw_down=BASE + (1 << 27) + (1 << 26), ld_dw_down=1), "row stride of dw_down"),
    ({}, dict(dx=BASE), "dx and x overlap"), ({}, dict(dx=BASE + (1 << 28)), "dx and pre_gate overlap"),
    ({}, dict(dw_up=BASE + (1 << 24)), "dw_up and w_gate overlap"),
    ({}, dict(dw_gate=BASE + (1 << 29), dw_up=BASE + (1 << 29)), "dw_up and dw_gate overlap"), ({}, dict(dw_down=WS.value + 64), "overlap")])
def test_gated_ffn_backward_refusals(lib, kw, gr, words):
    a = ffn_kept(**kw)
    g = dict(dout=BASE + (1 << 27), dx=BASE + (1 << 29) + (1 << 26), dw_gate=BASE + (1 << 29) + (1 << 25))
    g.update(gr)
    r = _lib.Engine.gated_ffn_grads(**g)
    refused(lib, lib.rt_gated_ffn_backward_dev(lib.ctx, C.byref(a), C.byref(r), WS, 1 << 62), EINVAL, words)
    refused(lib, lib.rt_gated_ffn_backward_dev(lib.ctx, C.byref(a), None, WS, 1 << 62), EINVAL, "gradients are NULL")


def norm(**kw):
    a = dict(T=12, d=64, dtype=_lib.RT_F32, kind=0, rows_per_gate=5)
    a.update({k: BASE + i * (1 << 24) for i, k in enumerate(("x", "branch", "y", "n", "gate", "w_post", "w_pre"))})
    a.update(kw)
    return _lib.Engine.block_norm_args(**a)


@pytest.mark.parametrize("kw,code,words", [
    (dict(dtype=3), EINVAL, "dtype"), (dict(kind=2), EINVAL, "kind"), (dict(kind=-1), EINVAL, "kind"), (dict(T=-2), EINVAL, "T = -2"),
    (dict(T=1 << 31), EUNSUPPORTED, "one launch"), (dict(d=0), EINVAL, "d = 0"), (dict(d=16385), EUNSUPPORTED, "16384"),
    (dict(dtype=1, d=32769), EUNSUPPORTED, "32768"), (dict(eps=-1e-6), EINVAL, "eps"), (dict(eps=float("nan")), EINVAL, "eps"),
    (dict(res_scale=float("inf")), EINVAL, "finite"), (dict(branch_scale=float("nan")), EINVAL, "finite"), (dict(w_offset=float("nan")), EINVAL, "finite"),
    (dict(rows_per_gate=0), EINVAL, "rows_per_gate"), (dict(rows_per_gate=-4), EINVAL, "rows_per_gate"), (dict(x=None), EINVAL, "x is NULL"),
    (dict(y=None, n=None), EINVAL, "both NULL"), (dict(branch=None), EINVAL, "gate without a branch"), (dict(ldy=63), EINVAL, "row stride of y"),
    (dict(ld_gate=10), EINVAL, "row stride of gate"), (dict(ldx=1 << 21), EUNSUPPORTED, "row stride of x"), (dict(x=BASE + 2), EINVAL, "aligned"),
    (dict(y=BASE + 4), EINVAL, "y and x overlap"), (dict(y=BASE, ldy=65), EINVAL, "y and x overlap"), (dict(n=BASE + (1 << 24) + 256), EINVAL, "n and branch overlap"),
    (dict(n=BASE + (1 << 25)), EINVAL, "y and n overlap"), (dict(y=BASE + (1 << 26)), EINVAL, "y and gate overlap"),
    (dict(n=BASE + 5 * (1 << 24)), EINVAL, "n and w_post overlap"), (dict(n_lo=BASE + (1 << 27)), EINVAL, "n_lo is for 16-bit"),
    (dict(dtype=1, n=None, n_lo=BASE + (1 << 27)), EINVAL, "n_lo is for 16-bit"), (dict(dtype=1, n_lo=BASE), EINVAL, "n_lo and x overlap"),
    (dict(dtype=1, n_lo=BASE + 3 * (1 << 24) + 2), EINVAL, "n_lo and n overlap")])
def test_block_norm_refusals(lib, kw, code, words):
    a = norm(**kw)
    refused(lib, lib.rt_block_norm_dev(lib.ctx, C.byref(a)), code, words)


@pytest.mark.parametrize("kw,gr,words", [
    ({}, dict(dy=None, dn=None), "both NULL"), (dict(branch=None, gate=None), dict(dbranch=BASE + (1 << 29)), "without a branch"),
    (dict(branch=None, gate=None), dict(dw_post=BASE + (1 << 29)), "without a branch"), (dict(gate=None), dict(dgate=BASE + (1 << 29)), "without a gate"),
    (dict(branch=None), {}, "gate without"), (dict(y=None), {}, "y is NULL"), ({}, dict(dx=BASE + (1 << 24)), "dx and branch overlap"),
    ({}, dict(dx=BASE + (1 << 28) + 8), "dx and dy overlap"), ({}, dict(dbranch=BASE + (1 << 30) + 16), "overlap"),
    ({}, dict(dgate=BASE + (1 << 26)), "dgate and gate overlap"), ({}, dict(dw_pre=BASE + 6 * (1 << 24)), "dw_pre and w_pre overlap"),
    ({}, dict(dx=BASE + (1 << 28), dbranch=BASE + (1 << 28)), "dbranch and dx overlap"), ({}, dict(ld_dn=3), "row stride of dn")])
def test_block_norm_backward_refusals(lib, kw, gr, words):
    a = norm(**kw)
    g = dict(dy=BASE + (1 << 28), dn=BASE + (1 << 28) + (1 << 24), dx=BASE + (1 << 29) + (1 << 24))
    g.update(gr)
    r = _lib.Engine.block_norm_grads(**g)
    refused(lib, lib.rt_block_norm_backward_dev(lib.ctx, C.byref(a), C.byref(r), WS, 1 << 62), EINVAL, words)


def test_block_norm_workspace_is_asked_for(lib):
    a, n = norm(T=20000, rows_per_gate=15000), C.c_size_t()
    r = _lib.Engine.block_norm_grads(dy=BASE + (1 << 28), dx=BASE + (1 << 29))
    assert lib.rt_block_norm_workspace(lib.ctx, C.byref(a), C.byref(n)) == OK and n.value > 0
    refused(lib, lib.rt_block_norm_backward_dev(lib.ctx, C.byref(a), C.byref(r), WS, n.value - 1), EINVAL, "%d needed" % n.value)
    refused(lib, lib.rt_block_norm_backward_dev(lib.ctx, C.byref(a), C.byref(r), None, 0), EINVAL, "workspace is NULL")
    refused(lib, lib.rt_block_norm_dev(lib.ctx, None), EINVAL, "arguments are NULL")
    zero = norm(T=0)
    assert lib.rt_block_norm_dev(lib.ctx, C.byref(zero)) == OK
    refused(lib, lib.rt_ctx_stream(lib.ctx, None), EINVAL, "stream is NULL")


def test_columns_of_one_buffer_do_not_overlap(lib):
    """Gate and up, and what is kept of them, as the halves of one array: past every check (the call then needs a GPU, or the
    workspace that is refused here)."""
    a = ffn(w_up=BASE + (1 << 24) + 64, ld_in=64, pre_gate=BASE + (1 << 28), pre_up=BASE + (1 << 28) + 128, ld_pre=64)
    refused(lib, lib.rt_gated_ffn_dev(lib.ctx, C.byref(a), None, 0), EINVAL, "workspace is NULL")
    shifted = ffn(pre_gate=BASE + (1 << 28), pre_up=BASE + (1 << 28) + 124, ld_pre=64)
    refused(lib, lib.rt_gated_ffn_dev(lib.ctx, C.byref(shifted), WS, 1 << 62), EINVAL, "pre_up and pre_gate overlap")


def test_struct_layout_matches_the_header(tmp_path):
    """The ctypes structures against the compiler's view of include/rt_is.h."""
    import subprocess
    src = tmp_path / "s.c"
    names = {"rt_gated_ffn": _lib.RtGatedFfn, "rt_gated_ffn_grads": _lib.RtGatedFfnGrads, "rt_block_norm": _lib.RtBlockNorm,
             "rt_block_norm_grads": _lib.RtBlockNormGrads}
    lines = ["#include <stdio.h>", '#include "rt_is.h"', "int main(void) {"]
    for n, s in names.items():
        lines.append('printf("%s %%zu\\n", sizeof(%s));' % (n, n))
        lines += ['printf("%s.%s %%zu\\n", offsetof(%s, %s));' % (n, f, n, f) for f, _ in s._fields_]
    src.write_text("\n".join(lines + ["return 0; }"]))
    exe = str(tmp_path / "s")
    subprocess.check_call(["gcc", "-I", os.path.join(os.path.dirname(HERE), "include"), "-o", exe, str(src)])
    got = dict(line.split() for line in subprocess.check_output([exe]).decode().splitlines())
    for n, s in names.items():
        assert int(got[n]) == C.sizeof(s)
        for f, _ in s._fields_:
            assert int(got["%s.%s" % (n, f)]) == getattr(s, f).offset, (n, f)


def test_more_tiles_than_one_launch_holds_are_refused(lib):
    """A launch holds less than 2^32 threads, a tile takes up to 512."""
    a, n = ffn(T=1 << 34), C.c_size_t()
    for backward in (0, 1):
        refused(lib, lib.rt_gated_ffn_workspace(lib.ctx, C.byref(a), backward, C.byref(n)), EUNSUPPORTED, "one launch")
    a = ffn(T=1 << 28)
    assert lib.rt_gated_ffn_workspace(lib.ctx, C.byref(a), 0, C.byref(n)) == OK
