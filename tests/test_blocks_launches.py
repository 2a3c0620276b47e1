"""Which kernels the network-block operators launch, seen without a GPU (launches.py)."""
import ctypes as C
import os

import pytest

pytest.importorskip("torch")
import launches  # noqa: E402
import test_gpu_blocks as gpu  # noqa: E402
import test_gpu_blocks_kernels as kernels  # noqa: E402


@pytest.fixture(scope="module")
def double():
    if not os.path.exists(launches.SO):
        pytest.skip("built by __graft_entry__.build()")
    return launches.Double()


def marked(test, names):
    """The values a test is parametrised with."""
    for m in test.pytestmark:
        if m.name == "parametrize" and m.args[0] == names:
            return m.args[1]
    raise KeyError(names)


TYPES = ("f32", "bf16", "f16")


def ffn_calls():
    """What the GPU tests ask of the gated feed-forward block: (size, type, strides, shift, x_lo)."""
    none = (0,) * 5
    for size in gpu.SIZES + [(40, 64, 192, 32)]:
        for dt in TYPES:
            yield size, dt, none, 0, False
    for lds, shift in marked(gpu.test_gated_ffn_strides_and_alignment, "lds,shift"):
        for dt in TYPES:
            for T in (70, 5):
                yield (T, 64, 128, 96), dt, lds, shift, False
    for size, lds, shift in marked(gpu.test_gated_ffn_odd_widths_of_many_rows, "size,lds,shift"):
        for dt in TYPES:
            yield size, dt, lds, shift, dt != "f32"
    for size in marked(gpu.test_gated_ffn_with_the_rest_of_x, "size"):
        for dt in ("bf16", "f16"):
            yield size, dt, none, 0, True
    for size in marked(gpu.test_gated_ffn_few_rows_of_odd_widths, "size"):
        for dt in TYPES:
            yield size, dt, none, 0, False
            yield size, dt, (1, 3, 5, 7, 9), 1, False
    for size in marked(gpu.test_gated_ffn_many_tiles, "size"):
        for dt in TYPES:
            yield size, dt, none, 0, False
    for size, dt, shift, lo in kernels.ALL:
        yield size, dt, none, shift, lo


def norm_calls():
    for T, d, rpg in marked(gpu.test_block_norm, "T,d,rpg"):
        for kind in ("rms", "layer"):
            for dt in TYPES:
                yield (T, d, dt, kind, rpg), (0,) * 5, 0
    for dt in ("bf16", "f16"):
        yield (2, 32768, dt, "layer", 1), (0,) * 5, 0
        yield (3, 32761, dt, "rms", 2), (0,) * 5, 0
    for rpg in marked(gpu.test_block_norm_many_rows, "rpg"):
        for dt in ("f32", "bf16"):
            yield (12289, 24, dt, "rms", rpg), (0,) * 5, 0
    for rpg in marked(gpu.test_block_norm_many_rows_of_a_workgroup, "rpg"):
        for dt in ("f32", "bf16"):
            yield (2500, 2200, dt, "layer", rpg), (0,) * 5, 0
    for lds, shift in marked(gpu.test_block_norm_strides_and_alignment, "lds,shift"):
        for dt in TYPES:
            yield (21, 200, dt, "rms", 4), lds, shift
            yield (4, 2304, dt, "layer", 3), lds, shift
    for (T, d, rpg), dt, kind in kernels.ALL_NORMS:
        yield (T, d, dt, kind, rpg), (0,) * 5, 0


def test_every_kernel_is_run_by_a_gpu_test(double):
    seen = {"zero_rows_kernel"}                          # test_gated_ffn_without_tokens
    for size, dt, lds, shift, lo in ffn_calls():
        for call in double.ffn(*size, dt, lds=lds, shift=shift, lo=lo):
            seen.update(x.kernel for x in call)
    for size, lds, shift in norm_calls():
        for call in double.norm(*size, lds=lds, shift=shift):
            seen.update(x.kernel for x in call)
    assert sorted(double.kernels() - seen) == []


def product(double, size, dt, shift, lo, which):
    fwd, back = [[x for x in call if x.kernel.startswith("gemm_") and "join" not in x.kernel] for call in double.ffn(*size, dt, shift=shift, lo=lo)]
    return dict(zip(("gated", "down", "dh", "dx", "dw_in", "dw_down"), fwd + back))[which]


@pytest.mark.parametrize("case,which,steps,splits", list(zip(
    kernels.BIG, ["gated", "gated", "gated", "down", "down", "dh", "dx", "dx", "dw_in", "dw_in"],
    [4, 3, 110, 3, 87, 3, 4, 96, 3, 52], [1, 1, 8, 1, 8, 1, 1, 8, 1, 4])))
def test_the_largest_tiles_turn_their_buffers(double, case, which, steps, splits):
    """256 x 256 tiles in every layout and with every epilogue: odd and even steps, two segments, K in one run and in several."""
    size, types, shift, lo = case
    for dt in types.split():
        x = product(double, size, dt, shift, lo, which)
        assert x.kernel.startswith("gemm_big_kernel<"), x
        assert (x.steps, x.splits) == (steps, splits), x
        assert x.splits == 1 or x.each >= 3, x


@pytest.mark.parametrize("case,which,steps,splits", list(zip(
    kernels.TILES, ["gated", "gated", "gated", "dh", "dh", "dw_in", "dw_in", "down", "down", "dx", "dx", "gated", "gated", "down", "down"],
    [3, 143, 4, 3, 6, 3, 3, 3, 9, 176, 286, 4, 38, 3, 17], [1, 8, 1, 1, 1, 1, 1, 1, 1, 8, 16, 1, 13, 1, 6])))
def test_tiles_of_128(double, case, which, steps, splits):
    size, types, shift, lo = case
    for dt in types.split():
        x = product(double, size, dt, shift, lo, which)
        assert ", 128, 128, 2, 2, " in x.kernel, x
        assert (x.steps, x.splits) == (steps, splits), x


def test_sizes_of_the_measured_figures_get_the_kernels_named_there(double):
    """The launches of the cases whose figures stand beside the kernels."""
    names = lambda call: [x.kernel for x in call]  # noqa: E731
    fwd, back = double.ffn(4096, 2048, 8192, 2048, "bf16")
    assert names(fwd) == ["gemm_big_kernel<1, 0, 1, 1>", "gemm_kernel<1, 0, 1, 0, 128, 128, 2, 2, true>"]
    assert names(back) == ["gemm_big_kernel<1, 0, 0, 2>", "gemm_big_kernel<1, 0, 0, 0>", "gemm_join_kernel<1, 0>"] + ["gemm_big_kernel<1, 1, 1, 0>"] * 2
    fwd, _ = double.ffn(10000, 512, 1024, 512, "f32")
    assert names(fwd) == ["gemm_kernel<0, 0, 1, 1, 128, 128, 2, 2, true>", "gemm_kernel<0, 0, 1, 0, 64, 64, 2, 2, true>"]
    fwd, _ = double.ffn(1, 4096, 16384, 4096, "bf16")
    assert names(fwd) == ["gemv_kernel<1, 1, 1, 16, false>", "gemv_kernel<1, 0, 1, 16, false>", "gemm_join_kernel<1, 0>"]


def every_entry(double):
    """(name, a call that launches) of each entry point."""
    f, r = double.ffn_args(40, 64, 96, 32, "bf16")
    n, s = double.norm_args(20, 64, "f32", "rms", 3)
    L, ws = double.lib, (double.WS, 1 << 62)
    return [("rt_gated_ffn_dev", lambda: L.rt_gated_ffn_dev(double.ctx, C.byref(f), *ws)),
            ("rt_gated_ffn_backward_dev", lambda: L.rt_gated_ffn_backward_dev(double.ctx, C.byref(f), C.byref(r), *ws)),
            ("rt_block_norm_dev", lambda: L.rt_block_norm_dev(double.ctx, C.byref(n))),
            ("rt_block_norm_backward_dev", lambda: L.rt_block_norm_backward_dev(double.ctx, C.byref(n), C.byref(s), *ws))]


def test_the_current_device_stays_current(double):
    """A context of another device than the current one: its device is current for the launches, the other one again behind
    them, also where one fails half-way."""
    other = launches.Double(device=3)
    for name, call in every_entry(other):
        other.reset(current=1)
        assert call() == 0, name
        lines = other.calls()
        assert lines[0] == "device 3" and lines[-1] == "device 1", (name, lines)
        assert len(lines) > 2 and all(line.endswith("on device 3") for line in lines[1:-1]), (name, lines)
        for fail_at in range(len(lines) - 2):
            other.reset(current=1, fail_at=fail_at)
            assert call() == 2 and "an error of the double" in other.error(), (name, fail_at)       # RT_EHIP
            assert other.lib.double_current() == 1, (name, fail_at)
            assert len(other.calls()) == fail_at + 3, (name, fail_at)      # and nothing is launched behind the one that failed
    for name, call in every_entry(double):
        double.reset(current=0)
        assert call() == 0
        assert not [line for line in double.calls() if line.startswith("device")], name
