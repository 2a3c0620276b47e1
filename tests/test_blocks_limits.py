"""How many rows and columns a call of the gated feed-forward block covers, without a GPU (launches.py)."""
import ctypes as C
import os

import pytest

import launches

UNSUPPORTED = 4
MOST = (1 << 23) - 1            # tiles of a launch


@pytest.fixture(scope="module")
def double():
    if not os.path.exists(launches.SO):
        pytest.skip("built by __graft_entry__.build()")
    return launches.Double()


def workspace(double, size, dt, backward):
    a, _ = double.ffn_args(*size, dt)
    n = C.c_size_t()
    return double.lib.rt_gated_ffn_workspace(double.ctx, C.byref(a), backward, C.byref(n)), n.value


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_rows_that_only_larger_tiles_cover(double, dt):
    """2^29 rows and more: more tiles of 64 rows than a launch holds, but not of 128."""
    T = (MOST << 6) + 1
    for size in ((T, 16, 64, 16), (128 * MOST, 16, 64, 16)):
        for call in double.ffn(*size, dt):
            for x in call:
                assert x.grid[0] * x.block < 1 << 32, x
        for backward in (0, 1):
            assert workspace(double, size, dt, backward)[0] == 0
    for backward in (0, 1):
        rc, _ = workspace(double, (128 * MOST + 1, 16, 64, 16), dt, backward)
        assert rc == UNSUPPORTED and "one launch" in double.error()


def test_a_forward_call_is_not_held_to_the_backward_pass(double):
    """The gradients of 2^20 x 2^20 weights have more tiles than a launch holds; one row through those weights has not."""
    size = (1, 1 << 20, 1 << 20, 8)
    assert workspace(double, size, "bf16", 0)[0] == 0
    rc, _ = workspace(double, size, "bf16", 1)
    assert rc == UNSUPPORTED and "one launch" in double.error()
