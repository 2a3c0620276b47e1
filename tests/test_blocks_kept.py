"""The type of the gate and up that a gated feed-forward block keeps: what its field says and refuses, without a GPU (launches.py)."""
import ctypes as C
import os

import pytest

import launches
from roundtrip_amd import _lib

F32, BF16, F16 = _lib.RT_F32, _lib.RT_BF16, _lib.RT_F16


@pytest.fixture(scope="module")
def double():
    if not os.path.exists(launches.SO):
        pytest.skip("built by __graft_entry__.build()")
    return launches.Double()


def forward(double, a):
    double.reset()
    return double.lib.rt_gated_ffn_dev(double.ctx, C.byref(a), double.WS, 1 << 62)


def backward(double, a, r):
    double.reset()
    return double.lib.rt_gated_ffn_backward_dev(double.ctx, C.byref(a), C.byref(r), double.WS, 1 << 62)


@pytest.mark.parametrize("dt,pre", [("bf16", F16), ("f16", BF16), ("f32", BF16), ("f32", F16), ("bf16", 3), ("bf16", -1), ("f32", 7)])
def test_types_that_are_refused(double, dt, pre):
    a, r = double.ffn_args(10, 16, 32, 16, dt, pre_dtype=pre)
    for rc in (forward(double, a), backward(double, a, r)):
        assert rc == 1 and "pre_dtype %d" % pre in double.error()
    n = C.c_size_t()
    assert double.lib.rt_gated_ffn_workspace(double.ctx, C.byref(a), 0, C.byref(n)) == 1


@pytest.mark.parametrize("dt,code", [("bf16", BF16), ("f16", F16)])
def test_arrays_of_sixteen_bits(double, dt, code):
    """Gate and up one behind the other, as a program allocates them: of the call's type they lie apart, as float32 they would not."""
    T, f = 4096, 8192
    at = 40 * launches.BASE
    kw = dict(pre_gate=at, pre_up=at + T * f * 2)
    a, r = double.ffn_args(T, 2048, f, 2048, dt, pre_dtype=code, **kw)
    assert forward(double, a) == 0 and backward(double, a, r) == 0
    a.pre_up -= 2
    assert forward(double, a) == 1 and "pre_up and pre_gate overlap" in double.error()
    a, r = double.ffn_args(T, 2048, f, 2048, dt, **kw)
    assert forward(double, a) == 1 and "pre_up and pre_gate overlap" in double.error()
    # an element's alignment is enough, and needed
    a, r = double.ffn_args(10, 16, 32, 16, dt, pre_dtype=code, pre_gate=at + 2, pre_up=at + 4096)
    assert forward(double, a) == 0 and backward(double, a, r) == 0
    a.pre_gate += 1
    assert forward(double, a) == 1 and "pre_gate is not aligned" in double.error()
    a, r = double.ffn_args(10, 16, 32, 16, dt, pre_gate=at + 2, pre_up=at + 4096)
    assert forward(double, a) == 1 and "pre_gate is not aligned" in double.error()


def test_the_field_lies_in_what_was_the_upper_half_of_dtype():
    """A program compiled when dtype had 32 bits says float32 with its zeros there."""
    s = _lib.RtGatedFfn
    assert (s.dtype.offset, s.dtype.size, s.pre_dtype.offset, s.pre_dtype.size, s.act.offset) == (0, 2, 2, 2, 4)
    a = _lib.Engine.gated_ffn_args(1, 8, 8, 8, BF16, 0)
    assert a.pre_dtype == F32 and bytes(a)[:4] == (BF16).to_bytes(4, "little")
