"""The launches that calls of the network-block operators make, without a GPU: rt_block.hip and its kernels' host stubs linked
with a stand-in for the context and for HIP's launches (tests/launch_double)."""
import ctypes as C
import os
import re

from roundtrip_amd import _lib

SO = os.path.join(os.path.dirname(os.path.abspath(__file__)), "launch_double", "librt_launch_double.so")
BASE = 1 << 40                  # addresses that nothing reads, a terabyte apart
CODE = {"f32": _lib.RT_F32, "bf16": _lib.RT_BF16, "f16": _lib.RT_F16}
KIND = {"rms": _lib.RT_NORM_RMS, "layer": _lib.RT_NORM_LAYER}


class Launch(object):
    """One launch: kernel, grid (x, y, z), block, the device current at it; of a tiled product also splits and each split's steps."""

    def __init__(self, line):
        m = re.match(r"launch (.+?) \| grid (\d+) (\d+) (\d+) block (\d+)(?: \| splits (\d+) each (\d+) steps (\d+))? on device (\d+)$", line)
        self.kernel = m.group(1)
        n = [int(v) if v else 0 for v in m.groups()[1:]]
        self.grid, self.block, self.splits, self.each, self.steps, self.device = tuple(n[:3]), n[3], n[4], n[5], n[6], n[7]

    def __repr__(self):
        return "%s %r splits %d each %d of %d" % (self.kernel, self.grid, self.splits, self.each, self.steps)


class Double(object):
    def __init__(self, device=0, cus=256):
        self.lib = C.CDLL(SO)
        for n in ("double_error", "double_calls", "double_kernels"):
            getattr(self.lib, n).restype = C.c_char_p
        self.lib.double_ctx.restype = C.c_void_p
        self.lib.double_error.argtypes = [C.c_void_p]
        real = _lib.load()
        for n in ("rt_gated_ffn_workspace", "rt_gated_ffn_dev", "rt_gated_ffn_backward_dev", "rt_block_norm_workspace", "rt_block_norm_dev",
                  "rt_block_norm_backward_dev"):
            getattr(self.lib, n).argtypes = getattr(real, n).argtypes
        self.ctx = C.c_void_p(self.lib.double_ctx(device, cus))

    def kernels(self):
        return set(k for k in self.lib.double_kernels().decode().split("\n") if k)

    def error(self):
        return self.lib.double_error(self.ctx).decode()

    def reset(self, current=0, fail_at=-1):
        self.lib.double_reset(current, fail_at)

    def calls(self):
        return self.lib.double_calls().decode().splitlines()

    def launches(self, rc):
        assert rc == 0, self.error()
        return [Launch(line) for line in self.calls() if line.startswith("launch ")]

    WS = C.c_void_p(30 * BASE)

    @staticmethod
    def ffn_args(T, di, f, do, dt, lds=(0, 0, 0, 0, 0), shift=0, lo=False, **kw):
        """As test_gpu_blocks.ffn_case lays its arrays out."""
        es = 4 if dt == "f32" else 2
        at = lambda i, s=es: (i + 1) * BASE + shift * s  # noqa: E731
        ld = [w + k for w, k in zip((di, f, do, do, f), lds)]
        a = dict(x=at(0), w_gate=at(1), w_up=at(2), w_down=at(3), out=at(4), pre_gate=at(5, 4), pre_up=at(6, 4), x_lo=at(7) if lo else None,
                 ldx=ld[0], ld_in=ld[1], ld_down=ld[2], ld_out=ld[3], ld_pre=ld[4])
        a.update(kw)
        r = dict(dout=at(8), dx=at(9), dw_gate=at(10), dw_up=at(11), dw_down=at(12), ld_dout=ld[3], ld_dx=ld[0], ld_dw_in=ld[1], ld_dw_down=ld[2])
        return _lib.Engine.gated_ffn_args(T, di, f, do, CODE[dt], 0, **a), _lib.Engine.gated_ffn_grads(**r)

    def ffn(self, *size, **kw):
        """(the forward call's launches, the backward call's)"""
        a, r = self.ffn_args(*size, **kw)
        got = []
        self.reset()
        got.append(self.launches(self.lib.rt_gated_ffn_dev(self.ctx, C.byref(a), self.WS, 1 << 62)))
        self.reset()
        got.append(self.launches(self.lib.rt_gated_ffn_backward_dev(self.ctx, C.byref(a), C.byref(r), self.WS, 1 << 62)))
        return got

    @staticmethod
    def norm_args(T, d, dt, kind, rpg, lds=(0, 0, 0, 0, 0), shift=0):
        """As test_gpu_blocks.norm_case lays its arrays out."""
        es = 4 if dt == "f32" else 2
        at = lambda i: (i + 1) * BASE + shift * es  # noqa: E731
        ld = [d + k for k in lds]
        a = dict(x=at(0), branch=at(1), y=at(2), n=at(3), w_post=at(4), w_pre=at(5), gate=at(6) if rpg else None, rows_per_gate=rpg or 1, ldx=ld[0],
                 ld_branch=ld[1], ldy=ld[2], ldn=ld[3], ld_gate=ld[4])
        r = dict(dy=at(8), dn=at(9), dx=at(10), dbranch=at(11), dgate=at(12) if rpg else None, dw_post=at(13), dw_pre=at(14), ld_dy=ld[0], ld_dn=ld[1],
                 ld_dx=ld[2], ld_dbranch=ld[3], ld_dgate=ld[4])
        return _lib.Engine.block_norm_args(T, d, CODE[dt], KIND[kind], **a), _lib.Engine.block_norm_grads(**r)

    def norm(self, *size, **kw):
        a, r = self.norm_args(*size, **kw)
        got = []
        self.reset()
        got.append(self.launches(self.lib.rt_block_norm_dev(self.ctx, C.byref(a))))
        self.reset()
        got.append(self.launches(self.lib.rt_block_norm_backward_dev(self.ctx, C.byref(a), C.byref(r), self.WS, 1 << 62)))
        return got
