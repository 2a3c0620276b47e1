"""perf/operators.py as a program uses it: its arrays are torch's, its calls the engine's."""
import importlib
import os
import subprocess
import sys

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    if root not in sys.path:
        sys.path.insert(0, root)
    m = importlib.import_module("perf.operators")
    m.own = True
    yield m
    m.own = False


CASES = [{"op": "ffn", "T": 300, "d": 256, "f": 512, "dtype": "bf16", "act": "silu", "train": True},
         {"op": "norm", "T": 300, "d": 256, "dtype": "f32", "kind": "rms", "rows_per_gate": 3, "train": True},
         {"op": "block", "T": 8, "d": 256, "f": 512, "dtype": "f16", "act": "gelu", "kind": "layer", "rows_per_gate": 0, "train": False}]


def late():
    """Some milliseconds of work on torch's stream."""
    a = b = torch.randn(4096, 4096, device="cuda")
    for _ in range(12):
        b = (b @ a) * 2.0 ** -6


@pytest.mark.parametrize("case", CASES, ids=lambda c: c["op"])
def test_inputs_that_torch_has_yet_to_write_are_waited_for(engine, ops, case):
    s = ops.prepare(case, 3)
    torch.cuda.synchronize()
    ops.run(s)
    torch.cuda.synchronize()
    want = {k: v.clone() for k, v in s["out"].items() if v is not None}
    del s
    for _ in range(3):
        torch.cuda.empty_cache()                         # new memory, in which the inputs of the pass before do not lie
        filler = torch.full((1 << 26,), float("nan"), device="cuda")
        del filler
        torch.cuda.synchronize()
        late()
        s = ops.prepare(case, 3)                         # enqueued behind it, and nothing waits
        ops.run(s)
        s["eng"].sync()
        for k, v in want.items():
            assert torch.equal(s["out"][k], v), k
        del s


def test_arrays_of_a_pass_under_way_go_to_nobody_else(engine, ops):
    case = {"op": "ffn", "T": 2048, "d": 2048, "f": 4096, "dtype": "bf16", "act": "silu", "train": True}
    s = ops.prepare(case, 4)
    torch.cuda.synchronize()
    eng = s["eng"]
    for _ in range(20):                                  # some milliseconds on the engine's stream
        ops.run(s)
    del s
    new = [torch.full((2048, 2048), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(8)]
    torch.cuda.synchronize()
    for t in new:
        assert bool((t == 7.0).all())
    eng.sync()


def test_a_program_that_ends_with_states_alive_ends_well(engine):
    """In whatever order the interpreter lets go of the engine and of the states."""
    code = ("import torch, perf.operators as p\n"
            "p.own = True\n"
            "c = %r\n"
            "states = [p.prepare(c, i) for i in range(2)]\n"
            "torch.cuda.synchronize()\n"
            "outs = [p.run(s) for s in states]\n"
            "torch.cuda.synchronize()\n"
            "print('done', flush=True)\n" % (CASES[0],))
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, stdout=subprocess.PIPE, stderr=subprocess.PIPE, timeout=100)
    assert r.returncode == 0 and r.stdout.strip() == b"done", (r.returncode, r.stdout[-500:], r.stderr[-2000:])
    assert b"Exception ignored" not in r.stderr, r.stderr[-2000:]
