"""What the compiler made of the kernels, read from the library built here."""
import collections
import concurrent.futures

import pytest

import codegen
from roundtrip_amd import _lib

LOST = """
s_and_saveexec_b64 s[4:5], vcc
s_cbranch_execz L0
v_add_u32_e32 v1, 1, v1
L0:
s_nop 0
v_accvgpr_write_b32 a154, v21
s_or_b64 exec, exec, s[4:5]
ds_bpermute_b32 v1, v2, v3
s_endpgm
""".split("\n")


def test_the_search_finds_a_register_saved_before_its_lanes_are_on():
    lines = [t for t in LOST if t]
    assert codegen.before_the_lanes_are_back(lines) == [("L0", "v_accvgpr_write_b32 a154, v21")]
    lines[5], lines[6] = lines[6], lines[5]
    assert codegen.before_the_lanes_are_back(lines) == []


def looked_at(path):
    found, n = [], collections.Counter()
    for name, body in codegen.kernels(codegen.disassembly(path)):
        n["kernels"] += 1
        n["branches"] += sum(t.startswith("s_cbranch_execz ") for t in body)
        found += [(name,) + f for f in codegen.before_the_lanes_are_back(body)]
        packed = [t for t in body if t.startswith(("v_pk_add_f32", "v_pk_mul_f32", "v_pk_fma_f32"))]
        found += [(name, t) for t in packed[:3]]
    return found, n


@pytest.mark.skipif(not codegen.tools(), reason="needs ROCm's llvm-objcopy and llvm-objdump")
def test_no_lane_is_lost_and_no_float32_is_packed(tmp_path):
    """The allocator once saved lane * rem where a branch's lanes were still off, in one form of the estimator's kernel; every point
    of a leftover pass then got the first one's score.  Packed float32 instructions are built out (-packed-fp32-ops)."""
    files = codegen.code_objects(_lib.LIB_PATH, str(tmp_path))
    with concurrent.futures.ProcessPoolExecutor(max(1, min(5, len(files)))) as pool:
        parts = list(pool.map(looked_at, files))
    n = sum((p[1] for p in parts), collections.Counter())
    assert n["kernels"] > 250 and n["branches"] > 1000, n          # the library was read
    assert [f for p in parts for f in p[0]] == []
