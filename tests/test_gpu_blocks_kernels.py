"""Every kernel of the network blocks, run on sizes that the plan gives it: test_blocks_launches.py holds these
lists against the launches that they make (on 256 CUs), so a change of the plan cannot leave a kernel untested unseen."""
import pytest

torch = pytest.importorskip("torch")
from test_gpu_blocks import ffn_case, norm_case  # noqa: E402

pytestmark = pytest.mark.gpu

# (size, types, shift of every array in elements, x_lo).  What the plan makes of each stands beside it: the product (gated and down
# forward; dh, dx, dw_in, dw_down backward), its tile, its steps of 128 bytes of k, and how many workgroups share them.
BIG = [
    ((3397, 88, 1168, 40), "bf16 f16", 0, True),         # gated 256, two segments of 2 steps
    ((3397, 136, 1168, 40), "bf16 f16", 0, False),       # gated 256, 3 steps
    ((130, 3488, 2056, 456), "bf16 f16", 0, True),       # gated 256, two segments of 55 in 8 runs, one of which holds the border
    ((2059, 42, 136, 3933), "bf16 f16", 1, False),       # down 256, 3 steps, copies of odd widths
    ((130, 8, 5536, 4120), "bf16 f16", 0, False),        # down 256, 87 steps in 8 runs
    ((4033, 45, 2184, 140), "bf16 f16", 1, False),       # dh 256, 3 steps
    ((1954, 4256, 72, 64), "bf16 f16", 0, False),        # dx 256, two segments of 2 steps
    ((131, 4416, 3032, 160), "bf16 f16", 0, False),      # dx 256, two segments of 48 steps in 8 runs
    ((133, 920, 4248, 64), "bf16 f16", 0, False),        # dw_in 256, 3 steps, the gate's and up's side by side
    ((3279, 4224, 136, 256), "bf16", 0, False),          # dw_in 256, 52 steps in 4 runs
]
TILES = [
    ((2022, 80, 1696, 40), "f32", 0, False),             # gated 128, 3 steps
    ((72, 4552, 2152, 984), "f32", 0, False),            # gated 128, 143 steps in 8 runs
    ((4619, 116, 652, 78), "f32", 1, False),             # gated 128 of unaligned arrays
    ((2757, 48, 2696, 96), "f32", 0, False),             # dh 128, 3 steps
    ((2644, 50, 2930, 164), "f32", 1, False),            # dh 128 of unaligned arrays, 6 steps
    ((68, 1712, 2288, 40), "f32", 0, False),             # dw_in 128, 3 steps
    ((75, 934, 3915, 46), "f32", 0, False),              # dw_in 128 of unaligned arrays, 3 steps
    ((3252, 139, 69, 2387), "f32", 0, False),            # down 128, 3 steps, copies of odd widths
    ((1787, 2233, 283, 4468), "f32", 1, False),          # down 128 of unaligned arrays, 9 steps
    ((75, 4856, 2816, 496), "f32", 0, False),            # dx 128, two segments of 88 steps in 8 runs
    ((70, 2131, 4567, 184), "f32", 1, False),            # the same of unaligned arrays, two of 143 in 16
    ((247, 69, 4149, 44), "bf16 f16", 0, True),          # gated 128 of unaligned arrays, two segments of 2 steps
    ((77, 1192, 540, 68), "bf16 f16", 0, True),          # the same, two of 19 in 13 runs
    ((515, 55, 133, 4108), "bf16 f16", 0, False),        # down 128 of unaligned arrays, 3 steps
    ((65, 203, 1069, 2129), "bf16 f16", 0, False),       # the same, 17 steps in 6 runs; dh in 12
]
# One to four rows on the vector unit: 32 and 64 columns a workgroup
ROWS = [
    ((1, 40, 8200, 24), "bf16 f16 f32", 0, True), ((2, 40, 8200, 24), "bf16 f16 f32", 0, True), ((3, 40, 8200, 24), "bf16 f16 f32", 0, True),
    ((1, 24, 40, 8200), "bf16 f16 f32", 0, False), ((2, 24, 40, 8200), "bf16 f16 f32", 0, False), ((4, 24, 40, 8200), "bf16 f16 f32", 0, False),
    ((1, 601, 16420, 8), "bf16 f16 f32", 0, True), ((2, 601, 16420, 8), "bf16 f16 f32", 0, True), ((4, 601, 16420, 8), "bf16 f16 f32", 0, True),
    ((1, 8, 602, 16421), "bf16 f16 f32", 1, False), ((2, 8, 602, 16421), "bf16 f16 f32", 1, False), ((3, 8, 602, 16421), "bf16 f16 f32", 1, False),
    ((1, 8, 4200, 4100), "bf16", 0, False),              # down: 64 columns, K split in 3
]
# Sixteen-bit types without x_lo
PLAIN_ROWS = [((n, 40, 8200, 24), "bf16 f16", 0, False) for n in (1, 2, 3)] + [((n, 601, 16420, 8), "bf16 f16", 0, False) for n in (1, 2, 4)]

ALL = [(size, dt, shift, lo and dt != "f32") for size, types, shift, lo in BIG + TILES + ROWS + PLAIN_ROWS for dt in types.split()]


@pytest.mark.parametrize("size,dt,shift,lo", ALL, ids=["%s-%s%s%s" % ("x".join(map(str, s)), d, "-unaligned" if h else "", "-lo" if o else "") for s, d, h, o in ALL])
def test_gated_ffn_kernel(engine, size, dt, shift, lo):
    act = ("silu", "gelu", "lrelu", "sigmoid")[sum(size) % 4]
    ffn_case(engine, *size, dt, act, shift=shift, seed=sum(size) % 1000, lo=lo)


# Norms of as many rows as there are CUs or more (a row to a wave up to 256 chunks of 16 bytes) and wide rows: (T, d, rows of a gate), types
NORMS = [
    ((300, 512, 7), "f32"), ((300, 511, 7), "f32"), ((270, 1016, 100), "f32"), ((270, 1019, 100), "f32"),
    ((300, 1024, 7), "bf16 f16"), ((300, 1023, 7), "bf16 f16"), ((270, 2040, 100), "bf16 f16"), ((270, 2043, 100), "bf16 f16"),
    ((260, 1032, 0), "f32"), ((5, 510, 2), "f32"), ((5, 2048, 2), "f32"),
    ((5, 7001, 2), "bf16 f16 f32"), ((5, 13001, 2), "bf16 f16 f32"),
]
ALL_NORMS = [(size, dt, kind) for size, types in NORMS for dt in types.split() for kind in ("rms", "layer")]


@pytest.mark.parametrize("size,dt,kind", ALL_NORMS, ids=["%s-%s-%s" % ("x".join(map(str, s)), d, k) for s, d, k in ALL_NORMS])
def test_block_norm_kernel(engine, size, dt, kind):
    T, d, rpg = size
    norm_case(engine, T, d, dt, kind, rpg, seed=T + d)
