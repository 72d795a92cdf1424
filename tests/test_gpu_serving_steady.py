"""Decode and matvec4 with far more work than resident blocks, where their pipelines are in steady state: rings
that wrap, shares of a block that pass from one unit to the next, units that many blocks join, and for the
products runs of scales that hand over to the next. Against the definitions in 64 bits on the GPU."""
import pytest

from .serving_util import Packed, Paged
from .test_gpu_serving import _reference_core_for_gpu_tests  # noqa: F401

pytestmark = pytest.mark.gpu


def ragged(n, hi, lo=1):
    return tuple(lo + int((i * 0.6180339887498949) % 1.0 * (hi - lo)) for i in range(n))


# a long sequence between ragged ones (its join goes past one step, and does not begin at block 0); many units
# shorter than a block's share; windows over ragged lengths
LENS = {"long": (ragged(6, 3000) + (0, 60013, 1) + ragged(5, 2900), 0, 0),
        "short": ((5, 0, 64) + ragged(190, 400) + (0, 1), 0, 0),
        "window": (ragged(90, 3000) + (0, 701), 700, 5)}

# every kernel: padded head size 64, 128 and 256, one and two blocks of rows, both bodies, whole rows and not
KERNELS = [("bf16", 3, 3, 64, 16, "token", 0), ("bf16", 36, 3, 64, 32, "head", 0), ("bf16", 12, 3, 128, 16, "head", 0),
           ("bf16", 27, 3, 128, 64, "token", 0), ("bf16", 6, 3, 80, 8, "head", 0), ("bf16", 12, 3, 256, 16, "head", 0),
           ("bf16", 36, 3, 256, 16, "head", 0), ("f32", 3, 3, 64, 16, "head", 0), ("f32", 24, 3, 64, 5, "token", 0),
           ("f32", 12, 3, 128, 16, "head", 0), ("f32", 24, 3, 128, 16, "token", 0), ("f32", 27, 3, 96, 16, "head", 0),
           ("f32", 12, 3, 256, 32, "head", 0), ("f32", 18, 3, 256, 16, "head", 0), ("bf16", 12, 3, 128, 16, "head", 1)]


@pytest.mark.parametrize("kind", list(LENS))
@pytest.mark.parametrize("dtype,heads,kv,d,page,order,shift", KERNELS)
def test_decode(cuda, irx, kind, dtype, heads, kv, d, page, order, shift):
    lens, window, sinks = LENS[kind]
    c = Paged(cuda, irx, dtype, heads, kv, d, page, lens, order=order, window=window, sinks=sinks, shift=shift)
    c.launch()
    irx.check()
    c.hold_all()
    out, lse = c.out.clone(), c.lse.clone()
    for _ in range(3):                                    # the same bits, from the workspace as a launch leaves it
        c.launch()
        irx.check()
        assert cuda.equal(c.out, out) and cuda.equal(c.lse, lse)


@pytest.mark.parametrize("m,n,k,group", [(1, 14337, 4096, 128), (13, 8193, 14336, 128), (4, 8193, 14336, 64), (16, 14337, 4128, 32),
                                         (2, 20001, 4096, 32), (6, 9000, 4160, 320), (40, 9000, 4128, 96), (3, 300, 14336, 14336)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("zeros", [False, True])
def test_matvec4(cuda, irx, dtype, zeros, m, n, k, group):
    p = Packed(cuda, irx, dtype, m, n, k, group, zeros)
    p.launch()
    irx.check()
    p.hold()
    y = p.y.clone()
    for _ in range(3):
        p.launch()
    irx.check()
    assert cuda.equal(p.y, y)
