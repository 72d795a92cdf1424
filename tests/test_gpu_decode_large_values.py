"""Decode over values near the top of bf16's range: a weight that is zero in f32 adds nothing, however large
its value."""
import math

import pytest

from .serving_util import Paged
from .test_gpu_serving import _reference_core_for_gpu_tests  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads,d", [(1, 64), (12, 64), (4, 128), (16, 128), (4, 256)])
def test_a_large_value_of_no_weight(cuda, irx, dtype, heads, d):
    """Scores of 0 for one key and -300 for the others: exp(-300) is 0 in f32 and 2^-432 of 2^120 in 64 bits.
    (70 values of 2^120 still have a sum in f32.)"""
    n = 70
    c = Paged(cuda, irx, dtype, heads, 1, d, 16, (n,), scale=1.0)
    unit = cuda.zeros(d, device="cuda")
    unit[0] = 1.0
    c.q.copy_(unit.expand_as(c.q))
    for j in range(n):
        c.put_key(0, j, 0, unit * (0.0 if j == 33 else -300.0))
        c.put_value(0, j, 0, cuda.full((d,), 1.0 if j == 33 else 2.0 ** 120 * (1 if j % 3 else -1), device="cuda"))
    c.launch()
    irx.check()
    assert bool((c.out == 1.0).all())


@pytest.mark.parametrize("heads,d", [(1, 64), (4, 128), (4, 256)])
def test_an_infinite_value_of_any_weight(cuda, irx, heads, d):
    """Weights whose 8 upper bits are all of them (1, 1/4) and one of 2^-72: infinity, not 0 times infinity."""
    for score in (0.0, -math.log(4.0), -50.0):
        c = Paged(cuda, irx, "bf16", heads, 1, d, 16, (40,), scale=1.0)
        unit = cuda.zeros(d, device="cuda")
        unit[0] = 1.0
        c.q.copy_(unit.expand_as(c.q))
        for j in range(40):
            c.put_key(0, j, 0, unit * (score if j == 20 else 0.0))
        c.put_value(0, 20, 0, cuda.full((d,), math.inf, device="cuda"))
        c.launch()
        irx.check()
        assert bool((c.out == math.inf).all())
