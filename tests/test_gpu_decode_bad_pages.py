"""Decode over a table with entries that name no page: their keys are left out, as keys outside the mask are,
and the launch is reported; the other keys, rows and sequences are not touched."""
import math

import pytest

from .serving_util import Paged
from .test_gpu_serving import _reference_core_for_gpu_tests  # noqa: F401

pytestmark = pytest.mark.gpu


def reported(irx):
    with pytest.raises(irx.IrxError) as e:
        irx.check()
    assert e.value.code == 93


@pytest.mark.parametrize("dtype,shift", [("bf16", 0), ("f32", 0), ("bf16", 1)])
@pytest.mark.parametrize("heads,kv,d,page,order", [(2, 2, 64, 16, "head"), (24, 2, 64, 5, "token"), (8, 2, 128, 16, "token"),
                                                   (12, 1, 128, 64, "head"), (6, 2, 80, 8, "head"), (4, 1, 256, 16, "head")])
@pytest.mark.parametrize("window,sinks", [(0, 0), (150, 9)])
def test_keys_of_bad_pages_are_left_out(cuda, irx, dtype, shift, heads, kv, d, page, order, window, sinks):
    lens = (1, 300, 77, 2100, 130)
    c = Paged(cuda, irx, dtype, heads, kv, d, page, lens, order=order, window=window, sinks=sinks, shift=shift)
    c.launch()
    irx.check()
    whole = c.out.clone()
    for row, entries, bad in ((1, (0,), -1), (1, (299 // page,), c.cache.pages), (3, (2, 3, 2000 // page, 2099 // page), 10 ** 9),
                              (3, tuple(range(0, 2100 // page, 2)), -(1 << 31))):
        keep = c.table.clone()
        for e in entries:
            c.table[row, e] = bad
        c.launch()
        seen = [j for j in c.visible(row) if j // page not in entries]
        if len(seen) < len(c.visible(row)):
            reported(irx)
        irx.check()
        assert seen
        c.hold(row, seen)
        for b in range(len(lens)):
            assert b == row or cuda.equal(c.out[b], whole[b])
        c.table.copy_(keep)


@pytest.mark.parametrize("dtype,d", [("bf16", 64), ("bf16", 128), ("bf16", 256), ("f32", 64), ("f32", 128), ("f32", 256)])
def test_a_row_with_no_key_left_is_nan(cuda, irx, dtype, d):
    """A sequence that has tokens, none of them in the cache: there is no softmax of nothing."""
    c = Paged(cuda, irx, dtype, 4, 2, d, 16, (40, 700))
    c.table[0] = -1
    c.launch()
    reported(irx)
    assert bool(c.out[0].isnan().all()) and bool((c.lse[0] == -math.inf).all())
    c.hold(1)
