"""Descriptors of the serving operators that no memory can hold or that would read and write outside it."""
import pytest

from .test_serving import cache, refused


@pytest.mark.parametrize("order", ["head", "token"])
def test_three_zero_strides_are_an_overlap(irx, order):
    """As every other stride that lays rows over each other (a packed cache is strides=None)."""
    def build(**k):
        c = cache(irx, order=order, strides=(0, 0, 0), **k)
        return irx.decode(c, 2 * c.heads), irx.kv_append(c, 3), irx.kv_copy(c, 2)
    for k in ({}, dict(pages=1), dict(heads=1), dict(page_size=1), dict(pages=1, heads=1), dict(heads=1, page_size=1)):
        refused(irx, 41, build, **k)
    for p in build(pages=1, heads=1, page_size=1):        # one row
        assert max(a.elems for a in p.args if a.name in ("k", "k_pool", "k_pools")) >= 64


@pytest.mark.parametrize("strides", [(), (0, 0), (0, 0, 0, 0)])
def test_strides_are_three_numbers(irx, strides):
    refused(irx, 42, cache, irx, strides=strides)
