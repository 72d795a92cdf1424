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


def test_products_past_64_bits_are_refused(irx):
    top, far = (1 << 31) - 1, 1 << 40
    one = cache(irx)
    refused(irx, 42, irx.kv_append, one, top, stride=far)
    refused(irx, 42, irx.decode, cache(irx, batch=1 << 29), 2, q_stride=far)
    refused(irx, 42, irx.decode, cache(irx, batch=top), (1 << 31) - 2)
    wide = cache(irx, heads=1, page_size=1, pages=2)
    refused(irx, 42, irx.kv_copy, cache(irx, heads=1 << 10, page_size=1 << 10, pages=2, head_dim=256), top, layers=1 << 22)
    for plan in (irx.kv_append(one, top, stride=1 << 28), irx.decode(cache(irx, batch=1 << 29), 2, q_stride=1 << 28),
                 irx.kv_copy(wide, top, layers=1 << 20)):
        assert all(0 < a.elems < 1 << 62 for a in plan.args)
