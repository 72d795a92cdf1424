"""A scale is held times log2(e): where f32 does not hold that, a plan is refused and no other scale takes its place."""
import pytest

from .test_step import cache, refused


@pytest.mark.parametrize("scale", [2.36e38, -2.36e38, 3.4028234663852886e38])
def test_scales_past_the_range_are_refused(irx, scale):
    refused(irx, 42, irx.prompt, 9, 2, 4, 2, 64, scale=scale)
    refused(irx, 42, irx.decode, cache(irx), 4, scale=scale)


@pytest.mark.parametrize("scale", [2.35e38, -2.35e38, 1e-45, 0.0])
def test_scales_within_it_are_taken(irx, scale):
    assert irx.prompt(9, 2, 4, 2, 64, scale=scale).family == "prompt"
    assert irx.decode(cache(irx), 4, scale=scale).family == "decode"
