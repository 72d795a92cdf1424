"""Prompt attention with a scale of 0 or next to it over large queries and keys: 0 weighs every key the same, and a small scale
is that scale."""
import math

import pytest

from .test_gpu_step import _reference_core_for_gpu_tests, prompt_case, prompt_check, prompt_run  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("scale", [0.0, -0.0, 2.0 ** -124, -(2.0 ** -124), 2.0 ** -122, 2.0 ** -130, 2.0 ** -149])
@pytest.mark.parametrize("heads,kv,d,window,sinks", [(4, 1, 64, 0, 0), (2, 2, 128, 70, 3), (3, 1, 80, 0, 0), (2, 1, 256, 0, 0), (2, 1, 33, 0, 0)])
def test_small_scales_of_large_scores(cuda, irx, dtype, scale, heads, kv, d, window, sinks):
    """Queries and keys around 2^60 (sums of d products up to 2^127 stay in f32): scores of a few units at 2^-124."""
    c = prompt_case(cuda, irx, dtype, heads, kv, d, [300, 17, 140], window=window, sinks=sinks, lead=2, behind=3, scale=scale, std=2.0 ** 59)
    c["v"].mul_(2.0 ** -59)
    prompt_check(cuda, c, *prompt_run(cuda, irx, c))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_a_scale_of_zero_is_the_mean(cuda, irx, dtype, d):
    torch = cuda
    n = 200
    c = prompt_case(torch, irx, dtype, 2, 1, d, [n], scale=0.0, std=2.0 ** 60)
    c["v"][:] = (torch.arange(n, device="cuda") % 5)[:, None, None].to(c["v"].dtype)
    out, lse = prompt_run(torch, irx, c)
    mean = torch.cumsum(torch.arange(n, device="cuda", dtype=torch.float64) % 5, 0) / torch.arange(1, n + 1, device="cuda")
    # weights of 1, whole sums of 0 to 4 in f32 and one division; on the matrix path some weights are 7.5e-5 off in the row's sum
    off = 2.0 ** -8 + 1e-4 if dtype == "bf16" else 2.0 ** -22
    assert bool(((out.double() - mean[:, None, None]).abs() <= off * mean[:, None, None]).all())
    assert bool(((lse.double() - torch.log(torch.arange(1, n + 1, device="cuda").double())[:, None]).abs() <= (1e-4 if dtype == "bf16" else 0.0) + 2.0 ** -20).all())
    assert math.isfinite(float(lse.max()))
