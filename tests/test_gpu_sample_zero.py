"""The draw where a filter ends at a logit of 0.0 or next to it: with both zeros, all or some of the tokens of that
number kept, and rows whose largest logit becomes 0.0 on the way (infinite ones, the type's lowest)."""
import math
import random

import pytest

from .step_util import tdt
from .test_gpu_step import _reference_core_for_gpu_tests, draw_check, normal  # noqa: F401

pytestmark = pytest.mark.gpu


def zeros(torch, count, both):
    x = torch.zeros(count, device="cuda")
    if both:
        x[::3] = -0.0
    return x


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("both", [False, True])
@pytest.mark.parametrize("hot,n", [(700, 1500), (1, 3000), (2000, 3000), (700, 20011), (1024, 20011), (1025, 20011), (3000, 20011), (6000, 60001)])
def test_all_zeros_kept_of_a_row_below_them(cuda, irx, dtype, both, hot, n):
    """`hot` zeros on top of minus infinities, or of numbers further down: filters end inside and right below them."""
    torch = cuda
    gen, rnd = torch.Generator(device="cuda").manual_seed(hot + n), random.Random(hot + n)
    for rest in (-math.inf, -1.0, None):
        x = torch.full((12, n), rest if rest is not None else 0.0, device="cuda")
        if rest is None:
            x = -normal(torch, gen, (12, n), "f32", 2.0).abs() - 0.25
        for r in range(12):
            x[r, torch.randperm(n, generator=gen, device="cuda")[:hot]] = zeros(torch, hot, both)
        share = 1.0 / max(1.0, float(torch.exp(x[0].double()).sum()))      # of one zero
        p = min((hot - 0.5) * share, 0.99999994)
        settings = [(1.0, k, q, 0.0, rnd.random()) for k in (0, hot, hot - 1 or 1, hot + 1) for q in (1.0, p, p / 2)]
        draw_check(torch, irx, x.to(tdt(torch, dtype)), settings)


@pytest.mark.parametrize("rows", [1, 4, 48])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("both", [False, True])
def test_top_p_ends_among_zeros(cuda, irx, dtype, rows, both):
    """As among equal logits elsewhere: 700 zeros under 3000 others, a row in one, four and eight blocks; kept half a
    token's weight away from the next."""
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(rows)
    n, x = 20011, torch.full((20011,), -30.0, device="cuda")
    place = torch.randperm(n, generator=gen, device="cuda")
    x[place[:3000]] = torch.empty(3000, device="cuda").uniform_(0.2, 0.8, generator=gen)
    x[place[3000:3700]] = zeros(torch, 700, both)
    x = x.to(tdt(torch, dtype))
    e = torch.exp(x.double() - x.double().max())
    above, one = float(e[place[:3000]].sum()), float(e[place[3000]])
    for kept in (0.5, 99.5, 350.5, 699.5):
        p = (above + kept * one) / float(e.sum())
        draw_check(torch, irx, x.expand(rows, n).contiguous(), [(1.0, 0, p, 0.0, (i + 0.45) / rows) for i in range(rows)])
    for k in (3001, 3350, 3699, 3700, 3701):
        draw_check(torch, irx, x.expand(rows, n).contiguous(), [(1.0, k, 1.0 if i % 2 else 0.9999, 0.0, (i + 0.45) / rows) for i in range(rows)])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("value", [0.0, -0.0, math.inf, "low"])
@pytest.mark.parametrize("n", [1025, 2000, 9000, 30000])
def test_rows_of_one_number(cuda, irx, dtype, value, n):
    """top-p above 1 - 1/n keeps all; whole rows of zeros, of infinities, of the type's lowest number."""
    torch = cuda
    v = torch.finfo(tdt(torch, dtype)).min if value == "low" else value
    ps = [1.0 - 0.5 / n, 1.0 - 1.5 / n, 0.5 + 0.25 / n, 1.0]
    settings = [(0.8, k, p, 0.0, (int(n * f) + 0.45) / n) for k in (0, n - 1, n // 2) for p in ps for f in (0.0, 0.37, 0.9)]
    draw_check(torch, irx, torch.full((len(settings), n), v, device="cuda").to(tdt(torch, dtype)), settings)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_infinite_logits_in_thousands(cuda, irx, dtype):
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(2)
    n, hot = 20011, 1500
    settings = [(0.8, k, p, 0.0, (int(200 * f) + 0.45) / hot) for k in (0, hot, hot + 7, hot - 1, 1100) for p in (1.0, 1.0 - 0.5 / hot, 0.6 + 0.1 / hot) for f in (0.1, 0.9)]
    x = normal(torch, gen, (len(settings), n), dtype, 2.0)
    for r in range(len(settings)):
        x[r, torch.randperm(n, generator=gen, device="cuda")[:hot]] = math.inf
    draw_check(torch, irx, x, settings)


@pytest.mark.parametrize("dtype,unit,t", [("f32", 2.0 ** -149, 1e-42), ("f32", 2.0 ** -149, 1e-44), ("bf16", 2.0 ** -133, 1e-39), ("f32", 2.0 ** -126, 1e-37)])
@pytest.mark.parametrize("n", [3000, 40011])
def test_thresholds_among_the_smallest_numbers(cuda, irx, dtype, unit, t, n):
    """Logits a few of the smallest steps around zero, zeros many times among them, at temperatures of that size."""
    torch = cuda
    gen, rnd = torch.Generator(device="cuda").manual_seed(n), random.Random(n)
    for low, high, none in ((-3000, 0, 0.3), (-50, 50, 0.1), (-4, 1, 0.3), (-2000, 2000, 0.02)):
        x = torch.randint(low, high + 1, (36, n), generator=gen, device="cuda").double() * unit
        x[torch.rand(36, n, generator=gen, device="cuda") < none] = 0.0
        x = x.float().to(tdt(torch, dtype))
        settings = [(t, rnd.choice([0, 0, 5, n // 50, n // 4, n // 2, n - 3]), rnd.choice([1.0, 0.2, 0.7, 0.9, 0.99]), rnd.choice([0.0, 0.0, 0.4]), rnd.random())
                    for _ in range(36)]
        draw_check(torch, irx, x, settings)
