"""Prompt attention over values near the top of the range and infinite ones, seen with weights that vanish: a weight of
zero adds nothing, however large its value."""
import math

import pytest

from .step_util import tdt
from .test_gpu_step import _reference_core_for_gpu_tests, ints  # noqa: F401

pytestmark = pytest.mark.gpu


def attend(torch, irx, dtype, heads, d, n, scores, values, window=0, scale=1.0):
    """One sequence of n tokens whose key j has the score `scores`[j] for every query. Returns out, lse."""
    td = tdt(torch, dtype)
    q, k = torch.zeros(n, heads, d, device="cuda"), torch.zeros(n, 1, d, device="cuda")
    q[..., 0] = 1.0
    k[:, 0, 0] = torch.tensor(scores, device="cuda")
    v = torch.tensor(values, device="cuda")[:, None, None].expand(n, 1, d)
    out, lse = torch.zeros(n, heads, d, dtype=td, device="cuda"), torch.zeros(n, heads, device="cuda")
    irx.prompt(n, 1, heads, 1, d, dtype=dtype, scale=scale, window=window, lse=True).launch(
        [q.to(td), k.to(td), v.to(td).contiguous(), ints(torch, [0, n]), out, lse])
    irx.check()
    return out, lse


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads,d", [(1, 64), (4, 128), (3, 80), (2, 256), (1, 33)])
@pytest.mark.parametrize("window,at", [(0, 0), (0, 33), (0, 300), (400, 150)])
def test_a_large_value_of_no_weight(cuda, irx, dtype, heads, d, window, at):
    """Scores of 0 for one key and -300 for the others, whose weights are 0 in f32: rows that see the one are its value.
    (700 values of 2^118 still have a sum in f32.) The one's weight is 1, on the matrix path within 7.5e-5, the largest
    error of its cubic: log(1 - 7.5e-5) is above -7.6e-5; 1 over it rounds to 1 in bf16, whose half step is 2^-9 below 1."""
    n = 700
    values = [1.0 if j == at else 2.0 ** 118 * (1 if j % 3 else -1) for j in range(n)]
    out, lse = attend(cuda, irx, dtype, heads, d, n, [0.0 if j == at else -300.0 for j in range(n)], values, window)
    see = slice(at, at + window if window else n)
    assert bool((out[see] == 1.0).all()) and bool((lse[see].abs() <= (7.6e-5 if dtype == "bf16" else 0.0)).all())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads,d", [(1, 64), (4, 128), (3, 80), (2, 256), (1, 33)])
@pytest.mark.parametrize("window,at", [(0, 5), (0, 130), (0, 400), (400, 150)])
@pytest.mark.parametrize("value", [math.inf, math.nan])
def test_an_infinite_value_shows_in_every_row_that_sees_it(cuda, irx, dtype, heads, d, window, at, value):
    """Key 0 has the score 0, the others -300: `value` stands behind a weight that vanishes, in tiles seen in part and in
    whole. Rows that see it are infinite or NaN, the others 1."""
    n = 700
    out, lse = attend(cuda, irx, dtype, heads, d, n, [0.0] + [-300.0] * (n - 1), [value if j == at else 1.0 for j in range(n)], window)
    see = cuda.zeros(n, dtype=cuda.bool, device="cuda")
    see[at:at + window if window else n] = True
    assert not bool(out[see].isfinite().any()) and bool((out[~see] == 1.0).all())
    assert bool(lse.isfinite().all())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads,d", [(1, 64), (4, 128), (3, 80), (2, 256), (1, 33)])
@pytest.mark.parametrize("step", [0.0, 5.5, 11.0, -5.5])
def test_values_times_keys_within_the_range(cuda, irx, dtype, heads, d, step):
    """300 values of 2^119 have a sum below 2^128. Scores that rise by 5.5 after every 128 keys (weights 245 times those before, which
    the running maximum may lag behind) leave it there: every row's result is the value."""
    n = 300
    out, lse = attend(cuda, irx, dtype, heads, d, n, [step * (j // 128) for j in range(n)], [2.0 ** 119] * n)
    # equal values: the weights' sum over itself, n + 2 roundings of 2^-24 in f32; on the matrix path weights 2^-9 and 1e-4 off and
    # the result's half step, 2^-9 below or at 2^119 and 2^-8 above
    off = 2.0 ** -8 + 2.0 ** -9 + 1e-4 if dtype == "bf16" else (n + 2) * 2.0 ** -24 * 2
    assert bool(((out.double() / 2.0 ** 119 - 1.0).abs() <= off).all()) and bool(lse.isfinite().all())
