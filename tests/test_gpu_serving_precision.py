"""Decode's softmax weights and matvec4's f32 tokens carry the bits that they are stated to carry: inputs whose
results show nothing but the roundings in between."""
import pytest

from .serving_util import Packed, Paged
from .test_gpu_serving import _reference_core_for_gpu_tests  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv,d,page,n", [(8, 8, 64, 16, 38), (4, 4, 128, 16, 38), (4, 4, 256, 8, 38), (16, 1, 64, 16, 150),
                                               (4, 4, 128, 16, 600)])
def test_weights_of_values_that_are_all_one(cuda, irx, heads, kv, d, page, n):
    """The output is 1 up to the weights' error, which is below a quarter of bf16's step there (2^-8): 1 itself.
    Weights cut to 8 bits lose 2^-8.5 on average."""
    c = Paged(cuda, irx, "bf16", heads, kv, d, page, (n,))
    c.v.fill_(1.0)
    c.launch()
    irx.check()
    assert bool((c.out == 1.0).all())


@pytest.mark.parametrize("heads,d,page,n", [(8, 64, 16, 38), (4, 128, 16, 38), (4, 256, 8, 38), (8, 64, 16, 101)])
def test_weights_of_values_that_cancel(cuda, irx, heads, d, page, n):
    """Values of -1 and 1, and two keys whose values bring the sum to about 0, so that the output's rounding is
    far below the weights'. Weights rounded once to 8 bits are off by 2^-10.3 each, 2^-13 of 38."""
    c = Paged(cuda, irx, "bf16", heads, heads, d, page, (n,), qmul=0.25)
    for h in range(heads):
        for j in range(n):
            c.put_value(0, j, h, cuda.where(c.values[0][j, h].float() > 0, 1.0, -1.0) if j < n - 2 else cuda.zeros(d, device="cuda"))
        for j in (n - 2, n - 1):                          # coarse, then what its rounding left
            part, _, _, _ = c.exact(0)
            p = cuda.softmax(c.scale * (c.keys[0][:, h].double() @ c.q[0, h].double()), 0)[j]
            c.put_value(0, j, h, -part[h] / p)
    c.launch()
    irx.check()
    out, _, spread, _ = c.exact(0)
    assert bool((out.abs() < 2.0 ** -14 * spread).all())
    c.hold(0)


@pytest.mark.parametrize("m,n,k,group", [(1, 130, 4096, 128), (5, 64, 1024, 64), (3, 40, 992, 32), (2, 9, 77, 11)])
def test_f32_tokens_to_their_last_bit(cuda, irx, m, n, k, group):
    """Weights and scales of 1 and tokens of 2 - 2^-23: each of the three parts has a sum that f32 holds, the sum
    of the three rounds twice. On the path for any size each of a lane's k / 32 additions rounds, and five more."""
    import torch
    q = torch.full((n, k), 9, dtype=torch.uint8, device="cuda")
    p = Packed(torch, irx, "f32", m, n, k, group, False, x=torch.full((m, k), 2.0 - 2.0 ** -23, device="cuda"), q=q,
               s=torch.ones(n, -(-k // group), device="cuda"))
    p.launch()
    irx.check()
    want = k * (2.0 - 2.0 ** -23)
    roundings = 2 if k % 32 == 0 and group % 32 == 0 else k / 32 + 5
    assert bool(((p.y.double() - want).abs() <= roundings * 2.0 ** -24 * want).all())


@pytest.mark.parametrize("m,n,k,group", [(1, 130, 4096, 128), (9, 64, 512, 64), (13, 40, 992, 32)])
def test_f32_tokens_and_weights_of_one_sign(cuda, irx, m, n, k, group):
    """No cancelling: what a part of the tokens would lose adds up."""
    gen = cuda.Generator(device="cuda").manual_seed(2)
    p = Packed(cuda, irx, "f32", m, n, k, group, True, x=cuda.rand(m, k, generator=gen, device="cuda") + 1.0)
    p.z.zero_()
    p.launch()
    irx.check()
    p.hold()
