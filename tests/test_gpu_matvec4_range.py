"""4-bit products whose tokens are near the ends of the range: a group's sum before its scale is larger than
any result, and must not overflow where the result does not."""
import pytest

from .serving_util import Packed
from .test_gpu_serving import _reference_core_for_gpu_tests  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("m,n,k,group", [(1, 130, 512, 128), (9, 40, 512, 128), (2, 64, 1024, 64), (3, 33, 96, 32), (12, 16, 640, 32),
                                         (1, 9, 512, 512), (2, 8, 77, 11)])
@pytest.mark.parametrize("power", [127, 110, 0, -100])
def test_tokens_over_the_range(cuda, irx, dtype, zeros, m, n, k, group, power):
    """Tokens of 1 to 2 times 2^power, scales that bring the results near 1. The bound is that of any size."""
    gen = cuda.Generator(device="cuda").manual_seed(power + 200)
    mant = 1 + cuda.rand(m, k, generator=gen, device="cuda") * 0.98
    s = (cuda.rand(n, -(-k // group), generator=gen, device="cuda") + 0.1) * 2.0 ** -min(power, 110)
    p = Packed(cuda, irx, dtype, m, n, k, group, zeros, x=mant * 2.0 ** power, s=s)
    p.launch()
    irx.check()
    p.hold()
