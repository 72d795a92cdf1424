"""No block of a cluster touches another's shared memory before that block has begun. Too early a store is undefined,
and whether one happens is up to the hardware's scheduling, so the order is read from the source; the launches that
start clusters on a busy GPU are a second look."""
import math
import os
import random
import re

import pytest

from .conftest import ROOT
from .step_util import sample_exact

KERNELS = os.path.join(ROOT, "irptx_b200", "csrc", "kernels")


@pytest.fixture(autouse=True)
def _reference_core_for_gpu_tests():
    """These tests compare with definitions, not with the reference core."""


def body(name, head):
    """The function that begins with `head`, up to the closing brace in the first column, without comments."""
    text = open(os.path.join(KERNELS, name)).read()
    at = text.index(head)
    return re.sub(r"//[^\n]*", "", text[at:text.index("\n}\n", at)])


def test_the_draw_waits_for_its_cluster_before_the_first_exchange():
    s = body("sample.cu", "void smp_body(")
    remote = [m.start() for m in re.finditer(r"\bsmp_(post|find|st32|st64|ld32|add32|hand_over|resolve|among|cluster_sync)\b", s)]
    assert s.count("cluster_arrive();") == 1 and s.count("cluster_wait();") == 1
    assert s.index("cluster_arrive();") < s.index("cluster_wait();") < min(remote)
    assert "return" not in s[:s.index("cluster_wait();")]            # every thread arrives


@pytest.mark.parametrize("name,remote", [("gemm.cu", r"\bcluster_addr\("), ("matvec4.cu", r"\bcluster_addr\(")])
def test_the_products_wait_for_their_clusters(name, remote):
    text = re.sub(r"//[^\n]*", "", open(os.path.join(KERNELS, name)).read())
    for k in re.split(r"\n}\n", text):
        uses = [m.start() for m in re.finditer(remote, k)]
        if uses and "cluster_rank()" in k:
            assert "cluster_sync();" in k[:uses[0]]


@pytest.mark.gpu
def test_draws_that_begin_on_a_busy_gpu(cuda, irx):
    """Clusters of eight blocks, short rows, begun while other work comes and goes on the GPU."""
    torch = cuda
    gen, rnd = torch.Generator(device="cuda").manual_seed(1), random.Random(1)
    n, rows = 17001, 6
    settings = [(1.0, rnd.choice([0, 40]), rnd.choice([1.0, 0.9]), 0.0, rnd.random()) for _ in range(rows)]
    x = torch.empty(rows, n, device="cuda").normal_(0.0, 2.0, generator=gen)
    cols = list(zip(*settings))
    dev = [torch.tensor(c, dtype=torch.int32 if i == 1 else torch.float32, device="cuda") for i, c in enumerate(cols)]
    plan = irx.sample(rows, n, logprob=True)
    f32 = [tuple(torch.tensor(v, dtype=torch.float32).item() if j != 1 else v for j, v in enumerate(s)) for s in settings]
    want = [sample_exact(torch, x[i], *s) for i, s in enumerate(f32)]
    busy = torch.cuda.Stream()
    a = torch.empty(1 << 22, device="cuda").normal_(generator=gen)
    b = torch.empty_like(a)
    outs = []
    torch.cuda.synchronize()
    for i in range(200):
        with torch.cuda.stream(busy):
            for _ in range(i % 5):
                torch.mul(a[: 1 << (10 + i % 12)], 1.0001, out=b[: 1 << (10 + i % 12)])
        token, lp = torch.full((rows,), -7, dtype=torch.int32, device="cuda"), torch.full((rows,), 7.0, device="cuda")
        plan.launch([x] + dev + [token, lp])
        outs.append((token, lp))
    torch.cuda.synchronize()
    irx.check()
    for token, lp in outs:
        assert token.tolist() == [w for w, _ in want]
        assert all(math.isclose(p, w, rel_tol=2.0 ** -23, abs_tol=2.0 ** -24) for p, (_, w) in zip(lp.tolist(), want))
