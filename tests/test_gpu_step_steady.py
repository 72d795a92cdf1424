"""The operators around the cache in steady state and at the limits of their paths: more work than resident blocks, counts next
to what one block finishes alone, thresholds inside long runs, shards."""
import math
import random

import pytest

from .test_gpu_step import (_reference_core_for_gpu_tests, append_case, draw, draw_check, ints, normal, prompt_case,  # noqa: F401
                            prompt_check, prompt_run)
from .step_util import tdt

pytestmark = pytest.mark.gpu


# ---- rotary positions ----

@pytest.mark.parametrize("dtype,dim,rot", [("bf16", 128, 128), ("bf16", 72, 48), ("f32", 96, 64), ("f32", 128, 64)])
def test_rope_shards_are_the_whole(cuda, irx, dtype, dim, rot):
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = normal(torch, gen, (1003, 6, dim), dtype)
    pos = torch.arange(1003, dtype=torch.int32, device="cuda") * 7
    plan = irx.rope(1003, 6, dim, irx.rope_freqs(rot), dtype=dtype)
    a, b = torch.zeros_like(x), torch.zeros_like(x)
    plan.launch([x, pos, a])
    for r in range(3):
        plan.launch_shard(r, 3, [x, pos, b])
    irx.check()
    assert torch.equal(a, b)


def test_rope_append_shards_are_the_whole(cuda, irx):
    torch = cuda
    c = append_case(torch, irx, "bf16", "token", False, 8, 2, 128, 64, 16, 3, True, False, seed=9)
    seq, pos = ints(torch, [s for s, _ in c["places"]]), ints(torch, [p for _, p in c["places"]])
    got = []
    for n in (1, 4):
        out = torch.zeros(c["n"], 8, 128, dtype=torch.bfloat16, device="cuda")
        pools = [t.clone() for t in c["pools"]]
        for r in range(n):
            c["plan"].launch_shard(r, n, [c["q"], c["k"], c["v"], seq, pos, c["table"], out] + pools)
        got.append([out] + pools)
    irx.check()
    assert all(torch.equal(a, b) for a, b in zip(*got))


# ---- attention over packed prompts ----

@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads,kv,d,lens,window,sinks", [
    (16, 16, 64, [1500, 900, 33, 700], 0, 0), (16, 4, 128, [2100, 40, 1300], 0, 0), (8, 8, 256, [1400, 700, 90], 0, 0),
    (16, 1, 256, [300, 150], 100, 4), (16, 16, 64, [1500, 900, 33], 300, 70), (32, 8, 128, [1200, 500], 130, 200)])
def test_prompt_more_units_than_blocks(cuda, irx, dtype, heads, kv, d, lens, window, sinks):
    c = prompt_case(cuda, irx, dtype, heads, kv, d, lens, window=window, sinks=sinks, behind=1)
    prompt_check(cuda, c, *prompt_run(cuda, irx, c))


@pytest.mark.parametrize("dtype,d", [("f32", 64), ("bf16", 128), ("bf16", 256)])
def test_prompt_hundreds_of_sequences(cuda, irx, dtype, d):
    rnd = random.Random(d)
    c = prompt_case(cuda, irx, dtype, 4, 2, d, [rnd.choice([0, 0, 1, 3, 64, 65, 129]) for _ in range(400)], window=60, sinks=2)
    prompt_check(cuda, c, *prompt_run(cuda, irx, c))


def test_prompt_rows_depend_on_their_sequence_alone(cuda, irx):
    """The same sequence packed with others, in another place, gives the same bits."""
    torch = cuda
    for dtype, d in (("bf16", 128), ("bf16", 64), ("bf16", 256), ("f32", 64)):
        a = prompt_case(torch, irx, dtype, 4, 2, d, [300, 77], seed=3)
        b = prompt_case(torch, irx, dtype, 4, 2, d, [5, 77, 300, 1000], seed=4)
        sa, sb = a["starts"], b["starts"]
        for x in "qkv":
            b[x][sb[2]:sb[3]] = a[x][sa[0]:sa[1]]
            b[x][sb[1]:sb[2]] = a[x][sa[1]:sa[2]]
        (oa, la), (ob, lb) = prompt_run(torch, irx, a), prompt_run(torch, irx, b)
        assert torch.equal(oa[:300], ob[sb[2]:sb[3]]) and torch.equal(oa[300:], ob[sb[1]:sb[2]])
        assert torch.equal(la[:300], lb[sb[2]:sb[3]]) and torch.equal(la[300:], lb[sb[1]:sb[2]])


# ---- the draw ----

@pytest.mark.parametrize("dtype,n", [("f32", 60001), ("bf16", 60001), ("f32", 450003), ("bf16", 850001)])
def test_sample_large_counts(cuda, irx, dtype, n):
    """top-k past what one block finishes alone, with and without the other filters; the longest rows are read again
    for each pass."""
    torch = cuda
    gen, rnd = torch.Generator(device="cuda").manual_seed(n), random.Random(n)
    settings = [(rnd.choice([0.7, 1.0, 3.0]), k, p, m, rnd.random()) for k in (1023, 1024, 1025, 5000, n - 1) for p, m in ((1.0, 0.0), (0.7, 0.0), (0.97, 0.001))]
    draw_check(torch, irx, normal(torch, gen, (len(settings), n), dtype, 2.0), settings)


@pytest.mark.parametrize("hot", [1, 1000, 1023, 1024, 1025, 1026, 3000])
def test_sample_counts_next_to_the_few(cuda, irx, hot):
    """`hot` equal logits above a spread of others, so that the filters end in or right below them."""
    torch = cuda
    gen, rnd = torch.Generator(device="cuda").manual_seed(hot), random.Random(hot)
    x = normal(torch, gen, (24, 9001), "f32", 1.0).clamp_max(2.0)
    for r in range(24):
        x[r, torch.randperm(9001, generator=gen, device="cuda")[:hot]] = 4.0
    settings = [(0.5, k, p, 0.0, rnd.random()) for k in (0, hot - 1, hot, hot + 1, 2 * hot, 1024) for p in (1.0, 0.3, 0.9, 0.999)]
    draw_check(torch, irx, x, settings)


def test_sample_flat_and_steep_rows(cuda, irx):
    """Rows whose cells are few or crowded: tiny spreads, huge ones, steps, one token far above the rest."""
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(8)
    n = 30011
    base = torch.empty(n, device="cuda").normal_(generator=gen)
    rows = [base * 1e-6, base * 1e-3, base * 100, base * 1e6, base * 1e-38, torch.arange(n, device="cuda") * 1e-4, (base > 1).float() * 5 + base * 1e-4,
            base - 1e5, base + 1e6, torch.where(torch.arange(n, device="cuda") == 77, 50.0, base), -base.abs() - 1e30, -base.abs() * 1e37]
    for t in (0.01, 1.0, 100.0):
        for k, p, m in ((0, 0.5, 0.0), (0, 0.999, 0.0), (2000, 0.9, 0.0), (0, 1.0, 0.5), (30, 0.9, 0.1)):
            for u in (0.1, 0.85):
                draw_check(torch, irx, torch.stack(rows), [(t, k, p, m, u)] * len(rows))


@pytest.mark.parametrize("rows", [1, 4, 48])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_sample_ends_among_equal_logits(cuda, irx, dtype, rows):
    """top-p alone ends inside 700 equal logits below 3000 others: too many for one block to finish, few enough to be gathered,
    and held by every block of the row. Where the running sum ends is half a token's weight away from the next one."""
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(rows)
    n, x = 20011, torch.full((20011,), -30.0, device="cuda")
    place = torch.randperm(n, generator=gen, device="cuda")
    x[place[:3000]] = torch.empty(3000, device="cuda").uniform_(1.2, 1.8, generator=gen)
    x[place[3000:3700]] = 1.0
    x = x.to(tdt(torch, dtype))
    e = torch.exp(x.double() - x.double().max())
    above, one = float(e[place[:3000]].sum()), float(e[place[3000]])
    for kept in (0.5, 99.5, 350.5, 699.5):
        p = (above + kept * one) / float(e.sum())
        draw_check(torch, irx, x.expand(rows, n).contiguous(), [(1.0, 0, p, 0.0, (i + 0.45) / rows) for i in range(rows)])


def test_sample_many_short_rows(cuda, irx):
    torch = cuda
    gen, rnd = torch.Generator(device="cuda").manual_seed(9), random.Random(9)
    settings = [(rnd.choice([0.0, 0.5, 1.0]), rnd.choice([0, 3, 40]), rnd.choice([1.0, 0.8]), rnd.choice([0.0, 0.1]), rnd.random()) for _ in range(900)]
    draw_check(torch, irx, normal(torch, gen, (900, 301), "bf16", 2.0), settings)


def test_sample_does_not_depend_on_the_launch(cuda, irx):
    """A row alone (a cluster of eight blocks) and among many (of one or two): the same token and the same bits."""
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(10)
    x = normal(torch, gen, (200, 40000), "f32", 2.0)
    settings = [(0.9, 0 if i % 2 else 60, 0.9 if i % 3 else 1.0, 0.0, (i + 0.5) / 200) for i in range(200)]
    token, lp = draw(torch, irx, x, settings)
    for i in range(0, 200, 17):
        t, l = draw(torch, irx, x[i:i + 1], settings[i:i + 1])
        assert t == token[i:i + 1] and l == lp[i:i + 1]


def test_a_captured_draw_reads_what_changed(cuda, irx):
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(11)
    x = normal(torch, gen, (4, 20000), "f32", 2.0)
    dev = [torch.full((4,), v, device="cuda") for v in (1.0, 1.0, 0.0, 0.5)]
    k, token = ints(torch, [0] * 4), ints(torch, [0] * 4)
    plan = irx.sample(4, 20000)
    args = [x, dev[0], k, dev[1], dev[2], dev[3], token]
    plan.launch(args)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        plan.launch(args)
    for i in range(6):
        x.copy_(normal(torch, gen, x.shape, "f32", 2.0))
        settings = [(0.5 + i / 8, 10 * i, 1.0 - i / 16, i / 64, (i + r) / 11) for r in range(4)]
        for d, col in zip(dev, (0, 2, 3, 4)):
            d.copy_(torch.tensor([s[col] for s in settings]))
        k.copy_(ints(torch, [s[1] for s in settings]))
        g.replay()
        irx.check()
        assert token.tolist() == draw(torch, irx, x, settings)[0]
    del g
