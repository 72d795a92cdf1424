"""The operators around the cache on a GPU against their definitions in 64 bits, at the sizes, layouts, masks and
settings where they can go wrong. Bounds: tests/step_util.py; drawn tokens have to be equal."""
import math
import random

import pytest

from .step_util import prompt_exact, rope_exact, sample_exact, tdt

pytestmark = pytest.mark.gpu
INF, NAN = math.inf, math.nan


@pytest.fixture(autouse=True)
def _reference_core_for_gpu_tests():
    """These operators have no counterpart in the reference, so its core is not needed here."""


def normal(torch, gen, shape, dtype, std=1.0):
    return (torch.empty(shape, device="cuda").normal_(generator=gen) * std).to(tdt(torch, dtype))


def ints(torch, v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def within(got, want, tol):
    bad = ~((got.double() - want).abs() <= tol) & ~((got.double() == want) | (got.isnan() & want.isnan()))
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[0].tolist(), float(got[bad][0]), float(want[bad][0]), float(tol[bad][0]))


# ---- rotary positions ----

@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("tokens,heads,dim,rot,extra", [(1, 1, 2, 2, 0), (3, 5, 64, 64, 0), (33, 40, 128, 128, 1024), (7, 3, 80, 20, 0),
                                                        (5, 2, 33, 32, 1), (2, 7, 96, 96, 8), (4, 9, 256, 256, 0), (6, 2, 256, 16, 24),
                                                        (9, 1, 128, 64, 3), (300, 8, 128, 128, 0), (2, 130, 64, 32, 0)])
@pytest.mark.parametrize("backward", [False, True])
def test_rope(cuda, irx, dtype, inter, tokens, heads, dim, rot, extra, backward):
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(tokens * dim + rot)
    wide = normal(torch, gen, (tokens, heads * dim + extra), dtype)
    x = wide[:, :heads * dim].unflatten(1, (heads, dim))
    pos = torch.randint(0, 1 << 20, (tokens,), generator=gen, device="cuda").to(torch.int32)
    pos[tokens // 2] = 0
    if tokens > 2:
        pos[1] = -1
    freqs = irx.rope_freqs(rot, base=5e5)
    ystride = heads * dim + extra
    y = torch.full((tokens, ystride), 7.0, dtype=x.dtype, device="cuda")
    plan = irx.rope(tokens, heads, dim, freqs, dtype=dtype, interleaved=inter, amplitude=1.25, backward=backward, x_stride=ystride, y_stride=ystride)
    plan.launch([x, pos, y[:, :heads * dim].unflatten(1, (heads, dim))])
    irx.check()
    want, tol = rope_exact(torch, x, pos, freqs, inter, 1.25, backward)
    live = pos >= 0
    got = y[:, :heads * dim].unflatten(1, (heads, dim))
    within(got[live], want[live], tol[live])
    assert torch.equal(got[live][..., rot:], x[live][..., rot:])
    assert bool((y[~live] == 7.0).all()) and bool((y[:, heads * dim:] == 7.0).all())
    # in place: the same bits, and nothing beside them
    before = wide.clone()
    plan.launch([x, pos, x])
    irx.check()
    assert torch.equal(x[live], got[live]) and torch.equal(wide[~live], before[~live])
    assert torch.equal(wide[:, heads * dim:], before[:, heads * dim:])


def test_rope_far_positions(cuda, irx):
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = normal(torch, gen, (6, 3, 64), "f32")
    pos = ints(torch, [0, 1, (1 << 24) + 1, (1 << 30) + 7, (1 << 31) - 2, (1 << 31) - 1])
    for freqs in (irx.rope_freqs(64), [1024.0, 3.0, 0.5]):
        y = torch.empty_like(x)
        irx.rope(6, 3, 64, freqs, dtype="f32").launch([x, pos, y])
        want, tol = rope_exact(torch, x, pos, freqs)
        within(y, want, tol)


def test_rope_gradient(cuda, irx):
    """backward against differences of the forward rotation: it is linear, so a difference is its derivative."""
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(2)
    freqs = irx.rope_freqs(24)
    for inter in (False, True):
        fwd = irx.rope(5, 2, 32, freqs, dtype="f32", interleaved=inter, amplitude=0.75)
        bwd = irx.rope(5, 2, 32, freqs, dtype="f32", interleaved=inter, amplitude=0.75, backward=True)
        pos = ints(torch, [3, 0, 1000, 77, 12345])
        x, g = normal(torch, gen, (5, 2, 32), "f32"), normal(torch, gen, (5, 2, 32), "f32")
        dx, a, b = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
        bwd.launch([g, pos, dx])
        for _ in range(4):
            e = normal(torch, gen, (5, 2, 32), "f32")
            fwd.launch([x + e, pos, a])
            fwd.launch([x - e, pos, b])
            slope = ((a.double() - b.double()) / 2 * g.double()).sum()
            # 320 products, each operand off by under 2^-20 of numbers of up to about 10
            assert abs(float(slope - (dx.double() * ((x + e).double() - (x - e).double()) / 2).sum())) < 320 * 100 * 2.0 ** -20


# ---- on the way into the cache ----

def append_case(torch, irx, dtype, order, inter, heads, kv, dim, rot, page, batch, fused, strided, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rnd = random.Random(seed)
    cols = 5
    pages = batch * cols + 3
    strides = None
    if strided:
        a, b = (kv, page) if order == "head" else (page, kv)
        strides = ((a * (b * (dim + 8) + 16)) + 8, b * (dim + 8) + 16, dim + 8)
    cache = irx.KvCache(dtype, kv, dim, page, pages, batch=batch, table_cols=cols, order=order, strides=strides)
    flat = [normal(torch, gen, (pages * cache.strides[0] + 8,), dtype) for _ in range(2)]
    pools = [f.as_strided(cache.shape, cache.strides + (1,)) for f in flat]
    table = torch.randperm(pages, generator=gen, device="cuda")[:batch * cols].to(torch.int32).reshape(batch, cols)
    places = [(s, p) for s in range(batch) for p in range(cols * page)]
    rnd.shuffle(places)
    places = places[:23] + [(0, -1), (batch + 5, -3)]
    n = len(places)
    if fused:
        rows = normal(torch, gen, (n, heads + 2 * kv, dim), dtype)
        q, k, v, stride = rows[:, :heads], rows[:, heads:heads + kv], rows[:, heads + kv:], (heads + 2 * kv) * dim
    else:
        q, k, v, stride = normal(torch, gen, (n, heads, dim), dtype), normal(torch, gen, (n, kv, dim), dtype), normal(torch, gen, (n, kv, dim), dtype), 0
    freqs = irx.rope_freqs(rot)
    plan = irx.rope_append(cache, n, heads, freqs, interleaved=inter, amplitude=1.5, stride=stride)
    return dict(cache=cache, flat=flat, pools=pools, table=table, places=places, q=q, k=k, v=v, freqs=freqs, plan=plan, n=n)


@pytest.mark.parametrize("dtype,order,inter,heads,kv,dim,rot,page,fused,strided", [
    ("bf16", "head", False, 8, 2, 128, 128, 16, True, False), ("bf16", "token", True, 4, 4, 64, 32, 8, False, True),
    ("f32", "head", True, 6, 3, 96, 96, 1, True, True), ("f32", "token", False, 2, 1, 33, 10, 5, False, False),
    ("bf16", "head", False, 7, 1, 80, 20, 24, True, False), ("bf16", "token", False, 32, 8, 256, 256, 64, True, True)])
def test_rope_append(cuda, irx, dtype, order, inter, heads, kv, dim, rot, page, fused, strided):
    torch = cuda
    c = append_case(torch, irx, dtype, order, inter, heads, kv, dim, rot, page, 3, fused, strided)
    seq, pos = ints(torch, [s for s, _ in c["places"]]), ints(torch, [p for _, p in c["places"]])
    out = torch.full((c["n"], heads, dim), 7.0, dtype=c["q"].dtype, device="cuda")
    before = [f.clone() for f in c["flat"]]
    c["plan"].launch([c["q"], c["k"], c["v"], seq, pos, c["table"], out] + c["pools"])
    irx.check()
    live = pos >= 0
    want, tol = rope_exact(torch, c["q"], pos, c["freqs"], inter, 1.5)
    within(out[live], want[live], tol[live])
    assert bool((out[~live] == 7.0).all())
    kw, kt = rope_exact(torch, c["k"], pos, c["freqs"], inter, 1.5)
    for i, (s, p) in enumerate(c["places"]):
        if p < 0:
            continue
        pg, sl = int(c["table"][s, p // page]), p % page
        got = [t[pg, :, sl] if order == "head" else t[pg, sl] for t in c["pools"]]
        within(got[0], kw[i], kt[i])
        assert torch.equal(got[1], c["v"][i])
        for t in got:                                    # put back what was there: nothing else may have changed
            t.fill_(0)
    for f, b, shape in zip(c["flat"], before, [c["cache"]] * 2):
        view = b.as_strided(shape.shape, shape.strides + (1,))
        for s, p in c["places"]:
            if p >= 0:
                pg, sl = int(c["table"][s, p // page]), p % page
                (view[pg, :, sl] if order == "head" else view[pg, sl]).fill_(0)
        assert torch.equal(f, b)


def test_rope_append_skips_and_reports_what_is_outside(cuda, irx):
    torch = cuda
    c = append_case(torch, irx, "bf16", "head", False, 4, 2, 64, 64, 16, 2, True, False)
    c["table"][1, 2], c["table"][0, 0] = -1, 10 ** 9
    seq, pos = ints(torch, [0, 1, 2, -1, 0, 1] + [0] * (c["n"] - 6)), ints(torch, [3, 40, 0, 0, 80, 0] + [-1] * (c["n"] - 6))
    out = torch.full((c["n"], 4, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    before = [f.clone() for f in c["flat"]]
    c["plan"].launch([c["q"], c["k"], c["v"], seq, pos, c["table"], out] + c["pools"])
    with pytest.raises(irx.IrxError) as e:
        irx.check()
    assert e.value.code == 93
    want, tol = rope_exact(torch, c["q"], pos, c["freqs"], False, 1.5)
    within(out[:6], want[:6], tol[:6])                   # the queries are turned all the same
    pg = int(c["table"][1, 0])
    for f, b, t in zip(c["flat"], before, c["pools"]):
        t[pg, :, 0] = b.as_strided(c["cache"].shape, c["cache"].strides + (1,))[pg, :, 0]
        assert torch.equal(f, b)
    irx.check()


def test_rope_append_in_place_equals_rope_and_kv_append(cuda, irx):
    torch = cuda
    c = append_case(torch, irx, "bf16", "head", False, 8, 2, 128, 128, 16, 3, True, False, seed=4)
    seq, pos = ints(torch, [s for s, _ in c["places"]]), ints(torch, [p for _, p in c["places"]])
    n, rows = c["n"], torch.cat([c["q"], c["k"], c["v"]], 1)
    turned = rows.clone()
    irx.rope(n, 10, 128, c["freqs"], amplitude=1.5, x_stride=12 * 128, y_stride=12 * 128).launch([rows[:, :10], pos, turned[:, :10]])
    pools = [t.clone() for t in c["pools"]]
    irx.kv_append(c["cache"], n, stride=12 * 128).launch([turned[:, 8:10], turned[:, 10:], seq, pos, c["table"]] + pools)
    irx.rope_append(c["cache"], n, 8, c["freqs"], amplitude=1.5, stride=12 * 128, out_stride=12 * 128).launch(
        [rows[:, :8], rows[:, 8:10], rows[:, 10:], seq, pos, c["table"], rows[:, :8]] + c["pools"])
    irx.check()
    assert torch.equal(rows[:, :8], turned[:, :8]) and all(torch.equal(a, b) for a, b in zip(pools, c["pools"]))


# ---- attention over packed prompts ----

def prompt_case(torch, irx, dtype, heads, kv, d, lens, window=0, sinks=0, lead=0, behind=0, scale=None, fused=True, seed=0, std=1.0, shift=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    starts = [lead]
    for n in lens:
        starts.append(starts[-1] + n)
    t = starts[-1] + behind
    wide = (heads + 2 * kv) * d
    flat = normal(torch, gen, (t * wide + shift,), dtype, std)
    rows = flat[shift:].view(t, heads + 2 * kv, d)
    rows[:lead] = NAN
    rows[starts[-1]:] = INF
    q, k, v = rows[:, :heads], rows[:, heads:heads + kv], rows[:, heads + kv:]
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    stride = wide if fused else 0
    plan = irx.prompt(t, len(lens), heads, kv, d, dtype=dtype, scale=scale, window=window, sinks=sinks, lse=True, q_stride=stride, kv_stride=stride)
    return dict(q=q, k=k, v=v, starts=starts, plan=plan, t=t, heads=heads, d=d, dtype=dtype, window=window, sinks=sinks,
                scale=d ** -0.5 if scale is None else scale)


def prompt_run(torch, irx, c, launch=None):
    out = torch.full((c["t"], c["heads"], c["d"]), 7.0, dtype=c["q"].dtype, device="cuda")
    lse = torch.full((c["t"], c["heads"]), 7.0, device="cuda")
    args = [c["q"], c["k"], c["v"], ints(torch, c["starts"]), out, lse]
    (launch or c["plan"].launch)(args)
    irx.check()
    return out, lse


def prompt_check(torch, c, out, lse):
    want, tol, wl, tl = prompt_exact(torch, c["q"], c["k"], c["v"], c["starts"], c["scale"], c["window"], c["sinks"], matrix=c["dtype"] == "bf16")
    a, b = c["starts"][0], c["starts"][-1]
    within(out[a:b], want[a:b], tol[a:b])
    within(lse[a:b], wl[a:b], tl[a:b])
    for x in (out, lse):
        assert bool((x[:a] == 7.0).all()) and bool((x[b:] == 7.0).all())


LENS = [[1], [1, 0, 2, 0], [64, 65, 63, 1], [127, 1, 128, 129], [300, 31, 33, 257], [0, 0, 5], [1000]]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("heads,kv,d", [(4, 1, 128), (2, 2, 64)])
def test_prompt_lengths(cuda, irx, dtype, lens, heads, kv, d):
    c = prompt_case(cuda, irx, dtype, heads, kv, d, lens, lead=3, behind=2)
    prompt_check(cuda, c, *prompt_run(cuda, irx, c))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads,kv,d", [(1, 1, 8), (3, 1, 16), (6, 2, 40), (7, 1, 64), (14, 2, 72), (8, 8, 80), (8, 1, 96), (16, 1, 128),
                                        (5, 1, 120), (2, 1, 136), (4, 2, 192), (4, 4, 256), (8, 1, 256), (130, 1, 16), (64, 1, 128), (3, 3, 33), (2, 1, 1), (4, 1, 250)])
def test_prompt_heads(cuda, irx, dtype, heads, kv, d):
    c = prompt_case(cuda, irx, dtype, heads, kv, d, [70, 5, 0, 150], behind=1, fused=d % 2 == 0)
    prompt_check(cuda, c, *prompt_run(cuda, irx, c))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 4), (64, 0), (100, 4), (128, 1), (129, 130), (200, 300), (250, 0), (10 ** 9, 5)])
@pytest.mark.parametrize("heads,kv,d", [(4, 1, 64), (1, 1, 128)])
def test_prompt_windows(cuda, irx, dtype, window, sinks, heads, kv, d):
    c = prompt_case(cuda, irx, dtype, heads, kv, d, [257, 1, 600, 64], window=window, sinks=sinks, behind=3)
    prompt_check(cuda, c, *prompt_run(cuda, irx, c))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0, 1e-6])
def test_prompt_scales(cuda, irx, dtype, scale):
    c = prompt_case(cuda, irx, dtype, 4, 2, 64, [200, 17], scale=scale)
    prompt_check(cuda, c, *prompt_run(cuda, irx, c))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_prompt_growing_scores(cuda, irx, dtype, d):
    """Keys whose scores grow along the sequence, so that the running maximum moves at every tile."""
    torch = cuda
    c = prompt_case(torch, irx, dtype, 2, 1, d, [700], scale=1.0)
    c["q"][:] = 0.25
    c["k"][:] = (torch.arange(700, device="cuda") / 8.0 / d)[:, None, None].to(c["k"].dtype)
    c["k"][350:360] = -30.0
    prompt_check(torch, c, *prompt_run(torch, irx, c))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (70, 3)])
@pytest.mark.parametrize("heads,kv,d", [(4, 1, 128), (2, 2, 64), (2, 1, 256)])
def test_prompt_hidden_values_have_no_effect(cuda, irx, dtype, window, sinks, heads, kv, d):
    """Infinities and NaN in values and keys that the mask hides from a row, in its own sequence."""
    torch = cuda
    c = prompt_case(torch, irx, dtype, heads, kv, d, [140, 300, 20], window=window, sinks=sinks)
    for at, x in ((139, INF), (140 + 299, NAN), (140 + 170, -INF), (140 + 100, INF), (140 + 2, INF), (459, NAN)):
        c["v"][at, 0, at % d] = x
    prompt_check(torch, c, *prompt_run(torch, irx, c))
    c = prompt_case(torch, irx, dtype, heads, kv, d, [140, 300, 20], window=window, sinks=sinks, seed=1)
    plain = prompt_run(torch, irx, c)
    for at in (139, 140 + 299, 459):                     # the last keys: only their own rows see them
        c["k"][at] = NAN
    out, lse = prompt_run(torch, irx, c)
    own = torch.zeros(c["t"], dtype=torch.bool, device="cuda")
    own[[139, 439, 459]] = True
    assert torch.equal(out[~own], plain[0][~own]) and torch.equal(lse[~own], plain[1][~own])
    assert bool(out[own].isnan().all())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 2)])
@pytest.mark.parametrize("heads,kv,d", [(4, 1, 128), (2, 2, 64), (2, 1, 256)])
def test_prompt_hidden_large_values_have_no_effect(cuda, irx, dtype, window, sinks, heads, kv, d):
    """The type's largest numbers in a token that the others do not see: their bits are those without it."""
    torch = cuda
    c = prompt_case(torch, irx, dtype, heads, kv, d, [190, 60], window=window, sinks=sinks)
    plain = prompt_run(torch, irx, c)
    for at in (189, 249):                                # the last tokens: only their own rows see them
        c["v"][at] = torch.finfo(c["v"].dtype).max
    if window:
        c["v"][5] = torch.finfo(c["v"].dtype).max         # seen by tokens 5 to 44
    out, lse = prompt_run(torch, irx, c)
    own = torch.zeros(c["t"], dtype=torch.bool, device="cuda")
    own[[189, 249]] = True
    if window:
        own[5:45] = True
    assert torch.equal(out[~own], plain[0][~own]) and torch.equal(lse, plain[1])


def test_prompt_reports_bad_starts(cuda, irx):
    torch = cuda
    c = prompt_case(torch, irx, "bf16", 4, 2, 64, [50, 60, 70])
    good = prompt_run(torch, irx, c)
    for bad in ([0, 50, 40, 180], [-1, 50, 110, 180], [0, 50, 110, 181], [0, 50, 2 ** 31 - 1, 180]):
        out = torch.full((c["t"], 4, 64), 7.0, dtype=torch.bfloat16, device="cuda")
        lse = torch.full((c["t"], 4), 7.0, device="cuda")
        c["plan"].launch([c["q"], c["k"], c["v"], ints(torch, bad), out, lse])
        with pytest.raises(irx.IrxError) as e:
            irx.check()
        assert e.value.code == 93
        for a, b in zip(bad, bad[1:]):
            if (a, b) in ((0, 50), (110, 180)):
                assert torch.equal(out[a:b], good[0][a:b])
    irx.check()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_prompt_unaligned_rows(cuda, irx, dtype):
    c = prompt_case(cuda, irx, dtype, 4, 2, 64, [90, 200], shift=1)
    prompt_check(cuda, c, *prompt_run(cuda, irx, c))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_prompt_shards_are_the_whole(cuda, irx, dtype):
    torch = cuda
    c = prompt_case(torch, irx, dtype, 6, 3, 64, [90, 0, 200], window=50, sinks=2)
    whole = prompt_run(torch, irx, c)

    def shards(args):
        for r in range(2):
            c["plan"].launch_shard(r, 2, args)
    split = prompt_run(torch, irx, c, shards)
    assert all(torch.equal(a, b) for a, b in zip(whole, split))


def test_prompt_many_sequences(cuda, irx):
    rnd = random.Random(5)
    c = prompt_case(cuda, irx, "bf16", 4, 2, 64, [rnd.choice([0, 1, 2, 5, 17, 64, 130]) for _ in range(150)])
    prompt_check(cuda, c, *prompt_run(cuda, irx, c))


def test_prompt_far_rows(cuda, irx):
    """Offsets past 32 bits: rows of a wide buffer."""
    torch = cuda
    stride, t = 1 << 24, 140
    big = torch.empty(t * stride, dtype=torch.bfloat16, device="cuda")
    q = big.as_strided((t, 2, 64), (stride, 64, 1))
    k, v = big[256:].as_strided((t, 1, 64), (stride, 64, 1)), big[512:].as_strided((t, 1, 64), (stride, 64, 1))
    gen = torch.Generator(device="cuda").manual_seed(0)
    for x in (q, k, v):
        x.copy_(normal(torch, gen, x.shape, "bf16"))
    c = dict(q=q, k=k, v=v, starts=[0, 3, t], plan=irx.prompt(t, 2, 2, 1, 64, lse=True, q_stride=stride, kv_stride=stride), t=t, heads=2, d=64,
             dtype="bf16", window=0, sinks=0, scale=0.125)
    prompt_check(torch, c, *prompt_run(torch, irx, c))


# ---- the draw ----

def draw(torch, irx, logits, settings, logprob=True, vocab=None):
    """settings: (temperature, top_k, top_p, min_p, u) a row. Returns tokens and logs."""
    m, n = len(settings), vocab or logits.shape[1]
    cols = list(zip(*settings))
    dev = [torch.tensor(c, dtype=torch.int32 if i == 1 else torch.float32, device="cuda") for i, c in enumerate(cols)]
    token, lp = torch.full((m,), -7, dtype=torch.int32, device="cuda"), torch.full((m,), 7.0, device="cuda")
    plan = irx.sample(m, n, dtype="bf16" if logits.dtype == torch.bfloat16 else "f32", stride=logits.stride(0) if m > 1 else 0, logprob=logprob)
    plan.launch([logits] + dev + [token] + ([lp] if logprob else []))
    irx.check()
    return token.tolist(), lp.tolist()


def draw_check(torch, irx, logits, settings):
    token, lp = draw(torch, irx, logits, settings)
    for i, s in enumerate(settings):
        # the settings as the kernel gets them, in f32
        t, k, p, least, u = (torch.tensor(x, dtype=torch.float32).item() if j != 1 else x for j, x in enumerate(s))
        want, wlp = sample_exact(torch, logits[i], t, k, p, least, u)
        assert token[i] == want, (i, s, token[i], want)
        assert lp[i] == wlp or abs(lp[i] - wlp) <= 2.0 ** -23 * abs(wlp) + 2.0 ** -24, (i, s, lp[i], wlp)


FILTERS = [(0, 1.0, 0.0), (1, 1.0, 0.0), (5, 1.0, 0.0), (50, 0.9, 0.0), (0, 0.5, 0.0), (0, 0.95, 0.0), (0, 1.0, 0.1), (40, 0.8, 0.05), (3, 0.01, 0.9)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 2, 31, 32, 129, 1000, 4097, 8191, 50000, 128001])
def test_sample(cuda, irx, dtype, n):
    torch = cuda
    gen, rnd = torch.Generator(device="cuda").manual_seed(n), random.Random(n)
    settings = [(rnd.choice([0.3, 0.7, 1.0, 1.7]), *f, rnd.random()) for f in FILTERS] + [(0.0, 5, 0.5, 0.1, 0.3)]
    draw_check(torch, irx, normal(torch, gen, (len(settings), n), dtype, 3.0), settings)


@pytest.mark.parametrize("n", [3, 1000, 33333])
@pytest.mark.parametrize("value", [0.0, -5.5, 3e38])
def test_sample_equal_logits(cuda, irx, n, value):
    """All equal: the kept ones are the lowest indexes, and sums meet their borders exactly."""
    torch = cuda
    settings = [(1.0, k, p, m, u) for k, p, m in [(0, 1.0, 0.0), (7, 1.0, 0.0), (0, 0.5, 0.0), (8, 0.5, 0.0), (0, 0.25, 1.0), (1, 0.0, 0.0)]
                for u in (0.0, 0.25, 0.5, 0.99999994)]
    draw_check(torch, irx, torch.full((len(settings), n), value, device="cuda"), settings)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [257, 20000])
def test_sample_few_values(cuda, irx, dtype, n):
    """Logits of a handful of values, both zeros among them: thresholds fall inside runs of equal ones."""
    torch = cuda
    gen, rnd = torch.Generator(device="cuda").manual_seed(n), random.Random(n)
    x = torch.tensor([1.0, 0.0, -0.0, -1.0, 2.0, -30.0], device="cuda")[torch.randint(0, 6, (48, n), generator=gen, device="cuda")].to(tdt(torch, dtype))
    settings = [(rnd.choice([0.5, 1.0]), rnd.choice([0, 1, 10, n // 6, n // 3, n - 1, n, n + 5]), rnd.choice([1.0, 0.1, 0.4, 0.73]), rnd.choice([0.0, 0.2, 0.5]),
                 rnd.random()) for _ in range(48)]
    draw_check(torch, irx, x, settings)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_sample_masks_and_numbers_out_of_range(cuda, irx, dtype):
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(3)
    n = 5000
    low = torch.finfo(tdt(torch, dtype)).min
    x = normal(torch, gen, (20, n), dtype, 2.0)
    x[0, ::2] = -INF
    x[1, 3:] = -INF
    x[2, :] = -INF
    x[3, :] = NAN
    x[4, ::3] = NAN
    x[5, 100], x[5, 4000] = INF, INF
    x[6, ::2] = low
    x[7, 5:] = low
    x[8, :] = low
    x[9, 10:] = -INF
    x[9, :10] = low
    x[10, 7] = -low
    x[11, :] = -INF
    x[11, 4999] = -3.0
    x[12, ::2] = -1e9
    x[13] = x[13] * 1e-30
    x[14, 17] = INF
    x[15, :] = INF
    for f in FILTERS:
        for u in (0.0, 0.37, 0.99999994):
            draw_check(torch, irx, x, [(0.8, *f, u)] * 20)
    draw_check(torch, irx, x, [(0.0, 3, 0.5, 0.1, 0.5)] * 20)


def test_sample_settings_out_of_range(cuda, irx):
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(4)
    n = 3001
    settings = [(1.0, -5, 2.0, -1.0, 0.4), (1.0, n, 1.5, 0.0, 0.4), (1.0, n + 9, NAN, NAN, 0.4), (NAN, 0, 1.0, 0.0, 0.4), (-1.0, 0, 1.0, 0.0, 0.4),
                (1.0, 0, -3.0, 0.0, 0.4), (1.0, 0, 1e-30, 0.0, 0.4), (1.0, 0, 1.0, 7.0, 0.4), (1.0, 0, 1.0, 0.0, 1.0), (1.0, 0, 1.0, 0.0, 5.0),
                (1.0, 0, 1.0, 0.0, -2.0), (1.0, 9, 1.0, 0.0, NAN), (1e-30, 50, 0.9, 0.0, 0.4), (1e-44, 0, 1.0, 0.0, 0.4), (1e30, 0, 0.5, 0.0, 0.4),
                (1e30, 100, 0.5, 0.5, 0.7), (3e38, 0, 1.0, 1.0, 0.7), (1.0, 2 ** 31 - 1, 0.9, 0.0, 0.4)]
    draw_check(torch, irx, normal(torch, gen, (len(settings), n), "f32", 3.0), settings)
    # an infinite temperature makes all weights equal
    token, lp = draw(torch, irx, torch.linspace(-5, 5, 1000, device="cuda")[None], [(INF, 0, 1.0, 0.0, 0.25)])
    assert token == [250] and abs(lp[0] + math.log(1000)) < 1e-6


def test_sample_rows_past_shared_memory(cuda, irx):
    """A vocabulary that a cluster's shared memory does not hold, and rows of a wider buffer."""
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(5)
    for dtype, n in (("f32", 500001), ("bf16", 900001)):
        wide = normal(torch, gen, (9, n + 7), dtype, 2.0)
        draw_check(torch, irx, wide[:, 3:n + 3], [(0.9, *f, 0.1 * i + 0.05) for i, f in enumerate(FILTERS)])


def test_sample_unaligned_rows(cuda, irx):
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(6)
    for dtype in ("f32", "bf16"):
        wide = normal(torch, gen, (9, 7001), dtype, 2.0)
        draw_check(torch, irx, wide[:, 1:6001], [(0.9, *f, 0.1 * i + 0.05) for i, f in enumerate(FILTERS)])


def test_sample_follows_its_distribution(cuda, irx):
    """Each token is drawn for the stretch of u that is its share."""
    torch = cuda
    w = torch.tensor([0.5, 0.25, 0.125, 0.0625, 0.0625])
    x = torch.log(w).cuda().repeat(4096, 1).contiguous()
    token, lp = draw(torch, irx, x, [(1.0, 0, 1.0, 0.0, (i + 0.5) / 4096) for i in range(4096)])
    assert [token.count(i) for i in range(5)] == [2048, 1024, 512, 256, 256] and token == sorted(token)
    assert all(abs(a - math.log(float(w[t]))) < 1e-6 for a, t in zip(lp, token))


def test_sample_shards_are_the_whole(cuda, irx):
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(7)
    x = normal(torch, gen, (7, 5000), "f32", 2.0)
    dev = [torch.full((7,), v, device="cuda") for v in (0.9, 0.9, 0.0)] + [torch.rand(7, generator=gen, device="cuda")]
    k = torch.full((7,), 60, dtype=torch.int32, device="cuda")
    plan = irx.sample(7, 5000)
    a, b = (torch.full((7,), -7, dtype=torch.int32, device="cuda") for _ in range(2))
    plan.launch([x, dev[0], k, dev[1], dev[2], dev[3], a])
    for r in range(3):
        plan.launch_shard(r, 3, [x, dev[0], k, dev[1], dev[2], dev[3], b])
    irx.check()
    assert torch.equal(a, b) and int(a.min()) >= 0


# ---- all of them: streams, graphs, repeats ----

def everything(torch, irx, seed):
    """A launch of each operator over buffers of its own: [(plan, args, outputs)]."""
    c = append_case(torch, irx, "bf16", "head", False, 8, 2, 64, 64, 16, 3, True, False, seed=seed)
    seq, pos = ints(torch, [s for s, _ in c["places"]]), ints(torch, [p for _, p in c["places"]])
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = normal(torch, gen, (50, 4, 64), "f32")
    y = torch.zeros_like(x)
    out = torch.zeros_like(c["q"].contiguous())
    jobs = [(irx.rope(50, 4, 64, c["freqs"], dtype="f32"), [x, ints(torch, list(range(50))), y], [y]),
            (c["plan"], [c["q"], c["k"], c["v"], seq, pos, c["table"], out] + c["pools"], [out] + c["pools"])]
    for dtype in ("bf16", "f32"):
        p = prompt_case(torch, irx, dtype, 4, 2, 64, [100, 37, 260], seed=seed)
        o, lse = torch.zeros(p["t"], 4, 64, dtype=p["q"].dtype, device="cuda"), torch.zeros(p["t"], 4, device="cuda")
        jobs.append((p["plan"], [p["q"], p["k"], p["v"], ints(torch, p["starts"]), o, lse], [o, lse]))
    logits = normal(torch, gen, (8, 30011), "f32", 2.5)
    token, lp = torch.zeros(8, dtype=torch.int32, device="cuda"), torch.zeros(8, device="cuda")
    full = [torch.full((8,), v, device="cuda") for v in (0.8, 0.9, 0.02)]
    jobs.append((irx.sample(8, 30011, logprob=True),
                 [logits, full[0], ints(torch, [40, 0] * 4), full[1], full[2], torch.rand(8, generator=gen, device="cuda"), token, lp], [token, lp]))
    return jobs


def test_streams_graphs_and_repeats_give_the_same_bits(cuda, irx):
    torch = cuda
    sets = [everything(torch, irx, s) for s in (1, 2)]
    want = []
    for jobs in sets:
        for plan, args, outs in jobs:
            plan.launch(args)
        irx.check()
        want.append([[o.clone() for o in outs] for _, _, outs in jobs])

    def clear():
        for jobs in sets:
            for _, _, outs in jobs:
                for o in outs:
                    if o.dim() < 4:
                        o.zero_()
        torch.cuda.synchronize()

    def same():
        torch.cuda.synchronize()
        irx.check()
        assert all(torch.equal(o, w) for jobs, ws in zip(sets, want) for (_, _, outs), wo in zip(jobs, ws) for o, w in zip(outs, wo))

    clear()                                              # two streams at once
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        for jobs, s in zip(sets, streams):
            for plan, args, _ in jobs:
                plan.launch(args, stream=s)
    same()
    clear()                                              # two graphs, replayed at once
    graphs = []
    for jobs in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            for plan, args, _ in jobs:
                plan.launch(args)
        graphs.append(g)
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    same()
    del graphs


def test_a_captured_step_reads_what_changed(cuda, irx):
    torch = cuda
    c = prompt_case(torch, irx, "bf16", 4, 2, 64, [100, 200, 60])
    starts = ints(torch, c["starts"])
    out, lse = torch.zeros(c["t"], 4, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(c["t"], 4, device="cuda")
    args = [c["q"], c["k"], c["v"], starts, out, lse]
    c["plan"].launch(args)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c["plan"].launch(args)
    for lens in ([300, 60, 0], [0, 7, 1], [120, 120, 120]):
        c["starts"] = [0]
        for n in lens:
            c["starts"].append(c["starts"][-1] + n)
        starts.copy_(ints(torch, c["starts"]))
        out.fill_(7.0)
        lse.fill_(7.0)
        g.replay()
        irx.check()
        prompt_check(torch, c, out, lse)
    del g


def test_refused_launches(cuda, irx):
    torch = cuda
    p = irx.sample(2, 100)
    good = [torch.zeros(2, 100, device="cuda")] + [torch.zeros(2, device="cuda"), ints(torch, [0, 0])] + [torch.zeros(2, device="cuda")] * 3 + [ints(torch, [0, 0])]

    def bad(i, x):
        args = list(good)
        args[i] = x
        with pytest.raises(irx.IrxError) as e:
            p.launch(args)
        assert e.value.code == 93
    bad(0, torch.zeros(2, 100))
    bad(0, torch.zeros(2, 100, device="cuda", dtype=torch.bfloat16))
    bad(0, torch.zeros(100, 2, device="cuda").t())
    bad(2, torch.zeros(2, device="cuda"))
    bad(6, ints(torch, [0, 0, 0]))
    bad(6, good[6].data_ptr() + 2)
    with pytest.raises(irx.IrxError):
        p.launch(good[:-1])
    p.launch(good)
    irx.check()
