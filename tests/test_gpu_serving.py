"""The serving operators on a GPU against their definitions in 64 bits: paged decode attention, cache
append and page copy, 4-bit matrix-vector products, at the sizes and masks where they can go
wrong. Tolerances are bounds on the roundings each operator makes (stated at `decode_tol` and
`mv_tol`); moved values have to be equal."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

DT = {"bf16": "bfloat16", "f32": "float32"}


@pytest.fixture(autouse=True)
def _reference_core_for_gpu_tests():
    """These operators have no counterpart in the reference, so its core is not needed here."""


def tdt(torch, dtype):
    return getattr(torch, DT[dtype])


def pool(torch, cache, gen, fill=None):
    t = torch.empty(cache.shape, dtype=torch.float32, device="cuda")
    t = t.normal_(generator=gen) if fill is None else t.fill_(fill)
    return t.to(tdt(torch, cache.dtype))


def visible(n, window, sinks):
    return [j for j in range(n) if not window or j >= n - window or j < sinks]


def rows(pool, order, page, slot, h):
    return pool[page, h, slot] if order == "head" else pool[page, slot, h]


def decode_exact(torch, q, k, v, table, lens, order, scale, window, sinks):
    """(out, lse, spread, scores) in float64: spread is sum_j p_j |v_j|, scores the largest of
    |scale| sum_i |q_i k_ij| of each row, for the tolerance."""
    b, heads, d = q.shape
    hk = k.shape[1] if order == "head" else k.shape[2]
    ps = k.shape[2] if order == "head" else k.shape[1]
    g = heads // hk
    out = torch.zeros(b, heads, d, dtype=torch.float64)
    spread = torch.zeros_like(out)
    lse = torch.full((b, heads), -math.inf, dtype=torch.float64)
    big = torch.zeros(b, heads, dtype=torch.float64)
    q, k, v, table = q.double().cpu(), k.double().cpu(), v.double().cpu(), table.cpu().long()
    for i, n in enumerate(lens):
        at = torch.tensor(visible(n, window, sinks), dtype=torch.long)
        if not len(at):
            continue
        page, slot = table[i][at // ps], at % ps
        for h in range(hk):
            ks, vs = rows(k, order, page, slot, h), rows(v, order, page, slot, h)
            qq = q[i, h * g:(h + 1) * g]
            s = scale * (qq @ ks.T)
            p = torch.softmax(s, -1)
            out[i, h * g:(h + 1) * g] = p @ vs
            spread[i, h * g:(h + 1) * g] = p @ vs.abs()
            lse[i, h * g:(h + 1) * g] = torch.logsumexp(s, -1)
            big[i, h * g:(h + 1) * g] = (abs(scale) * (qq.abs() @ ks.abs().T)).amax(-1)
    return out, lse, spread, big


def score_err(d, big):
    """Bound of a score's error: d products and sums and the scale, in f32, twice (the maximum's too)."""
    return 2 * (d + 4) * 2.0 ** -24 * big + 2.0 ** -21


def decode_tol(dtype, d, n, out, spread, big):
    """f32: each weight's error (its score's, the exp's 2^-22, n sums). bf16 besides: weights rounded to
    8 bits in the product and in their sum and the output rounded, 2^-9 allowed for each: half the
    worst case, which would need every rounding at its limit at once."""
    w = score_err(d, big)[..., None] + (n + 16) * 2.0 ** -23
    if dtype == "bf16":
        return (w + 2 * 2.0 ** -9) * spread + 2.0 ** -9 * out.abs() + 1e-30
    return w * spread + 2.0 ** -24 * out.abs()


def run_decode(torch, irx, dtype="bf16", heads=4, kv=2, d=64, page=16, lens=(5,), window=0, sinks=0, order="head", lse=True,
               strided=False, shift=0, scale=None, seed=0, stale=float("nan"), spare=3, qmul=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    b, cols = len(lens), max(1, -(-max(lens) // page)) + 1
    pages = b * cols + spare
    inner = (kv, page) if order == "head" else (page, kv)
    strides = None
    if strided or shift:
        # a view with gaps after each row, block and page, and a base `shift` elements in
        gap = 8 if not shift else 0
        s2 = d + gap
        s1 = inner[1] * s2 + gap
        strides = (inner[0] * s1 + gap, s1, s2)
    cache = irx.KvCache(dtype, kv, d, page, pages, batch=b, table_cols=cols, order=order, strides=strides)
    big = pages * cache.strides[0] + shift + 8

    def make():
        flat = torch.full((big,), stale, dtype=tdt(torch, dtype), device="cuda")
        return flat[shift:].as_strided(cache.shape, cache.strides + (1,))

    k, v = make(), make()
    table = torch.randperm(pages, generator=gen, device="cuda")[:b * cols].to(torch.int32).reshape(b, cols)
    ref_t = table.cpu().long()
    for i, n in enumerate(lens):                        # only the rows a token was written to hold numbers
        for j in range(n):
            pg, sl = int(ref_t[i, j // page]), j % page
            kr = torch.empty(kv, d, device="cuda").normal_(generator=gen)
            vr = torch.empty(kv, d, device="cuda").normal_(generator=gen)
            if order == "head":
                k[pg, :, sl], v[pg, :, sl] = kr.to(k.dtype), vr.to(v.dtype)
            else:
                k[pg, sl], v[pg, sl] = kr.to(k.dtype), vr.to(v.dtype)
    for i, n in enumerate(lens):                        # entries that no token reaches may hold anything
        table[i, -(-n // page):] = 10 ** 9
    wide = heads * d + (16 if strided else 0)
    q = (torch.empty(b, wide, device="cuda").normal_(generator=gen) * qmul).to(tdt(torch, dtype))
    q = q[:, :heads * d].unflatten(1, (heads, d))
    plan = irx.decode(cache, heads, scale=scale, window=window, sinks=sinks, lse=lse, q_stride=wide if strided else 0)
    out = torch.full((b, heads, d), float("nan"), dtype=q.dtype, device="cuda")
    ls = torch.full((b, heads), float("nan"), device="cuda")
    lt = torch.tensor(lens, dtype=torch.int32, device="cuda")
    ws = plan.workspace()
    args = [q, k, v, table, lt, out] + ([ls] if lse else []) + [ws]
    plan.launch(args)
    irx.check()
    sc = 1.0 / math.sqrt(d) if scale is None else scale
    return dict(plan=plan, args=args, out=out, lse=ls, ws=ws, table=table, lens=lt, order=order,
                exact=lambda ln=lens: decode_exact(torch, q, k, v, table, ln, order, sc, window, sinks))


def hold_decode(torch, r, dtype, d, lens):
    out, lse, spread, big = r["exact"]()
    err = (r["out"].double().cpu() - out).abs()
    tol = decode_tol(dtype, d, max(lens), out, spread, big)
    assert bool((err <= tol).all()), f"worst {float((err / tol.clamp_min(1e-300)).nan_to_num(9e9).max()):.3g} of the bound"
    got = r["lse"].double().cpu()
    live = torch.isfinite(lse)
    assert bool((got[~live] == -math.inf).all())
    slack = 2.0 ** -8 if dtype == "bf16" else 0.0         # the sum of rounded weights
    tl = score_err(d, big) + (max(lens) + 16) * 2.0 ** -23 + slack + 2.0 ** -22 * lse.abs().nan_to_num(posinf=0.0, neginf=0.0)
    assert bool(((got - lse).abs()[live] <= tl[live]).all())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads,kv,d,page", [(1, 1, 64, 16), (8, 8, 128, 16), (8, 1, 128, 8), (24, 2, 64, 1), (16, 1, 96, 5),
                                             (20, 1, 128, 64), (5, 5, 80, 24), (16, 2, 256, 16), (9, 1, 256, 3), (40, 2, 40, 16)])
def test_decode_shapes(cuda, irx, dtype, heads, kv, d, page):
    lens = (1, 0, 64, 65, 130, 17)
    r = run_decode(cuda, irx, dtype, heads, kv, d, page, lens, order="head" if page % 2 == 0 else "token")
    hold_decode(cuda, r, dtype, d, lens)


@pytest.mark.parametrize("d", [1, 7, 33, 100, 255])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_decode_odd_head_sizes(cuda, irx, dtype, d):
    lens = (3, 70)
    hold_decode(cuda, run_decode(cuda, irx, dtype, 6, 2, d, 4, lens), dtype, d, lens)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 3), (16, 4), (64, 1), (63, 200), (1000, 4), (129, 0)])
def test_decode_window_and_sinks(cuda, irx, dtype, window, sinks):
    lens = (0, 1, 16, 17, 64, 65, 129, 300)
    hold_decode(cuda, run_decode(cuda, irx, dtype, 8, 2, 64, 16, lens, window=window, sinks=sinks), dtype, 64, lens)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lens", [(1100,), (2500, 3), (0, 0, 1500, 0), (1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 900)])
def test_decode_split_and_joined(cuda, irx, dtype, lens):
    """One long sequence: its chunks spread over many blocks, past the join's one-step limit too."""
    r = run_decode(cuda, irx, dtype, 4, 1, 64, 16, lens)
    hold_decode(cuda, r, dtype, 64, lens)
    first = r["out"].clone()
    for _ in range(3):                                   # the workspace is left ready, the result is the same bits
        r["out"].fill_(float("nan"))
        r["plan"].launch(r["args"])
        irx.check()
        assert cuda.equal(first, r["out"])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("order", ["head", "token"])
def test_decode_strided_pools_and_queries(cuda, irx, dtype, order):
    lens = (33, 90)
    hold_decode(cuda, run_decode(cuda, irx, dtype, 8, 2, 64, 16, lens, order=order, strided=True), dtype, 64, lens)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_decode_unaligned_pools(cuda, irx, dtype):
    lens = (33, 90)
    hold_decode(cuda, run_decode(cuda, irx, dtype, 8, 2, 64, 16, lens, shift=1), dtype, 64, lens)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("qmul,scale", [(100.0, None), (1.0, 0.0), (1.0, -0.5), (1e-3, 1.0)])
def test_decode_score_ranges(cuda, irx, dtype, qmul, scale):
    """Sharp and flat softmax, a zero and a negative scale."""
    lens = (100, 40)
    hold_decode(cuda, run_decode(cuda, irx, dtype, 4, 2, 64, 16, lens, qmul=qmul, scale=scale), dtype, 64, lens)


def test_decode_infinite_stale_rows(cuda, irx):
    lens = (1, 63, 100)
    hold_decode(cuda, run_decode(cuda, irx, "bf16", 4, 2, 128, 16, lens, window=20, sinks=2, stale=float("inf")), "bf16", 128, lens)


def test_decode_nan_key_reaches_its_row_only(cuda, irx):
    r = run_decode(cuda, irx, "bf16", 4, 2, 64, 16, (40, 40))
    k = r["args"][1]
    k[int(r["table"][0, 1]), 0, 3] = float("nan")        # sequence 0, kv head 0
    r["plan"].launch(r["args"])
    irx.check()
    out = r["out"]
    assert bool(out[0, :2].isnan().all()) and not bool(out[0, 2:].isnan().any()) and not bool(out[1].isnan().any())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_decode_shards_are_the_whole(cuda, irx, dtype):
    lens = (0, 700, 65)
    r = run_decode(cuda, irx, dtype, 12, 3, 64, 16, lens)
    whole = r["out"].clone()
    r["out"].fill_(float("nan"))
    r["lse"].fill_(float("nan"))
    for s in range(2):
        r["plan"].launch_shard(s, 2, r["args"])
    irx.check()
    assert not bool(r["out"].isnan().any()) and not bool(r["lse"].isnan().any())
    hold_decode(cuda, r, dtype, 64, lens)
    assert cuda.equal(whole[0], r["out"][0])


def test_decode_in_a_graph_with_growing_lengths(cuda, irx):
    r = run_decode(cuda, irx, "bf16", 8, 2, 128, 16, (200, 130))
    bound, side = r["plan"].bind(r["args"]), cuda.cuda.Stream()
    side.wait_stream(cuda.cuda.current_stream())
    graph = cuda.cuda.CUDAGraph()
    with cuda.cuda.graph(graph, stream=side):
        r["plan"].launch(bound)
    for lens in ((200, 130), (64, 1), (0, 129)):
        r["lens"].copy_(cuda.tensor(lens, dtype=cuda.int32))
        r["out"].fill_(float("nan"))
        graph.replay()
        cuda.cuda.synchronize()
        rr = dict(r, exact=lambda: r["exact"](lens))
        hold_decode(cuda, rr, "bf16", 128, lens)
    del graph
    irx.check()


def test_decode_bad_indices_are_reported(cuda, irx):
    r = run_decode(cuda, irx, "bf16", 4, 2, 64, 16, (40, 40))
    good = r["out"].clone()
    keep = r["table"].clone()
    for bad in (-1, 10 ** 9):
        r["table"][0, 1] = bad
        r["plan"].launch(r["args"])
        with pytest.raises(irx.IrxError) as e:
            irx.check()
        assert e.value.code == 93
        irx.check()                                      # reported once
        assert cuda.equal(r["out"][1], good[1])
    r["table"].copy_(keep)
    r["lens"][1] = -5
    r["plan"].launch(r["args"])
    with pytest.raises(irx.IrxError):
        irx.check()
    assert bool((r["out"][1] == 0).all()) and cuda.equal(r["out"][0], good[0])


# ---- append ----

def append_exact(torch, k0, new, seq, pos, table, page, order):
    want = k0.clone()
    for i, (s, p) in enumerate(zip(seq, pos)):
        if p < 0:
            continue
        pg = int(table[s, p // page])
        if order == "head":
            want[pg, :, p % page] = new[i]
        else:
            want[pg, p % page] = new[i]
    return want


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kv,d,page,order,extra", [(8, 128, 16, "head", 0), (1, 64, 1, "token", 0), (3, 80, 5, "head", 40),
                                                   (2, 7, 4, "token", 3), (2, 33, 16, "head", 1), (32, 256, 8, "token", 0)])
def test_append(cuda, irx, dtype, kv, d, page, order, extra):
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(3)
    b, cols = 3, 7
    cache = irx.KvCache(dtype, kv, d, page, b * cols, batch=b, table_cols=cols, order=order)
    k, v = pool(torch, cache, gen), pool(torch, cache, gen)
    table = torch.randperm(b * cols, generator=gen, device="cuda").to(torch.int32).reshape(b, cols)
    cap = cols * page
    seq = [0, 0, 2, 1, 1, 2, 0]
    pos = [0, cap - 1, cap // 2, -1, 1 % cap, min(2, cap - 1), -7]
    new = [(torch.empty(len(seq), kv * d + extra, device="cuda").normal_(generator=gen)).to(k.dtype)[:, :kv * d].unflatten(1, (kv, d))
           for _ in range(2)]
    plan = irx.kv_append(cache, len(seq), stride=kv * d + extra)
    k0, v0 = k.clone(), v.clone()
    ints = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (seq, pos)]
    plan.launch(new + ints + [table, k, v])
    irx.check()
    assert torch.equal(k, append_exact(torch, k0, new[0], seq, pos, table, page, order))
    assert torch.equal(v, append_exact(torch, v0, new[1], seq, pos, table, page, order))
    # sharded: the same writes
    k2, v2 = k0.clone(), v0.clone()
    for s in range(3):
        plan.launch_shard(s, 3, new + ints + [table, k2, v2])
    irx.check()
    assert torch.equal(k, k2) and torch.equal(v, v2)
    # what lies outside the cache is skipped and reported
    for s, p in ((3, 0), (-1, 0), (0, cap)):
        ints[0][0], ints[1][0] = s, p
        plan.launch(new + ints + [table, k2, v2])
        with pytest.raises(irx.IrxError) as e:
            irx.check()
        assert e.value.code == 93
        assert torch.equal(k, k2) and torch.equal(v, v2)


# ---- page copy ----

@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kv,d,page,order,layers,strided", [(8, 128, 16, "head", 2, False), (1, 7, 3, "token", 1, False),
                                                            (3, 40, 5, "head", 3, True), (2, 33, 4, "token", 2, True)])
def test_copy(cuda, irx, dtype, kv, d, page, order, layers, strided):
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(4)
    pages = 40
    inner = (kv, page) if order == "head" else (page, kv)
    gap = 8 if strided else 0
    strides = (inner[0] * (inner[1] * (d + gap)) + gap, inner[1] * (d + gap), d + gap)
    cache = irx.KvCache(dtype, kv, d, page, pages, order=order, strides=strides)
    ls = pages * strides[0] + gap
    flat = [torch.empty(layers * ls, device="cuda").normal_(generator=gen).to(tdt(torch, dtype)) for _ in range(2)]
    view = [f.as_strided((layers,) + cache.shape, (ls,) + strides + (1,)) for f in flat]
    order_ = torch.randperm(pages, generator=gen, device="cuda").tolist()
    pairs = [(order_[0], order_[1]), (order_[0], order_[2]), (-1, -1), (order_[3], order_[4])]
    want = [f.clone() for f in flat]
    for f in want:
        w = f.as_strided(view[0].shape, view[0].stride())
        for s, t in pairs:
            if s >= 0:
                w[:, t] = w[:, s]
    plan = irx.kv_copy(cache, len(pairs), layers=layers, layer_stride=ls)
    pt = torch.tensor(pairs, dtype=torch.int32, device="cuda")
    plan.launch([pt] + view)
    irx.check()
    assert torch.equal(flat[0], want[0]) and torch.equal(flat[1], want[1])     # the gaps too
    for bad in ((0, pages), (-1, 0), (0, -2)):
        pt.fill_(-1)
        pt[1] = torch.tensor(bad, dtype=torch.int32)
        plan.launch([pt] + view)
        with pytest.raises(irx.IrxError) as e:
            irx.check()
        assert e.value.code == 93
        assert torch.equal(flat[0], want[0]) and torch.equal(flat[1], want[1])


# ---- 4-bit matrix-vector products ----

def mv_tol(dtype, k, y, mag):
    """Products are exact, k of them are summed in f32 with their groups' scales (one more rounding
    each); a weight times its scale rounds once on the path for any size. Outputs round once: half a
    unit in the last place, relative 2^-8 for bf16's 8 significant bits, 2^-24 for f32."""
    return (k + 8) * 2.0 ** -24 * mag + (2.0 ** -8 if dtype == "bf16" else 2.0 ** -24) * y.abs() + 1e-30


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("m,n,k,group,zeros,sd", [
    (1, 256, 512, 128, False, None), (1, 17, 128, 64, True, None), (3, 100, 1056, 32, True, "f32"), (8, 33, 4096, 128, True, None),
    (9, 65, 2048, 64, False, None), (16, 32, 96, 96, True, None), (17, 48, 320, 64, False, "f32"), (2, 31, 1312, 256, True, None),
    (1, 1, 1, 1, False, None), (5, 9, 77, 10, True, None), (2, 40, 130, 128, False, None), (4, 16, 160, 7, True, "bf16"),
    (1, 5, 4096, 4096, True, None), (33, 16, 64, 32, False, None)])
def test_matvec4(cuda, irx, dtype, m, n, k, group, zeros, sd):
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(5)
    groups = -(-k // group)
    q = torch.randint(0, 16, (n, k), generator=gen, device="cuda")
    w = irx.pack4(q)
    x = torch.empty(m, k, device="cuda").normal_(generator=gen).to(tdt(torch, dtype))
    s = (torch.rand(n, groups, generator=gen, device="cuda") + 0.1).to(tdt(torch, sd or dtype))
    z = torch.randint(0, 16, (n, groups), generator=gen, device="cuda", dtype=torch.uint8)
    plan = irx.matvec4(m, n, k, group=group, dtype=dtype, scale_dtype=sd, zeros=zeros)
    y = torch.full((m, n), float("nan"), dtype=x.dtype, device="cuda")
    args = [x, w, s] + ([z] if zeros else []) + [y]
    plan.launch(args)
    irx.check()
    col = torch.arange(k, device="cuda") // group
    wf = (q - (z.long()[:, col] if zeros else 8)).double() * s.double()[:, col]
    want, mag = x.double() @ wf.T, x.double().abs() @ wf.abs().T
    err = (y.double() - want).abs()
    assert bool((err <= mv_tol(dtype, k, want, mag)).all())
    y2 = torch.full_like(y, float("nan"))
    for sh in range(3):
        plan.launch_shard(sh, 3, args[:-1] + [y2])
    irx.check()
    assert torch.equal(y, y2)                            # rows are independent: the same bits


def test_matvec4_strides_and_unaligned(cuda, irx):
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(6)
    m, n, k = 3, 20, 256
    q = torch.randint(0, 16, (n, k), generator=gen, device="cuda")
    s = torch.rand(n, 2, generator=gen, device="cuda").to(torch.bfloat16)
    for xs, ws, off in ((k + 8, k // 2 + 16, 0), (k + 1, k // 2 + 3, 0), (k, k // 2, 1)):
        xb = torch.empty(m * xs + 8, device="cuda").normal_(generator=gen).to(torch.bfloat16)
        x = xb[off:].as_strided((m, k), (xs, 1))
        wb = torch.zeros(n * ws + 8, dtype=torch.uint8, device="cuda")
        w = wb[off:].as_strided((n, k // 2), (ws, 1))
        w.copy_(irx.pack4(q))
        y = torch.full((m, n), float("nan"), dtype=torch.bfloat16, device="cuda")
        irx.matvec4(m, n, k, x_stride=xs, w_stride=ws).launch([x, w, s, y])
        irx.check()
        wf = (q - 8).double() * s.double()[:, torch.arange(k, device="cuda") // 128]
        want, mag = x.double() @ wf.T, x.double().abs() @ wf.abs().T
        assert bool(((y.double() - want).abs() <= mv_tol("bf16", k, want, mag)).all())


def test_matvec4_special_values_stay_in_their_row(cuda, irx):
    torch = cuda
    m, n, k = 4, 48, 512
    x = torch.ones(m, k, dtype=torch.bfloat16, device="cuda")
    x[1, 77], x[2, 5] = float("inf"), float("nan")
    w = torch.full((n, k // 2), 0xFF, dtype=torch.uint8, device="cuda")       # every weight 7
    s = torch.full((n, 4), 0.5, dtype=torch.bfloat16, device="cuda")
    y = torch.zeros(m, n, dtype=torch.bfloat16, device="cuda")
    irx.matvec4(m, n, k).launch([x, w, s, y])
    irx.check()
    assert bool((y[0] == 1792).all()) and bool((y[1] == math.inf).all()) and bool(y[2].isnan().all()) and bool((y[3] == 1792).all())


# ---- the checks of arguments ----

def test_launch_refusals(cuda, irx):
    torch = cuda
    r = run_decode(cuda, irx, "bf16", 4, 2, 64, 16, (20,))
    plan, args = r["plan"], r["args"]
    bad = {0: [args[0].float(), args[0][:, :2], args[0].cpu()], 1: [args[1].transpose(1, 2).contiguous().transpose(1, 2)],
           3: [args[3].long()], 5: [args[5].transpose(1, 2).contiguous().transpose(1, 2)]}
    for i, xs in bad.items():
        for x in xs:
            with pytest.raises(irx.IrxError) as e:
                plan.launch(args[:i] + [x] + args[i + 1:])
            assert e.value.code == 93
    with pytest.raises(irx.IrxError):
        plan.launch(args[:-1])
    with pytest.raises(irx.IrxError):
        plan.launch(args[:-1] + [args[-1].data_ptr() + 4])       # the workspace's alignment
    with pytest.raises(irx.IrxError):
        plan.launch([args[0].data_ptr() + 1] + args[1:])
    with pytest.raises(irx.IrxError):
        plan.run_host([np.zeros(4, np.float32)] * len(args))
    irx.check()


# ---- caches past 32 bits ----

@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_offsets_past_32_bits(cuda, irx, dtype):
    """Two pages more than 2^31 elements apart, written by append, copied and attended to."""
    torch = cuda
    kv, d, page = 2, 64, 16
    far = (1 << 31) + 4096
    cache = irx.KvCache(dtype, kv, d, page, 3, batch=1, table_cols=3, strides=(far // 2, page * d, d))
    k = torch.empty(far + 4096, dtype=tdt(torch, dtype), device="cuda").as_strided(cache.shape, cache.strides + (1,))
    v = torch.empty(far + 4096, dtype=tdt(torch, dtype), device="cuda").as_strided(cache.shape, cache.strides + (1,))
    gen = torch.Generator(device="cuda").manual_seed(1)
    n = 2 * page
    new = [torch.empty(n, kv, d, device="cuda").normal_(generator=gen).to(k.dtype) for _ in range(2)]
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda")
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    irx.kv_append(cache, n).launch(new + [torch.zeros_like(pos), pos, table, k, v])
    assert torch.equal(k[2].transpose(0, 1), new[0][:page]) and torch.equal(v[0].transpose(0, 1), new[1][page:])
    irx.kv_copy(cache, 1).launch([torch.tensor([[2, 1]], dtype=torch.int32, device="cuda"), k[None], v[None]])
    assert torch.equal(k[1], k[2]) and torch.equal(v[1], v[2])
    q = torch.empty(1, 4, d, device="cuda").normal_(generator=gen).to(k.dtype)
    plan, outs = irx.decode(cache, 4), []
    for order in ([2, 0, 0], [1, 0, 0]):                 # the far page, and its copy
        outs.append(torch.empty_like(q))
        plan.launch([q, k, v, torch.tensor([order], dtype=torch.int32, device="cuda"), torch.tensor([n], dtype=torch.int32, device="cuda"),
                     outs[-1], plan.workspace()])
    irx.check()
    assert torch.equal(outs[0], outs[1])
    kk, vv = new[0].double(), new[1].double()
    for h in range(4):
        s = (q[0, h].double() @ kk[:, h // 2].T) / math.sqrt(d)
        p = torch.softmax(s, -1)
        want, spread = p @ vv[:, h // 2], p @ vv[:, h // 2].abs()
        big = (q[0, h].double().abs() @ kk[:, h // 2].abs().T).max() / math.sqrt(d)
        assert bool(((outs[0][0, h].double() - want).abs() <= decode_tol(dtype, d, n, want, spread, big.reshape(())[None])).all())


# ---- together, as a decoding program runs them ----

def test_example_decodes_like_the_dense_model(cuda):
    """Prompt, forks with copy on write, a replayed step graph, a closed sequence and a compaction. The
    bound: each of the two layers rounds its activations to bf16 about ten times (2^-9 of their size
    each, adding like noise), which stays well below a twentieth of the largest logit; a page or
    position gone wrong changes logits by their own size."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "decode_layers.py")
    spec = importlib.util.spec_from_file_location("decode_layers", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    assert mod.main(out=lambda *_: None) < 0.05
