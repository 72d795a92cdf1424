"""The serving operators: paged decode attention, the paged cache's append and page copy, and
matrix-vector products with 4-bit weights, as cases that can be measured.

``listed()`` gives the named cases, ``draw(rng)`` one more of the same ranges. ``prepare(case,
seed)`` makes what a decoding program has in hand (pools, page table, lengths, activations, the
plan), ``run(state)`` is one pass, ``work(case)`` the bytes and operations it cannot do without
and ``exact(case, seed)`` the outputs in 64 bits. With ``own`` false a pass runs the operators'
plain forms in torch; with ``own`` true it launches this package's plans.
"""
import math

import torch

own = False

DT = {"bf16": torch.bfloat16, "f32": torch.float32}
ES = {"bf16": 2, "f32": 4}


# ---- the cases ----

def listed():
    return [
        # one sequence a few tokens into its answer: the smallest decode call, all latency
        dict(name="decode one short", op="decode", dtype="bf16", batch=1, heads=32, kv_heads=8, dim=128, page=16,
             lo=17, hi=17, empty=0, window=0, sinks=0, order="head"),
        # a serving batch in mid-flight: ragged lengths, one slot of the batch empty, one at its first token
        dict(name="decode batch ragged", op="decode", dtype="bf16", batch=32, heads=32, kv_heads=8, dim=128, page=16,
             lo=1, hi=4096, empty=1, window=0, sinks=0, order="head"),
        # two long documents: few rows, a cache that has to be split over its length
        dict(name="decode long", op="decode", dtype="bf16", batch=2, heads=32, kv_heads=8, dim=128, page=64,
             lo=120001, hi=131071, empty=0, window=0, sinks=0, order="head"),
        # a sliding window with the first tokens kept, a key-value head for every query head, token-major pages
        dict(name="decode window sinks", op="decode", dtype="bf16", batch=16, heads=32, kv_heads=32, dim=64, page=32,
             lo=700, hi=16385, empty=0, window=1024, sinks=4, order="token"),
        # an f32 cache, as f32 graphs keep
        dict(name="decode f32", op="decode", dtype="f32", batch=6, heads=16, kv_heads=4, dim=128, page=16,
             lo=1000, hi=3001, empty=0, window=0, sinks=0, order="head"),
        # one new token for each sequence of a serving batch
        dict(name="append step", op="append", dtype="bf16", batch=32, kv_heads=8, dim=128, page=16, start=1021, new=1,
             pad=1, order="head"),
        # the prompts of a batch going in after their prefill, padded to one length
        dict(name="append prompts", op="append", dtype="bf16", batch=8, kv_heads=8, dim=128, page=16, start=3, new=2047,
             pad=40, order="head"),
        # copy on write of the last page of a few forked sequences
        dict(name="copy forked tails", op="copy", dtype="bf16", pairs=7, layers=4, kv_heads=8, dim=128, page=16,
             pages=64, order="head"),
        # a compaction: half of a fragmented pool's pages move down
        dict(name="copy compaction", op="copy", dtype="bf16", pairs=1023, layers=4, kv_heads=8, dim=128, page=16,
             pages=2048, order="head"),
        # a square projection for one token
        dict(name="matvec4 one token", op="matvec4", dtype="bf16", m=1, n=4096, k=4096, group=128, zeros=False),
        # a feed-forward projection with zero points for a few tokens; an odd number of rows
        dict(name="matvec4 few tokens", op="matvec4", dtype="bf16", m=4, n=14337, k=4096, group=64, zeros=True),
        # a feed-forward projection for a small batch, the other way
        dict(name="matvec4 batch", op="matvec4", dtype="bf16", m=13, n=8192, k=14336, group=128, zeros=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["decode", "decode", "matvec4", "matvec4", "append", "copy"])
    order = rng.choice(["head", "token"])
    if op == "matvec4":
        group = rng.choice([32, 64, 128])
        m = _log_int(rng, 1, 16)
        n = _log_int(rng, 256, 16384)
        k = group * max(1, _log_int(rng, 256, 14336) // group)
        return dict(op=op, dtype=rng.choice(["bf16", "bf16", "f32"]), m=m, n=n, k=k, group=group,
                    zeros=rng.random() < 0.5)
    dim = rng.choice([64, 80, 96, 128, 128, 256])
    page = rng.choice([1, 8, 16, 16, 24, 32, 64, 128])
    kv_heads = rng.choice([1, 2, 4, 8, 16])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    row = kv_heads * dim * ES[dtype]              # bytes of one token's keys
    if op == "append":
        batch = _log_int(rng, 1, 32)
        new = max(1, min(2048, _log_int(rng, 1, 2048), (1 << 27) // (row * batch)))
        return dict(op=op, dtype=dtype, batch=batch, kv_heads=kv_heads, dim=dim, page=page, start=rng.randrange(0, 500),
                    new=new, pad=rng.randrange(0, 4), order=order)
    if op == "copy":
        layers = rng.choice([1, 2, 4])
        most = max(2, (1 << 28) // (row * page * layers))
        pairs = max(1, min(_log_int(rng, 1, 1024), most // 2))
        return dict(op=op, dtype=dtype, pairs=pairs, layers=layers, kv_heads=kv_heads, dim=dim, page=page,
                    pages=2 * pairs + rng.randrange(1, 20), order=order)
    batch = _log_int(rng, 1, 48)
    most = max(1, (1 << 29) // (row * batch))     # the padded keys stay below half a gigabyte
    hi = min(131072, most, _log_int(rng, 1, 131072))
    lo = rng.randrange(max(1, hi // 8), hi + 1)
    windowed = rng.random() < 0.35
    return dict(op=op, dtype=dtype, batch=batch, heads=kv_heads * rng.choice([1, 2, 3, 4, 7, 8, 8, 16]),
                kv_heads=kv_heads, dim=dim, page=page, lo=lo, hi=hi, empty=int(batch > 2 and rng.random() < 0.3),
                window=_log_int(rng, 1, hi) if windowed else 0, sinks=rng.choice([0, 1, 4]) if windowed else 0,
                order=order)


# ---- sizes that follow from a case ----

def _lens(c):
    """The sequences' lengths: from lo to hi, spread by the golden ratio's multiples; the first
    `empty` ones hold nothing yet."""
    out = []
    for b in range(c["batch"]):
        f = (b * 0.6180339887498949) % 1.0
        out.append(int(round(c["lo"] + f * (c["hi"] - c["lo"]))))
    for b in range(c["empty"]):
        out[-1 - b] = 0
    return out


def _visible(c, n):
    """How many keys a sequence of n tokens shows its newest token."""
    if not c["window"] or n <= c["window"]:
        return n
    return c["window"] + min(c["sinks"], n - c["window"])


def _pool_shape(c, pages):
    if c["order"] == "head":
        return (pages, c["kv_heads"], c["page"], c["dim"])
    return (pages, c["page"], c["kv_heads"], c["dim"])


def _append_tokens(c):
    """(sequence, position) of every new token; position -1 marks padding. Sequence b gets
    new - (b * pad) % new of its `new` slots filled, the rest is padding."""
    seq, pos = [], []
    for b in range(c["batch"]):
        fill = c["new"] - (b * c["pad"]) % max(1, c["new"])
        for j in range(c["new"]):
            seq.append(b)
            pos.append(c["start"] + b + j if j < fill else -1)
    return seq, pos


def work(c):
    if c["op"] == "decode":
        es = ES[c["dtype"]]
        lens = _lens(c)
        vis = sum(_visible(c, n) for n in lens)
        table = sum((_visible(c, n) + c["page"] - 1) // c["page"] for n in lens)
        return {"bytes": 2 * vis * c["kv_heads"] * c["dim"] * es + 2 * c["batch"] * c["heads"] * c["dim"] * es
                + 4 * table + 4 * c["batch"],
                "flops": 4 * vis * c["heads"] * c["dim"]}
    if c["op"] == "append":
        seq, pos = _append_tokens(c)
        live = sum(p >= 0 for p in pos)
        return {"bytes": 4 * live * c["kv_heads"] * c["dim"] * ES[c["dtype"]] + 8 * len(pos), "flops": 0}
    if c["op"] == "copy":
        page = c["kv_heads"] * c["page"] * c["dim"] * ES[c["dtype"]]
        return {"bytes": 4 * c["pairs"] * c["layers"] * page + 8 * c["pairs"], "flops": 0}
    es, groups = ES[c["dtype"]], c["k"] // c["group"]
    return {"bytes": c["n"] * (c["k"] // 2) + c["n"] * groups * (es + (1 if c["zeros"] else 0))
            + c["m"] * (c["n"] + c["k"]) * es,
            "flops": 2 * c["m"] * c["n"] * c["k"]}


# ---- inputs ----

def _inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DT.get(c["dtype"])

    def normal(*shape, std=1.0):
        return torch.empty(shape, device="cuda", dtype=torch.float32).normal_(0.0, std, generator=g).to(dt)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    def shuffled(n):
        return torch.randperm(n, generator=g, device="cuda").to(torch.int32)

    if c["op"] == "decode":
        lens = _lens(c)
        cols = max(1, (max(lens) + c["page"] - 1) // c["page"])
        pages = c["batch"] * cols
        return dict(q=normal(c["batch"], c["heads"], c["dim"], std=1.5), k=normal(*_pool_shape(c, pages)),
                    v=normal(*_pool_shape(c, pages)), table=shuffled(pages).reshape(c["batch"], cols).contiguous(),
                    lens=ints(lens))
    if c["op"] == "append":
        seq, pos = _append_tokens(c)
        cols = (max(pos) + c["page"]) // c["page"]
        pages = c["batch"] * cols
        return dict(k_new=normal(len(seq), c["kv_heads"], c["dim"]), v_new=normal(len(seq), c["kv_heads"], c["dim"]),
                    seq=ints(seq), pos=ints(pos), table=shuffled(pages).reshape(c["batch"], cols).contiguous(),
                    k=normal(*_pool_shape(c, pages)), v=normal(*_pool_shape(c, pages)))
    if c["op"] == "copy":
        shape = (c["layers"],) + _pool_shape(c, c["pages"])
        order = shuffled(c["pages"])
        pairs = torch.stack([order[:c["pairs"]], order[c["pairs"]:2 * c["pairs"]]], 1).contiguous()
        return dict(pairs=pairs, k=normal(*shape), v=normal(*shape))
    groups = c["k"] // c["group"]
    w = torch.randint(0, 256, (c["n"], c["k"] // 2), generator=g, device="cuda", dtype=torch.uint8)
    s = (torch.rand((c["n"], groups), generator=g, device="cuda") * 0.02 + 0.005).to(dt)
    d = dict(x=normal(c["m"], c["k"]), w=w, scales=s)
    if c["zeros"]:
        d["zeros"] = torch.randint(0, 16, (c["n"], groups), generator=g, device="cuda", dtype=torch.uint8)
    return d


def prepare(c, seed):
    st = dict(_inputs(c, seed), case=c)
    if not own:
        return st
    import irptx_b200 as irx
    if c["op"] == "matvec4":
        st["out"] = torch.empty((c["m"], c["n"]), device="cuda", dtype=DT[c["dtype"]])
        plan = irx.matvec4(c["m"], c["n"], c["k"], group=c["group"], dtype=c["dtype"], zeros=c["zeros"])
        args = [st["x"], st["w"], st["scales"]] + ([st["zeros"]] if c["zeros"] else []) + [st["out"]]
    elif c["op"] == "copy":
        cache = irx.KvCache(c["dtype"], c["kv_heads"], c["dim"], c["page"], c["pages"], order=c["order"])
        plan = irx.kv_copy(cache, c["pairs"], layers=c["layers"])
        args = [st["pairs"], st["k"], st["v"]]
    else:
        batch, cols = st["table"].shape
        cache = irx.KvCache(c["dtype"], c["kv_heads"], c["dim"], c["page"], st["k"].shape[0], batch=batch,
                            table_cols=cols, order=c["order"])
        if c["op"] == "append":
            plan = irx.kv_append(cache, st["k_new"].shape[0])
            args = [st["k_new"], st["v_new"], st["seq"], st["pos"], st["table"], st["k"], st["v"]]
        else:
            st["out"] = torch.empty_like(st["q"])
            plan = irx.decode(cache, c["heads"], window=c["window"], sinks=c["sinks"])
            args = [st["q"], st["k"], st["v"], st["table"], st["lens"], st["out"], plan.workspace()]
    st["plan"], st["args"] = plan, plan.bind(args)      # a decoding loop binds its buffers once
    return st


# ---- one pass ----

def run(st):
    c = st["case"]
    if own:
        st["plan"].launch(st["args"])
        return (st["k"], st["v"]) if c["op"] in ("append", "copy") else st["out"]
    return {"decode": _decode, "append": _append, "copy": _copy, "matvec4": _matvec4}[c["op"]](c, st)


def _decode(c, st):
    """Every sequence's keys and values gathered through the table, padded to the longest."""
    b, h, g, d = c["batch"], c["kv_heads"], c["heads"] // c["kv_heads"], c["dim"]
    k, v = st["k"][st["table"].long()], st["v"][st["table"].long()]
    if c["order"] == "head":
        k, v = k.transpose(2, 3), v.transpose(2, 3)
    k, v = k.reshape(b, -1, h, d).float(), v.reshape(b, -1, h, d).float()
    n = st["lens"].long()[:, None]
    pos = torch.arange(k.shape[1], device="cuda")[None, :]
    seen = pos < n
    if c["window"]:
        seen = seen & ((pos >= n - c["window"]) | (pos < c["sinks"]))
    q = st["q"].float().reshape(b, h, g, d) * (1.0 / math.sqrt(d))
    s = torch.einsum("bhgd,blhd->bhgl", q, k)
    s = torch.where(seen[:, None, None, :], s, torch.full_like(s, -1e30))
    p = torch.exp(s - s.amax(-1, keepdim=True)) * seen[:, None, None, :]
    o = torch.einsum("bhgl,blhd->bhgd", p, v) / p.sum(-1, keepdim=True).clamp_min(1e-30)
    return o.reshape(b, h * g, d).to(st["q"].dtype)


def _append(c, st):
    live = st["pos"] >= 0
    pos, seq = st["pos"].long().clamp_min(0), st["seq"].long()
    page, slot = st["table"].long()[seq, pos // c["page"]], pos % c["page"]
    page, slot = page[live], slot[live]
    for pool, new in (("k", "k_new"), ("v", "v_new")):
        if c["order"] == "head":
            st[pool][page, :, slot] = st[new][live]
        else:
            st[pool][page, slot] = st[new][live]
    return st["k"], st["v"]


def _copy(c, st):
    src, dst = st["pairs"][:, 0].long(), st["pairs"][:, 1].long()
    for pool in ("k", "v"):
        st[pool][:, dst] = st[pool][:, src]
    return st["k"], st["v"]


def _matvec4(c, st):
    n, k, group = c["n"], c["k"], c["group"]
    q = torch.stack([st["w"] & 15, st["w"] >> 4], -1).reshape(n, k // group, group).float()
    z = st["zeros"].float()[:, :, None] if c["zeros"] else 8.0
    w = ((q - z) * st["scales"].float()[:, :, None]).reshape(n, k)
    return (st["x"].float() @ w.t()).to(st["x"].dtype)


# ---- the definition in 64 bits ----

def exact(c, seed):
    """What `run` returns, from the definition: float64 numbers; append and copy, which only move
    values, by an index of where each page or slot comes from."""
    x = _inputs(c, seed)
    if c["op"] == "copy":
        come = list(range(c["pages"]))
        for src, dst in x["pairs"].tolist():
            come[dst] = src
        come = torch.tensor(come, device="cuda")
        return x["k"].index_select(1, come).double(), x["v"].index_select(1, come).double()
    if c["op"] == "append":
        table, res = x["table"].tolist(), []
        seq, pos = _append_tokens(c)
        went = [(t, table[s][p // c["page"]] * c["page"] + p % c["page"]) for t, (s, p) in enumerate(zip(seq, pos)) if p >= 0]
        tok, slot = torch.tensor(went, device="cuda").t()
        for pool, new in (("k", "k_new"), ("v", "v_new")):
            flat = (x[pool].transpose(1, 2) if c["order"] == "head" else x[pool]).double()
            shape = flat.shape                        # [page, slot, head, dim]
            flat = flat.reshape(-1, c["kv_heads"], c["dim"]).index_copy(0, slot, x[new].double().index_select(0, tok))
            flat = flat.reshape(shape)
            res.append(flat.transpose(1, 2).contiguous() if c["order"] == "head" else flat)
        return tuple(res)
    if c["op"] == "matvec4":
        out = torch.empty((c["m"], c["n"]), device="cuda", dtype=torch.float64)
        xd, step = x["x"].double(), max(1, (1 << 25) // c["k"])
        col = torch.arange(c["k"], device="cuda")
        for a in range(0, c["n"], step):
            rows = x["w"][a:a + step].to(torch.int64)
            nib = (rows[:, col // 2] >> (4 * (col % 2))) & 15
            zero = x["zeros"][a:a + step].to(torch.int64)[:, col // c["group"]] if c["zeros"] else 8
            out[:, a:a + step] = xd @ ((nib - zero).double() * x["scales"][a:a + step].double()[:, col // c["group"]]).t()
        return out
    d, g = c["dim"], c["heads"] // c["kv_heads"]
    out = torch.zeros((c["batch"], c["heads"], d), device="cuda", dtype=torch.float64)
    for b, n in enumerate(_lens(c)):
        if n == 0:
            continue                                  # nothing to see: zeros
        keep = list(range(n))
        if c["window"] and n > c["window"]:
            keep = list(range(min(c["sinks"], n - c["window"]))) + list(range(n - c["window"], n))
        at = torch.tensor(keep, device="cuda")
        page, slot = x["table"][b].long()[at // c["page"]], at % c["page"]
        for h in range(c["kv_heads"]):
            ks = x["k"][page, h, slot] if c["order"] == "head" else x["k"][page, slot, h]
            vs = x["v"][page, h, slot] if c["order"] == "head" else x["v"][page, slot, h]
            s = x["q"][b, h * g:(h + 1) * g].double() @ ks.double().t() / math.sqrt(d)
            out[b, h * g:(h + 1) * g] = torch.softmax(s, -1) @ vs.double()
    return out
