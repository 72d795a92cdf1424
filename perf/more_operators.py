"""The operators of a model's step around the cache: rotary positions, alone and on the way into a paged
cache, causal attention over packed prompts, and the draw of the next token, as cases that can be
measured.

``listed()`` gives the named cases, ``draw(rng)`` one more of the same ranges. ``prepare(case,
seed)`` makes what a program has in hand (activations, positions, pools, logits, random numbers,
the plan), ``run(state)`` is one pass, ``work(case)`` the bytes and operations it cannot do without
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
        # a decoding step of a batch: the queries and keys of a fused projection's rows, before an append
        dict(name="rope step", op="rope", dtype="bf16", tokens=32, heads=40, dim=128, rot=128, inter=False, back=False,
             scaling="none", factor=1.0, original=0, start=1021, extra=1024),
        # gradients through the rotation of a long context: interleaved pairs in half of each head, scaled frequencies
        dict(name="rope backward long f32", op="rope", dtype="f32", tokens=16381, heads=32, dim=128, rot=64, inter=True,
             back=True, scaling="yarn", factor=16.0, original=8192, start=115001, extra=0),
        # one new token for each sequence of a serving batch, one slot empty
        dict(name="append step", op="append", dtype="bf16", batch=32, heads=32, kv_heads=8, dim=128, rot=128, inter=False,
             scaling="none", factor=1.0, original=0, page=16, start=1021, new=1, pad=1, order="head"),
        # the prompts of a batch going in, padded to one length
        dict(name="append prompts", op="append", dtype="bf16", batch=8, heads=32, kv_heads=8, dim=128, rot=128, inter=False,
             scaling="linear", factor=4.0, original=0, page=16, start=3, new=2047, pad=40, order="head"),
        # one short question: the smallest prompt, all latency
        dict(name="prompt one short", op="prompt", dtype="bf16", heads=32, kv_heads=8, dim=128, batch=1, lo=37, hi=37,
             window=0, sinks=0, behind=0),
        # prompts of a serving batch, packed, with rows of padding behind the last
        dict(name="prompt batch ragged", op="prompt", dtype="bf16", heads=32, kv_heads=8, dim=128, batch=16, lo=1, hi=2048,
             window=0, sinks=0, behind=13),
        # one long document
        dict(name="prompt long", op="prompt", dtype="bf16", heads=32, kv_heads=8, dim=128, batch=1, lo=16001, hi=16001,
             window=0, sinks=0, behind=0),
        # a sliding window with the first tokens kept, a key-value head for every query head, small heads
        dict(name="prompt window sinks", op="prompt", dtype="bf16", heads=32, kv_heads=32, dim=64, batch=2, lo=7001, hi=8190,
             window=1024, sinks=4, behind=0),
        # f32 activations, as f32 graphs have
        dict(name="prompt f32", op="prompt", dtype="f32", heads=16, kv_heads=4, dim=128, batch=5, lo=200, hi=701,
             window=0, sinks=0, behind=0),
        # one answer being written: one row of a large vocabulary through every filter
        dict(name="sample one row", op="sample", dtype="f32", rows=1, vocab=128001, filters="kpm", banned=0),
        # a batch whose requests ask for different things, greedy among them; banned tokens are at minus infinity
        dict(name="sample batch mixed", op="sample", dtype="f32", rows=64, vocab=128001, filters="mixed", banned=64),
        # many rows of a large bf16 vocabulary, full of equal logits, top-p over all of it
        dict(name="sample many bf16", op="sample", dtype="bf16", rows=256, vocab=151999, filters="p", banned=0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_rot(rng, dim):
    rot = rng.choice([dim, dim, dim // 2, 2 * max(1, dim // 8)])
    scaling = rng.choice(["none", "none", "linear", "ntk", "yarn"])
    return dict(rot=rot, inter=rng.random() < 0.4, scaling=scaling, factor=1.0 if scaling == "none" else rng.choice([2.0, 4.0, 16.0]),
                original=rng.choice([4096, 8192]) if scaling == "yarn" else 0)


def draw(rng):
    op = rng.choice(["rope", "append", "prompt", "prompt", "sample", "sample"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op == "sample":
        rows = _log_int(rng, 1, 512)
        return dict(op=op, dtype=dtype, rows=rows, vocab=min(_log_int(rng, 500, 262144), 256 * 151999 // rows),
                    filters=rng.choice(["none", "k", "p", "m", "kp", "kpm", "mixed", "mixed"]), banned=rng.choice([0, 64]))
    dim = rng.choice([64, 80, 96, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8, 16])
    group = rng.choice([1, 2, 3, 4, 7, 8])
    if op == "rope":
        tokens = max(1, min(_log_int(rng, 1, 16384), (1 << 26) // (kv_heads * group * dim)))
        return dict(op=op, dtype=dtype, tokens=tokens, heads=kv_heads * group, dim=dim, back=rng.random() < 0.4,
                    start=_log_int(rng, 1, 1 << 20), extra=rng.choice([0, 0, dim, 1024]), **_draw_rot(rng, dim))
    if op == "append":
        batch = _log_int(rng, 1, 32)
        new = max(1, min(2048, _log_int(rng, 1, 2048), (1 << 25) // (kv_heads * group * dim * batch)))
        return dict(op=op, dtype=dtype, batch=batch, heads=kv_heads * group, kv_heads=kv_heads, dim=dim,
                    page=rng.choice([1, 8, 16, 16, 24, 32, 64, 128]), start=rng.randrange(0, 500), new=new,
                    pad=rng.randrange(0, 4), order=rng.choice(["head", "token"]), **_draw_rot(rng, dim))
    batch = _log_int(rng, 1, 24)
    heads = min(64, kv_heads * group) // kv_heads * kv_heads
    # pairs of tokens and the head's numbers stay below the long document's; f32 below a sixteenth of that
    most = 16001 ** 2 * 32 * 128 // (heads * dim * batch) // (16 if dtype == "f32" or dim > 128 else 1)
    hi = max(1, min(_log_int(rng, 1, 16001), int(math.sqrt(most))))
    windowed = rng.random() < 0.35
    return dict(op=op, dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim, batch=batch, lo=rng.randrange(max(1, hi // 8), hi + 1),
                hi=hi, window=_log_int(rng, 1, hi) if windowed else 0, sinks=rng.choice([0, 1, 4]) if windowed else 0,
                behind=rng.choice([0, 0, 5]))


# ---- sizes that follow from a case ----

def _lens(c):
    """The prompts' lengths: from lo to hi, spread by the golden ratio's multiples."""
    return [int(round(c["lo"] + ((b * 0.6180339887498949) % 1.0) * (c["hi"] - c["lo"]))) for b in range(c["batch"])]


def _pairs(c, n):
    """How many keys the n tokens of a prompt see, together."""
    w = c["window"]
    if not w or n <= w:
        return n * (n + 1) // 2
    seen = w * (w + 1) // 2 + (n - w) * w
    before = n - w                                    # the last token has this many keys before its window
    s = min(c["sinks"], before)
    return seen + s * (s + 1) // 2 + (before - s) * s


def _append_tokens(c):
    """(sequence, position) of every new token; position -1 marks padding."""
    seq, pos = [], []
    for b in range(c["batch"]):
        fill = c["new"] - (b * c["pad"]) % max(1, c["new"])
        for j in range(c["new"]):
            seq.append(b)
            pos.append(c["start"] + b + j if j < fill else -1)
    if c["new"] == 1 and c["batch"] > 2:
        pos[1] = -1                                   # a slot that holds no request
    return seq, pos


def _pool_shape(c, pages):
    if c["order"] == "head":
        return (pages, c["kv_heads"], c["page"], c["dim"])
    return (pages, c["page"], c["kv_heads"], c["dim"])


def _amplitude(c):
    return 0.1 * math.log(c["factor"]) + 1.0 if c["scaling"] == "yarn" else 1.0


def work(c):
    if c["op"] == "rope":
        n = c["tokens"] * c["heads"]
        return {"bytes": 2 * n * c["dim"] * ES[c["dtype"]] + 4 * c["tokens"], "flops": 3 * n * c["rot"]}
    if c["op"] == "append":
        _, pos = _append_tokens(c)
        live = sum(p >= 0 for p in pos)
        return {"bytes": 2 * live * (c["heads"] + 2 * c["kv_heads"]) * c["dim"] * ES[c["dtype"]] + 8 * len(pos),
                "flops": 3 * live * (c["heads"] + c["kv_heads"]) * c["rot"]}
    if c["op"] == "prompt":
        lens = _lens(c)
        return {"bytes": 2 * sum(lens) * (c["heads"] + c["kv_heads"]) * c["dim"] * ES[c["dtype"]] + 4 * (c["batch"] + 1),
                "flops": 4 * sum(_pairs(c, n) for n in lens) * c["heads"] * c["dim"]}
    return {"bytes": c["rows"] * (c["vocab"] * ES[c["dtype"]] + 28), "flops": c["rows"] * c["vocab"]}


# ---- inputs ----

def _inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DT[c["dtype"]]

    def normal(*shape, std=1.0):
        return torch.empty(shape, device="cuda", dtype=torch.float32).normal_(0.0, std, generator=g).to(dt)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    if c["op"] == "rope":
        wide = normal(c["tokens"], c["heads"] * c["dim"] + c["extra"])         # rows of a fused projection
        x = wide[:, :c["heads"] * c["dim"]].unflatten(1, (c["heads"], c["dim"]))
        return dict(x=x, pos=torch.arange(c["start"], c["start"] + c["tokens"], dtype=torch.int32, device="cuda"))
    if c["op"] == "append":
        seq, pos = _append_tokens(c)
        cols = (max(pos) + c["page"]) // c["page"]
        pages = c["batch"] * cols
        h, kv = c["heads"], c["kv_heads"]
        rows = normal(len(seq), h + 2 * kv, c["dim"])
        table = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).reshape(c["batch"], cols).contiguous()
        return dict(q=rows[:, :h], k_new=rows[:, h:h + kv], v_new=rows[:, h + kv:], seq=ints(seq), pos=ints(pos), table=table,
                    q_out=torch.zeros(len(seq), h, c["dim"], device="cuda", dtype=dt),
                    k=normal(*_pool_shape(c, pages)), v=normal(*_pool_shape(c, pages)))
    if c["op"] == "prompt":
        lens = _lens(c)
        starts = [0]
        for n in lens:
            starts.append(starts[-1] + n)
        h, kv = c["heads"], c["kv_heads"]
        rows = normal(starts[-1] + c["behind"], h + 2 * kv, c["dim"], std=1.2)
        return dict(q=rows[:, :h], k=rows[:, h:h + kv], v=rows[:, h + kv:], starts=ints(starts),
                    out=torch.zeros(starts[-1] + c["behind"], h, c["dim"], device="cuda", dtype=dt))
    m, n = c["rows"], c["vocab"]
    x = torch.empty(m, n, device="cuda").normal_(0.0, 2.0, generator=g)
    x += 9.0 * torch.rand(m, n, generator=g, device="cuda").pow_(400.0)        # a few tokens stand out
    if c["banned"]:
        x[:, torch.randperm(n, generator=g, device="cuda")[:n // c["banned"]]] = -math.inf
    kinds = ["greedy", "none", "k", "p", "m", "kp", "kpm"] if c["filters"] == "mixed" else [c["filters"]]
    kinds = [kinds[i % len(kinds)] for i in range(m)]

    def each(f):
        return torch.tensor([f(i, kind) for i, kind in enumerate(kinds)], device="cuda")

    return dict(logits=x.to(dt), temperature=each(lambda i, kind: 0.0 if kind == "greedy" else 0.6 + 0.2 * (i % 5)).float(),
                top_k=each(lambda i, kind: 20 + 30 * (i % 4) if "k" in kind else 0).int(),
                top_p=each(lambda i, kind: 0.8 + 0.05 * (i % 4) if "p" in kind else 1.0).float(),
                min_p=each(lambda i, kind: 0.02 + 0.01 * (i % 5) if "m" in kind else 0.0).float(),
                u=torch.rand(m, generator=g, device="cuda"))


def prepare(c, seed):
    st = dict(_inputs(c, seed), case=c)
    if not own:
        return st
    import irptx_b200 as irx
    if c["op"] in ("rope", "append"):
        freqs = irx.rope_freqs(c["rot"], scaling=c["scaling"], factor=c["factor"], original=c["original"])
    if c["op"] == "rope":
        st["out"] = torch.empty(c["tokens"], c["heads"], c["dim"], device="cuda", dtype=DT[c["dtype"]])
        plan = irx.rope(c["tokens"], c["heads"], c["dim"], freqs, dtype=c["dtype"], interleaved=c["inter"],
                        amplitude=_amplitude(c), backward=c["back"], x_stride=c["heads"] * c["dim"] + c["extra"])
        args = [st["x"], st["pos"], st["out"]]
    elif c["op"] == "append":
        batch, cols = st["table"].shape
        cache = irx.KvCache(c["dtype"], c["kv_heads"], c["dim"], c["page"], st["k"].shape[0], batch=batch,
                            table_cols=cols, order=c["order"])
        plan = irx.rope_append(cache, st["pos"].shape[0], c["heads"], freqs, interleaved=c["inter"],
                               amplitude=_amplitude(c), stride=(c["heads"] + 2 * c["kv_heads"]) * c["dim"])
        args = [st["q"], st["k_new"], st["v_new"], st["seq"], st["pos"], st["table"], st["q_out"], st["k"], st["v"]]
    elif c["op"] == "prompt":
        wide = (c["heads"] + 2 * c["kv_heads"]) * c["dim"]
        plan = irx.prompt(st["q"].shape[0], c["batch"], c["heads"], c["kv_heads"], c["dim"], dtype=c["dtype"],
                          window=c["window"], sinks=c["sinks"], q_stride=wide, kv_stride=wide)
        args = [st["q"], st["k"], st["v"], st["starts"], st["out"]]
    else:
        st["token"] = torch.empty(c["rows"], dtype=torch.int32, device="cuda")
        st["logprob"] = torch.empty(c["rows"], dtype=torch.float32, device="cuda")
        plan = irx.sample(c["rows"], c["vocab"], dtype=c["dtype"], logprob=True)
        args = [st["logits"], st["temperature"], st["top_k"], st["top_p"], st["min_p"], st["u"], st["token"], st["logprob"]]
    st["plan"], st["args"] = plan, plan.bind(args)      # a serving loop binds its buffers once
    return st


# ---- one pass ----

def run(st):
    c = st["case"]
    if own:
        st["plan"].launch(st["args"])
        return {"rope": lambda: st["out"], "append": lambda: (st["q_out"], st["k"], st["v"]), "prompt": lambda: st["out"],
                "sample": lambda: (st["token"], st["logprob"])}[c["op"]]()
    return {"rope": _rope, "append": _append, "prompt": _prompt, "sample": _sample}[c["op"]](c, st)


def _freqs(c):
    """Radians a position, float64 [rot / 2]. linear: every frequency divided by the factor; ntk: the base
    stretched so that the slowest is; yarn: those that turn less than once in the original context
    divided, those that turn more than 32 times kept, a ramp between."""
    r, base = c["rot"], 10000.0
    i = torch.arange(r // 2, dtype=torch.float64)
    if c["scaling"] == "ntk":
        base *= c["factor"] ** (r / (r - 2.0)) if r > 2 else 1.0
    f = base ** (-2.0 * i / r)
    if c["scaling"] == "linear":
        f = f / c["factor"]
    if c["scaling"] == "yarn":
        def turns(n):
            return r * math.log(c["original"] / (n * 2.0 * math.pi)) / (2.0 * math.log(base))
        low, high = max(math.floor(turns(32.0)), 0), min(math.ceil(turns(1.0)), r - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
        f = f / c["factor"] * ramp + f * (1.0 - ramp)
    return f


def _rotate(c, x, pos, sign=1.0):
    """x [tokens, heads, dim] turned by its positions' angles; angles in 64 bits, the rest in 32."""
    r = c["rot"]
    angle = pos.double()[:, None] * _freqs(c).to(x.device)[None, :]
    cos, sin = (t.float()[:, None, :] * _amplitude(c) for t in (torch.cos(angle), sign * torch.sin(angle)))
    y = x.float().clone()
    a, b = (y[..., 0:r:2].clone(), y[..., 1:r:2].clone()) if c["inter"] else (y[..., :r // 2].clone(), y[..., r // 2:r].clone())
    p, q = a * cos - b * sin, a * sin + b * cos
    if c["inter"]:
        y[..., 0:r:2], y[..., 1:r:2] = p, q
    else:
        y[..., :r // 2], y[..., r // 2:r] = p, q
    return y.to(x.dtype)


def _rope(c, st):
    return _rotate(c, st["x"], st["pos"], -1.0 if c["back"] else 1.0)


def _append(c, st):
    live = st["pos"] >= 0
    pos, seq = st["pos"].long().clamp_min(0), st["seq"].long()
    page, slot = st["table"].long()[seq, pos // c["page"]], pos % c["page"]
    page, slot = page[live], slot[live]
    st["q_out"][live] = _rotate(c, st["q"], pos)[live]
    for pool, new in (("k", _rotate(c, st["k_new"], pos)), ("v", st["v_new"])):
        if c["order"] == "head":
            st[pool][page, :, slot] = new[live]
        else:
            st[pool][page, slot] = new[live]
    return st["q_out"], st["k"], st["v"]


def _prompt(c, st):
    """Each prompt by itself, its queries in runs so that the scores stay below two gigabytes."""
    d, kv, g = c["dim"], c["kv_heads"], c["heads"] // c["kv_heads"]
    first = 0
    for n in _lens(c):
        rows = slice(first, first + n)
        first += n
        q = st["q"][rows].float().unflatten(1, (kv, g)).permute(1, 2, 0, 3) * (1.0 / math.sqrt(d))   # [kv, g, n, d]
        k, v = (st[t][rows].float().transpose(0, 1)[:, None] for t in ("k", "v"))                    # [kv, 1, n, d]
        step = max(1, (1 << 29) // (c["heads"] * n))
        for a in range(0, n, step):
            b = min(n, a + step)
            i, j = torch.arange(a, b, device="cuda")[:, None], torch.arange(b, device="cuda")[None, :]
            seen = j <= i
            if c["window"]:
                seen = seen & ((j > i - c["window"]) | (j < c["sinks"]))
            s = q[:, :, a:b] @ k[:, :, :b].transpose(2, 3)
            s.masked_fill_(~seen, -math.inf)
            s.sub_(s.amax(-1, keepdim=True)).exp_()
            o = (s @ v[:, :, :b]).div_(s.sum(-1, keepdim=True))
            st["out"][rows][a:b] = o.permute(2, 0, 1, 3).flatten(1, 2).to(st["out"].dtype)
    return st["out"]


def _sample(c, st):
    """Filters on the tokens in order of their logits, equal ones by index, the draw in order of index; in 64
    bits, since a sum next to a border decides which token it is."""
    x = st["logits"].double()
    n = x.shape[1]
    x, order = torch.sort(x, dim=1, descending=True, stable=True)
    t = st["temperature"].double()[:, None]
    w = torch.exp((x - x[:, :1]) / torch.where(t > 0, t, 1.0))
    rank = torch.arange(n, device="cuda")[None, :]
    k, p = st["top_k"].long()[:, None], st["top_p"].double()[:, None]
    w = torch.where((k <= 0) | (rank < k), w, 0.0)
    before = torch.cumsum(w, 1) - w
    w = torch.where((p >= 1.0) | (rank == 0) | (before < p * w.sum(1, keepdim=True)), w, 0.0)
    w = torch.where(w >= st["min_p"].double()[:, None], w, 0.0)
    w = torch.zeros_like(w).scatter_(1, order, w)
    total = w.sum(1, keepdim=True)
    token = (torch.cumsum(w, 1) <= st["u"].double()[:, None] * total).sum(1, keepdim=True)
    last = (w * 0.0 + (w > 0) * rank).amax(1, keepdim=True).long()
    token = torch.minimum(token, last)
    token = torch.where(t > 0, token, order[:, :1])
    logprob = torch.log(w.gather(1, token) / total)
    logprob = torch.where(t > 0, logprob, 0.0)
    return token[:, 0].int(), logprob[:, 0].float()


# ---- the definition in 64 bits ----

def _turned(c, x, pos, back):
    """The rotation as complex numbers."""
    r = c["rot"]
    x = x.double().clone()
    z = torch.polar(torch.full((len(pos), r // 2), _amplitude(c), dtype=torch.float64, device=x.device),
                    torch.outer(pos.double(), _freqs(c).to(x.device)))[:, None]
    z = z.conj() if back else z
    even, odd = (slice(0, r, 2), slice(1, r, 2)) if c["inter"] else (slice(0, r // 2), slice(r // 2, r))
    y = torch.complex(x[..., even], x[..., odd]) * z
    x[..., even], x[..., odd] = y.real, y.imag
    return x


def exact(c, seed):
    """What `run` returns, from the definition in 64 bits."""
    x = _inputs(c, seed)
    if c["op"] == "rope":
        return _turned(c, x["x"], x["pos"], c["back"])
    if c["op"] == "append":
        table = x["table"].tolist()
        seq, pos = _append_tokens(c)
        went = [(i, table[s][p // c["page"]] * c["page"] + p % c["page"]) for i, (s, p) in enumerate(zip(seq, pos)) if p >= 0]
        tok, slot = torch.tensor(went, device="cuda").t()
        at = x["pos"][tok]
        res = [x["q_out"].double().index_copy(0, tok, _turned(c, x["q"][tok], at, False))]
        for pool, new in (("k", _turned(c, x["k_new"][tok], at, False)), ("v", x["v_new"][tok].double())):
            flat = (x[pool].transpose(1, 2) if c["order"] == "head" else x[pool]).double()
            shape = flat.shape                        # [page, slot, head, dim]
            flat = flat.reshape(-1, c["kv_heads"], c["dim"]).index_copy(0, slot, new).reshape(shape)
            res.append(flat.transpose(1, 2).contiguous() if c["order"] == "head" else flat)
        return tuple(res)
    if c["op"] == "prompt":
        d, g, first = c["dim"], c["heads"] // c["kv_heads"], 0
        out = x["out"].double()
        for n in _lens(c):
            for h in range(c["heads"]):
                q, k, v = (x[t][first:first + n, i].double() for t, i in (("q", h), ("k", h // g), ("v", h // g)))
                for a in range(0, n, 4096):
                    b = min(n, a + 4096)
                    s = q[a:b] @ k[:b].t() / math.sqrt(d)
                    far = torch.arange(a, b, device="cuda")[:, None] - torch.arange(b, device="cuda")[None, :]
                    gone = far < 0
                    if c["window"]:
                        gone |= (far >= c["window"]) & (torch.arange(b, device="cuda") >= c["sinks"])[None, :]
                    out[first + a:first + b, h] = torch.softmax(s.masked_fill(gone, -math.inf), -1) @ v[:b]
            first += n
        return out
    tokens, logs = [], []
    for i in range(c["rows"]):                        # one row after the other, kept as a set of indexes
        row = x["logits"][i].double()
        t, k, p, least, u = (float(x[f][i]) for f in ("temperature", "top_k", "top_p", "min_p", "u"))
        if not t > 0:
            tokens.append(int((row == row.max()).nonzero()[0]))
            logs.append(0.0)
            continue
        e = torch.exp((row - row.max()) / t)
        kept = torch.argsort(row, descending=True, stable=True)
        if k > 0:
            kept = kept[:int(k)]
        if p < 1.0:
            sums = torch.cumsum(e[kept], 0)
            kept = kept[:int((sums < p * sums[-1]).sum()) + 1]
        kept = torch.sort(kept[e[kept] >= least]).values
        sums = torch.cumsum(e[kept], 0)
        j = min(int((sums <= u * sums[-1]).sum()), int(e[kept].nonzero()[-1]))
        tokens.append(int(kept[j]))
        logs.append(float(torch.log(e[kept[j]] / sums[-1])))
    return torch.tensor(tokens, device="cuda").int(), torch.tensor(logs, device="cuda", dtype=torch.float64)
