"""The serving operators without a GPU: plans, refusals, the weight packing and the page manager."""
import random

import numpy as np
import pytest


def refused(irx, code, f, *a, **k):
    with pytest.raises(irx.IrxError) as e:
        f(*a, **k)
    assert e.value.code == code, e.value.line
    assert e.value.line.startswith(f"error[E{code:03d}]: irptx: cannot lower ")


def cache(irx, **k):
    d = dict(dtype="bf16", heads=2, head_dim=64, page_size=16, pages=8, batch=3, table_cols=4)
    d.update(k)
    return irx.KvCache(**d)


def test_plans_state_their_arguments(irx):
    c = cache(irx)
    p = irx.decode(c, 8, lse=True)
    assert p.family == "decode" and [a.name for a in p.args] == ["q", "k", "v", "table", "lens", "out", "lse", "workspace"]
    assert [a.kind for a in p.args] == ["in"] * 5 + ["out", "out", "work"]
    assert [a.dtype for a in p.args] == ["bf16"] * 3 + ["i32"] * 2 + ["bf16", "f32", "u8"]
    assert p.args[1].shape == (8, 2, 16, 64) and p.args[1].elems == 8 * 2 * 16 * 64
    assert p.units() == 2 and "decode batch=3 heads=8 kv_heads=2" in p.describe()
    b, f = p.work()                                       # a full cache
    assert b == 2 * 3 * 64 * 2 * 64 * 2 + 2 * 3 * 8 * 64 * 2 and f == 4 * 3 * 64 * 8 * 64
    assert irx.decode(cache(irx, order="token"), 8).args[1].shape == (8, 16, 2, 64)
    a = irx.kv_append(c, 5)
    assert a.family == "kv_append" and a.units() == 5 and [x.kind for x in a.args] == ["in"] * 5 + ["out"] * 2
    y = irx.kv_copy(c, 3, layers=2)
    assert y.family == "kv_copy" and y.args[1].shape == (2, 8, 2, 16, 64) and y.work()[0] == 4 * 3 * 2 * 2 * 16 * 64 * 2 + 24
    m = irx.matvec4(3, 10, 100, group=32, zeros=True, scale_dtype="f32")
    assert [(x.name, x.dtype, x.shape) for x in m.args] == [("x", "bf16", (3, 100)), ("w", "u8", (10, 50)), ("scales", "f32", (10, 4)),
                                                            ("zeros", "u8", (10, 4)), ("y", "bf16", (3, 10))]
    assert m.shard(1, 4) == (3, 6, "none")


def test_windowed_work_counts_the_visible_keys(irx):
    c = cache(irx, batch=1)
    full, win = irx.decode(c, 2).work()[0], irx.decode(c, 2, window=10, sinks=3).work()[0]
    assert full - win == 2 * (64 - 13) * 2 * 64 * 2


@pytest.mark.parametrize("bad,code", [(dict(dtype="f16"), 24), (dict(heads=0), 42), (dict(head_dim=0), 42), (dict(head_dim=257), 42),
                                      (dict(page_size=0), 42), (dict(pages=0), 42), (dict(batch=0), 42), (dict(table_cols=0), 42),
                                      (dict(page_size=1 << 20, table_cols=1 << 20), 42), (dict(pages=1 << 31), 42),
                                      (dict(strides=(2048, 1024, 63)), 41), (dict(strides=(2047, 1024, 64)), 41),
                                      (dict(strides=(2048, 1024, -64)), 42), (dict(strides=(0, 1024, 64)), 41)])
def test_cache_refusals(irx, bad, code):
    def build():
        c = cache(irx, **bad)
        irx.decode(c, 2 * max(1, c.heads))
    refused(irx, code, build)


def test_overlap_is_told_from_interleaving(irx):
    irx.decode(cache(irx, strides=(64, 8 * 64 * 16, 8 * 64)), 2)            # pages innermost: no overlap
    refused(irx, 41, lambda: irx.decode(cache(irx, strides=(64, 8 * 64 * 15, 8 * 64)), 2))
    irx.decode(cache(irx, heads=1, strides=(1024, 0, 64)), 2)               # an axis of one needs no stride


def test_operator_refusals(irx):
    c = cache(irx)
    refused(irx, 42, irx.decode, c, 3)
    refused(irx, 42, irx.decode, c, 0)
    refused(irx, 42, irx.decode, c, 4, window=-1)
    refused(irx, 42, irx.decode, c, 4, sinks=2)
    refused(irx, 42, irx.decode, c, 4, scale=float("nan"))
    refused(irx, 42, irx.decode, c, 4, scale=float("inf"))
    refused(irx, 42, irx.decode, c, 4, q_stride=255)
    refused(irx, 42, irx.kv_append, c, 0)
    refused(irx, 42, irx.kv_append, c, 4, stride=100)
    refused(irx, 42, irx.kv_copy, c, 0)
    refused(irx, 42, irx.kv_copy, c, 1, layers=0)
    refused(irx, 41, irx.kv_copy, c, 1, layers=2, layer_stride=100)
    for bad in (dict(m=0), dict(n=0), dict(k=0), dict(group=0), dict(x_stride=10), dict(w_stride=3), dict(m=1 << 31)):
        refused(irx, 42, irx.matvec4, **{**dict(m=1, n=4, k=64), **bad})
    refused(irx, 24, irx.matvec4, 1, 4, 64, dtype="f16")
    refused(irx, 93, irx.kv_append(c, 4).workspace)
    refused(irx, 93, irx.decode(c, 4).run_host, [np.zeros(1, np.float32)] * 7)
    refused(irx, 93, irx.decode(c, 4).host_chunks)
    refused(irx, 93, irx.matvec4(1, 4, 64).source)


def test_pack4(irx):
    import torch
    q = np.random.default_rng(0).integers(0, 16, (5, 7))
    w = irx.pack4(q)
    assert w.shape == (5, 4) and w.dtype == np.uint8
    assert all((int(w[r, k // 2]) >> (4 * (k % 2))) & 15 == q[r, k] for r in range(5) for k in range(7))
    assert np.array_equal(irx.pack4(torch.from_numpy(q)).numpy(), w)
    refused(irx, 42, irx.pack4, q + 1 + 15)
    refused(irx, 42, irx.pack4, torch.from_numpy(q) - 16)


# ---- the page manager, against a model that keeps each sequence's tokens ----

def test_pages_refusals(irx):
    refused(irx, 42, irx.Pages, 0, 4, 2, 2)
    m = irx.Pages(3, 4, 2, 4)
    refused(irx, 93, m.extend, 0)
    refused(irx, 93, m.close, 1)
    refused(irx, 93, m.fork, -1)
    a = m.open()
    refused(irx, 93, m.extend, a, -1)
    assert m.extend(a, 12) is None and m.free == 0
    refused(irx, 94, m.extend, a)                          # out of pages, and nothing has changed
    assert m.length(a) == 12 and m.free == 0
    b = m.fork(a)
    refused(irx, 81, m.open)
    refused(irx, 81, m.fork, a)
    refused(irx, 81, m.extend, b, 5)                       # past its row
    m.close(a)
    assert m.free == 0 and m.length(a) == -1
    m.close(b)
    assert m.free == 3 and (m.table == -1).all()


@pytest.mark.parametrize("seed", range(6))
def test_pages_keep_every_sequences_tokens(irx, seed):
    rng = random.Random(seed)
    pages, ps, seqs, cols = rng.choice([7, 24, 60]), rng.choice([1, 3, 4, 16]), 5, 9
    m = irx.Pages(pages, ps, seqs, cols)
    pool, model, fresh = {}, {}, 0                         # (page, slot) -> token; sequence -> its tokens

    def copy(pairs):
        src, dst = [p[0] for p in pairs], [p[1] for p in pairs]
        assert len(set(dst)) == len(dst) and not set(src) & set(dst)
        for s, d in pairs:
            for t in range(ps):
                pool[d, t] = pool.get((s, t))

    for _ in range(400):
        op = rng.choice(["open", "extend", "extend", "extend", "fork", "close", "compact"])
        seq = rng.choice(list(model)) if model else None
        try:
            if op == "open":
                model[m.open()] = []
            elif op == "compact":
                copy(m.compact())
                assert {int(p) for p in m.table.reshape(-1) if p >= 0} == set(range(pages - m.free))
            elif seq is None:
                continue
            elif op == "extend":
                n = rng.randrange(0, 2 * ps + 1)
                pair = m.extend(seq, n)
                if pair:
                    copy([pair])
                for _ in range(n):
                    pos = len(model[seq])
                    pool[int(m.table[seq, pos // ps]), pos % ps] = fresh
                    model[seq].append(fresh)
                    fresh += 1
            elif op == "fork":
                model[m.fork(seq)] = list(model[seq])
            else:
                m.close(seq)
                del model[seq]
        except irx.IrxError as e:
            assert e.code in (81, 94)
        t = m.table
        for s, toks in model.items():
            assert m.length(s) == len(toks)
            assert [pool[int(t[s, j // ps]), j % ps] for j in range(len(toks))] == toks
            assert (t[s, -(-len(toks) // ps):] == -1).all()
        held = {int(p) for p in t.reshape(-1) if p >= 0}
        assert m.free == pages - len(held)
