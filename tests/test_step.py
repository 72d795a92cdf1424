"""The operators around the cache without a GPU: plans, refusals, rotation frequencies."""
import math

import numpy as np
import pytest

NAN, INF = math.nan, math.inf


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
    f = irx.rope_freqs(64)
    p = irx.rope(5, 3, 64, f, x_stride=256)
    assert p.family == "rope" and [(a.name, a.kind, a.dtype, a.shape, a.stride) for a in p.args] == [
        ("x", "in", "bf16", (5, 3, 64), (256, 64, 1)), ("pos", "in", "i32", (5,), (1,)), ("y", "out", "bf16", (5, 3, 64), (192, 64, 1))]
    assert p.args[0].elems == 4 * 256 + 192 and p.work() == (2 * 5 * 3 * 64 * 2 + 20, 5 * 3 * 32 * 6) and p.shard(1, 2) == (3, 5, "none")
    p = irx.rope_append(cache(irx), 5, 4, f, stride=512)
    assert p.family == "rope_append" and p.units() == 5
    assert [a.name for a in p.args] == ["q", "k", "v", "seq", "pos", "table", "q_out", "k_pool", "v_pool"]
    assert p.args[1].shape == (5, 2, 64) and p.args[1].stride == (512, 64, 1) and p.args[6].shape == (5, 4, 64)
    assert p.args[7].shape == (8, 2, 16, 64) and p.work()[0] == 2 * 5 * 8 * 64 * 2 + 40
    p = irx.prompt(100, 3, 8, 2, 64, lse=True, kv_stride=999)
    assert p.family == "prompt" and p.units() == 2 and [a.shape for a in p.args] == [(100, 8, 64), (100, 2, 64), (100, 2, 64), (4,), (100, 8, 64), (100, 8)]
    assert p.args[1].stride == (999, 64, 1) and p.args[5].dtype == "f32"
    assert p.work() == (2 * 100 * 10 * 64 * 2, 4 * 5050 * 8 * 64)
    p = irx.sample(7, 1000, stride=1024, logprob=True)
    assert p.family == "sample" and p.units() == 7 and [a.dtype for a in p.args] == ["f32", "f32", "i32", "f32", "f32", "f32", "i32", "f32"]
    assert p.work()[0] == 7 * 4028 and "vocab=1000" in p.describe()


@pytest.mark.parametrize("n,window,sinks", [(9, 4, 0), (9, 4, 2), (9, 4, 30), (9, 9, 3), (9, 30, 3), (1, 1, 1)])
def test_prompt_work_counts_the_visible_pairs(irx, n, window, sinks):
    seen = sum(j > i - window or j < sinks for i in range(n) for j in range(i + 1))
    assert irx.prompt(n, 1, 1, 1, 8, window=window, sinks=sinks).work()[1] == 4 * seen * 8


def test_refusals(irx):
    f = irx.rope_freqs(64)
    for k in (dict(tokens=0), dict(heads=0), dict(head_dim=0), dict(head_dim=257), dict(head_dim=62), dict(freqs=[]), dict(freqs=[NAN]),
              dict(freqs=[1025.0]), dict(amplitude=INF), dict(x_stride=100), dict(y_stride=-1), dict(tokens=1 << 31), dict(heads=1 << 15),
              dict(x_stride=1 << 41)):
        refused(irx, 42, irx.rope, **{**dict(tokens=2, heads=4, head_dim=64, freqs=f), **k})
    refused(irx, 24, irx.rope, 2, 4, 64, f, dtype="f16")
    for k in (dict(tokens=0), dict(heads=0), dict(stride=255), dict(out_stride=255), dict(freqs=irx.rope_freqs(128)), dict(amplitude=NAN),
              dict(heads=1 << 15)):
        refused(irx, 42, irx.rope_append, **{**dict(cache=cache(irx), tokens=2, heads=4, freqs=f), **k})
    refused(irx, 42, irx.rope_append, cache(irx), 2, 1, f, stride=100)       # narrower than the keys
    refused(irx, 41, irx.rope_append, cache(irx, strides=(2048, 1024, 63)), 2, 4, f)
    refused(irx, 24, irx.rope_append, cache(irx, dtype="f16"), 2, 4, f)
    for k in (dict(tokens=0), dict(batch=0), dict(heads=0), dict(kv_heads=0), dict(heads=5), dict(head_dim=0), dict(head_dim=257),
              dict(window=-1), dict(sinks=-1), dict(sinks=1), dict(scale=NAN), dict(scale=INF), dict(q_stride=255), dict(kv_stride=127),
              dict(tokens=(1 << 30) + 1), dict(batch=(1 << 16) + 1), dict(tokens=1 << 30, heads=256, kv_heads=2), dict(q_stride=1 << 41)):
        refused(irx, 42, irx.prompt, **{**dict(tokens=9, batch=2, heads=4, kv_heads=2, head_dim=64), **k})
    refused(irx, 24, irx.prompt, 9, 2, 4, 2, 64, dtype="f64")
    for k in (dict(rows=0), dict(vocab=0), dict(vocab=(1 << 30) + 1), dict(rows=1 << 28), dict(stride=99), dict(stride=1 << 41)):
        refused(irx, 42, irx.sample, **{**dict(rows=2, vocab=100), **k})
    refused(irx, 24, irx.sample, 2, 100, dtype="i32")
    refused(irx, 93, irx.sample(2, 100).workspace)
    refused(irx, 93, irx.sample(2, 100).run_host, [np.zeros(1, np.float32)] * 7)
    refused(irx, 93, irx.prompt(9, 2, 4, 2, 64).host_chunks)
    refused(irx, 93, irx.rope(2, 4, 64, f).launch, [])


def test_frequencies(irx):
    assert np.allclose(irx.rope_freqs(8), [1.0, 0.1, 0.01, 0.001], rtol=1e-15)
    assert np.allclose(irx.rope_freqs(64, base=5e5), [5e5 ** (-2 * i / 64) for i in range(32)], rtol=1e-14)
    assert np.allclose(irx.rope_freqs(8, scaling="linear", factor=4), np.array([1.0, 0.1, 0.01, 0.001]) / 4, rtol=1e-15)
    plain, ntk = irx.rope_freqs(64), irx.rope_freqs(64, scaling="ntk", factor=8)
    assert ntk[0] == 1.0 and math.isclose(ntk[-1] * 8, plain[-1], rel_tol=1e-12)          # the slowest is divided by the factor
    assert irx.rope_freqs(2, scaling="ntk", factor=8) == [1.0]
    for kind in ("yarn", "bands"):
        f = irx.rope_freqs(128, scaling=kind, factor=16, original=4096)
        turns = [4096 * x / (2 * math.pi) for x in irx.rope_freqs(128)]
        share = [a / b for a, b in zip(f, irx.rope_freqs(128))]
        assert all(s == 1.0 for s, t in zip(share, turns) if t > 40)
        assert all(math.isclose(s, 1 / 16) for s, t in zip(share, turns) if t < 0.8)
        assert all(x >= y - 1e-15 for x, y in zip(share, share[1:])) and any(0.1 < s < 0.9 for s in share)
        assert irx.rope_freqs(128, scaling=kind, factor=1, original=4096) == pytest.approx(irx.rope_freqs(128), rel=1e-15)


def test_frequency_refusals(irx):
    for k in (dict(rot=0), dict(rot=7), dict(rot=258), dict(rot=-2), dict(base=1.0), dict(base=NAN), dict(base=INF), dict(scaling="other"),
              dict(scaling="linear", factor=0.5), dict(scaling="ntk", factor=NAN), dict(scaling="yarn", factor=2.0),
              dict(scaling="yarn", factor=2.0, original=-1.0), dict(scaling="bands", factor=2.0, original=4096, fast=1.0, slow=4.0),
              dict(scaling="yarn", factor=2.0, original=4096, slow=0.0)):
        refused(irx, 42, irx.rope_freqs, **{**dict(rot=64), **k})
