"""The operators around the cache in a model's step as Python plans: rotary positions, attention over packed
prompts, and the draw of the next token.

    freqs  = irx.rope_freqs(128, base=500000.0)             # radians a position, one a pair
    turn   = irx.rope(4096, 40, 128, freqs)                 # [x, pos, y]
    append = irx.rope_append(cache, 32, 32, freqs)          # [q, k, v, seq, pos, table, q_out, k_pool, v_pool]
    prompt = irx.prompt(4096, 16, 32, 8, 128)               # [q, k, v, starts, out]
    draw   = irx.sample(32, 128000)                         # [logits, temperature, top_k, top_p, min_p, u, token]

Each is an ordinary plan, like the cache's own operators (``serve.py``), with their checks of tensors;
``include/irx.h`` states the formulas. Positions, starts and the draw's settings are read on the
device, so launches can be captured in a CUDA graph and replayed after they change. No counterpart
in the reference.
"""
from __future__ import annotations

import ctypes
import math

import irptx_b200 as _irx

from .serve import KvCache, OpPlan, _dtype, _int, _refuse

_SCALING = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3, "bands": 4}


class _RopeDesc(ctypes.Structure):
    _fields_ = [("freqs", ctypes.POINTER(ctypes.c_double)), ("pairs", ctypes.c_int), ("interleaved", ctypes.c_int),
                ("backward", ctypes.c_int), ("amplitude", ctypes.c_float)]


class _PromptDesc(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_int), ("tokens", ctypes.c_longlong), ("batch", ctypes.c_int), ("heads", ctypes.c_int),
                ("kv_heads", ctypes.c_int), ("head_dim", ctypes.c_int), ("q_stride", ctypes.c_longlong),
                ("kv_stride", ctypes.c_longlong), ("scale", ctypes.c_float), ("window", ctypes.c_int), ("sinks", ctypes.c_int),
                ("lse", ctypes.c_int)]


class _SampleDesc(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_int), ("rows", ctypes.c_longlong), ("vocab", ctypes.c_longlong), ("stride", ctypes.c_longlong),
                ("logprob", ctypes.c_int)]


def _number(name: str, v) -> float:
    v = float(v)
    if not math.isfinite(v) or abs(v) > 3.4028234663852886e38:
        _refuse(42, f"{name} that is not finite")
    return v


def rope_freqs(rot: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0, original: float = 0,
               fast: float | None = None, slow: float = 1.0) -> list[float]:
    """The rot / 2 rotation frequencies base ** (-2 i / rot), in radians a position, scaled for a context ``factor``
    times the ``original`` one: "linear", "ntk", "yarn" or "bands" (``irx_rope_freqs``). Pairs that turn more than
    ``fast`` times within the original context are kept: 32 unless given, with "bands" 4. YaRN's
    amplitude, 0.1 ln(factor) + 1, is the caller's to give to :func:`rope`."""
    if scaling not in _SCALING:
        _refuse(42, f"a scaling {scaling!r} ({', '.join(_SCALING)})")
    if fast is None:
        fast = 4.0 if scaling == "bands" else 32.0
    out = (ctypes.c_double * max(1, min(_int("rot", rot), 256)))()
    if _irx._lib().irx_rope_freqs(_int("rot", rot), float(base), _SCALING[scaling], float(factor), float(original), float(fast),
                                  float(slow), out):
        _irx._raise()
    return list(out[:rot // 2])


def _rope_desc(freqs, interleaved, amplitude, backward):
    freqs = [float(f) for f in freqs]
    arr = (ctypes.c_double * max(1, len(freqs)))(*freqs)
    return _RopeDesc(ctypes.cast(arr, ctypes.POINTER(ctypes.c_double)), len(freqs), int(bool(interleaved)), int(bool(backward)),
                     _number("an amplitude", amplitude)), arr


def rope(tokens: int, heads: int, head_dim: int, freqs, dtype: str = "bf16", interleaved: bool = False, amplitude: float = 1.0,
         backward: bool = False, x_stride: int = 0, y_stride: int = 0) -> OpPlan:
    """Rotary positions: [x, pos, y]. The first 2 * len(freqs) numbers of each head are turned by pos * freqs, pairs being
    (i, i + len(freqs)) or, ``interleaved``, (2 i, 2 i + 1); the rest is copied. ``backward`` turns y's gradient
    into x's. pos < 0 is padding. y may be x itself. The strides (elements from one token's rows to the
    next's, 0: packed) describe slices of wider rows."""
    d, keep = _rope_desc(freqs, interleaved, amplitude, backward)
    tokens, heads, head_dim = _int("tokens", tokens, 62), _int("heads", heads), _int("head_dim", head_dim)
    x_stride, y_stride = _int("x_stride", x_stride, 62), _int("y_stride", y_stride, 62)
    row = (tokens, heads, head_dim)
    args = [("x", row, (x_stride or heads * head_dim, head_dim, 1)), ("pos", (tokens,), None),
            ("y", row, (y_stride or heads * head_dim, head_dim, 1))]
    code = _dtype(dtype)
    return OpPlan(lambda lib, p: lib.irx_compile_rope(ctypes.byref(d), code, tokens, heads, head_dim, x_stride, y_stride, p), args)


def rope_append(cache: KvCache, tokens: int, heads: int, freqs, interleaved: bool = False, amplitude: float = 1.0, stride: int = 0,
                out_stride: int = 0) -> OpPlan:
    """:func:`rope` and ``kv_append`` in one launch: [q, k, v, seq, pos, table, q_out, k_pool, v_pool]. The queries are
    turned into q_out, the keys on their way into their page, the values go as they are. ``stride``: elements
    from one token's rows to the next's in q, k and v (0: each packed), as in slices of a fused projection.
    pos < 0 is padding. q_out may be q itself, with the same stride."""
    c = cache._desc()
    d, keep = _rope_desc(freqs, interleaved, amplitude, False)
    tokens, heads = _int("tokens", tokens, 62), _int("heads", heads)
    stride, out_stride = _int("stride", stride, 62), _int("out_stride", out_stride, 62)
    dim = cache.head_dim
    q, kv = (tokens, heads, dim), (tokens, cache.heads, dim)
    args = [("q", q, (stride or heads * dim, dim, 1)), ("k", kv, (stride or cache.heads * dim, dim, 1)),
            ("v", kv, (stride or cache.heads * dim, dim, 1)), ("seq", (tokens,), None), ("pos", (tokens,), None),
            ("table", (cache.batch, cache.table_cols), None), ("q_out", q, (out_stride or heads * dim, dim, 1)),
            ("k_pool", cache.shape, cache.strides + (1,)), ("v_pool", cache.shape, cache.strides + (1,))]
    return OpPlan(lambda lib, p: lib.irx_compile_rope_append(ctypes.byref(c), ctypes.byref(d), tokens, heads, stride, out_stride, p),
                  args)


def prompt(tokens: int, batch: int, heads: int, kv_heads: int, head_dim: int, dtype: str = "bf16", scale: float | None = None,
           window: int = 0, sinks: int = 0, lse: bool = False, q_stride: int = 0, kv_stride: int = 0) -> OpPlan:
    """Causal attention over packed prompts: [q, k, v, starts, out, (lse)]. Sequence s is the rows starts[s] to
    starts[s + 1]; rows outside all of them are left as they were. ``scale`` defaults to head_dim ** -0.5; ``window``
    tokens are visible (0: all) and, before them, the sequence's first ``sinks``."""
    tokens, batch = _int("tokens", tokens, 62), _int("batch", batch)
    heads, kv_heads, head_dim = _int("heads", heads), _int("kv_heads", kv_heads), _int("head_dim", head_dim)
    scale = 1.0 / math.sqrt(max(1, head_dim)) if scale is None else _number("a scale", scale)
    q_stride, kv_stride = _int("q_stride", q_stride, 62), _int("kv_stride", kv_stride, 62)
    d = _PromptDesc(_dtype(dtype), tokens, batch, heads, kv_heads, head_dim, q_stride, kv_stride, scale, _int("window", window),
                    _int("sinks", sinks), int(bool(lse)))
    row = (tokens, heads, head_dim)
    kv = ((tokens, kv_heads, head_dim), (kv_stride or kv_heads * head_dim, head_dim, 1))
    args = [("q", row, (q_stride or heads * head_dim, head_dim, 1)), ("k",) + kv, ("v",) + kv, ("starts", (batch + 1,), None),
            ("out", row, None)]
    if lse:
        args.append(("lse", (tokens, heads), None))
    return OpPlan(lambda lib, p: lib.irx_compile_prompt(ctypes.byref(d), p), args)


def sample(rows: int, vocab: int, dtype: str = "f32", stride: int = 0, logprob: bool = False) -> OpPlan:
    """The draw of the next token: [logits, temperature, top_k, top_p, min_p, u, token, (logprob)], one setting and one
    uniform random number a row. Filters apply in the order of their names: top-k of the logits (equal ones
    by index), top-p of what is left, min-p relative to the largest; the draw runs through the kept tokens by
    index. temperature 0 takes the largest logit. top_k 0, top_p 1 and min_p 0 are off."""
    rows, vocab, stride = _int("rows", rows, 62), _int("vocab", vocab, 62), _int("stride", stride, 62)
    d = _SampleDesc(_dtype(dtype), rows, vocab, stride, int(bool(logprob)))
    args = [("logits", (rows, vocab), (stride or vocab, 1))]
    args += [(n, (rows,), None) for n in ("temperature", "top_k", "top_p", "min_p", "u", "token")]
    if logprob:
        args.append(("logprob", (rows,), None))
    return OpPlan(lambda lib, p: lib.irx_compile_sample(ctypes.byref(d), p), args)
