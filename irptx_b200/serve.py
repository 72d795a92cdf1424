"""The serving operators as Python plans: what a decoding program runs between KIR graphs.

    cache  = irx.KvCache("bf16", heads=8, head_dim=128, page_size=16, pages=4096, batch=32, table_cols=256)
    append = irx.kv_append(cache, tokens=32)          # [k, v, seq, pos, table, k_pool, v_pool]
    step   = irx.decode(cache, heads=32)              # [q, k_pool, v_pool, table, lens, out, workspace]
    copy   = irx.kv_copy(cache, pairs=8)              # [pairs, k_pool, v_pool]
    proj   = irx.matvec4(32, 4096, 4096, group=128)   # [x, w, scales, y]
    pages  = irx.Pages(4096, 16, max_seqs=32, table_cols=256)

Each of the four is an ordinary :class:`Plan` (``launch``, ``launch_shard``, ``bind``, ``describe``,
``work``), compiled from a descriptor by the C ABI (``irx_compile_decode`` and so on in
``include/irx.h``, which states the operators' formulas, argument order and strides). Tensors are
checked against the plan: device, dtype, shape and strides. Launches only queue work on the
stream: lengths, tables and positions are read on the device, so a launch can be captured in a
CUDA graph and replayed after they change; an index outside the cache is skipped and reported by
``irx.check`` as E093. No counterpart in the reference, which has no cache and no packed weights.
"""
from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass

import irptx_b200 as _irx

_CODE = {"f32": 1, "bf16": 2}
_TORCH = {"f32": "torch.float32", "bf16": "torch.bfloat16", "i32": "torch.int32", "u8": "torch.uint8"}


def _refuse(code: int, what: str):
    raise _irx.IrxError(code, f"error[E{code:03d}]: irptx: cannot lower {what}")


def _dtype(dtype: str) -> int:
    if dtype not in _CODE:
        _refuse(24, f"a dtype {dtype!r} (f32 or bf16)")
    return _CODE[dtype]


def _int(name: str, v, bits: int = 31) -> int:
    v = int(v)
    if not -(1 << bits) <= v < 1 << bits:
        _refuse(42, f"{name}={v}: past {bits + 1} bits")
    return v


class _CacheDesc(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_int), ("heads", ctypes.c_int), ("head_dim", ctypes.c_int), ("page_size", ctypes.c_int),
                ("pages", ctypes.c_longlong), ("page_stride", ctypes.c_longlong), ("head_stride", ctypes.c_longlong),
                ("token_stride", ctypes.c_longlong), ("batch", ctypes.c_int), ("table_cols", ctypes.c_int)]


class _Matvec4Desc(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_int), ("scale_dtype", ctypes.c_int), ("m", ctypes.c_longlong), ("n", ctypes.c_longlong),
                ("k", ctypes.c_longlong), ("group", ctypes.c_int), ("zeros", ctypes.c_int), ("x_stride", ctypes.c_longlong),
                ("w_stride", ctypes.c_longlong)]


class KvCache:
    """A paged cache's geometry: two pools, keys and values, of the same shape and strides.

    ``order`` "head" is [pages, heads, page_size, head_dim], "token" [pages, page_size, heads,
    head_dim]; ``strides`` (elements, of the pool's first three axes in that order) describes a
    view, None a packed pool. ``batch`` and ``table_cols`` are the page table's shape."""

    def __init__(self, dtype: str, heads: int, head_dim: int, page_size: int, pages: int, batch: int = 1,
                 table_cols: int = 1, order: str = "head", strides=None):
        if order not in ("head", "token"):
            _refuse(42, f"a cache order {order!r} (head or token)")
        self.dtype, self.order = dtype, order
        self.heads, self.head_dim, self.page_size = _int("heads", heads), _int("head_dim", head_dim), _int("page_size", page_size)
        self.pages, self.batch, self.table_cols = _int("pages", pages), _int("batch", batch), _int("table_cols", table_cols)
        inner = (self.heads, self.page_size) if order == "head" else (self.page_size, self.heads)
        given = strides is not None
        if not given:
            strides = (inner[0] * inner[1] * self.head_dim, inner[1] * self.head_dim, self.head_dim)
        if len(strides) != 3:
            _refuse(42, "cache strides that are not three numbers")
        if given and not any(strides) and max(self.pages, self.heads, self.page_size) > 1:
            _refuse(41, "a cache whose strides make rows overlap")        # (to the C ABI three zeros mean packed)
        self.strides = tuple(_int("stride", s, 62) for s in strides)
        self.shape = (self.pages,) + inner + (self.head_dim,)

    def _desc(self) -> _CacheDesc:
        page, a, b = self.strides
        head, token = (a, b) if self.order == "head" else (b, a)
        return _CacheDesc(_dtype(self.dtype), self.heads, self.head_dim, self.page_size, self.pages, page, head, token,
                          self.batch, self.table_cols)


@dataclass
class OpArg:
    index: int
    name: str
    kind: str
    dtype: str
    elems: int
    shape: tuple
    stride: tuple


def _packed(shape):
    st, n = [], 1
    for s in reversed(shape):
        st.append(n)
        n *= s
    return tuple(reversed(st))


class OpPlan(_irx.Plan):
    """A plan compiled from an operator's descriptor. Its ``args`` carry shapes and strides, which
    every tensor given to a launch has to have."""

    def __init__(self, compile_into, args):
        self.kir = None
        self._buf = (ctypes.c_ulonglong * (_irx.PLAN_BYTES // 8))()
        lib = _irx._lib()
        if compile_into(lib, ctypes.byref(self._buf)):
            _irx._raise()
        self.family = _irx.FAMILIES[lib.irx_plan_family(self.handle)]
        self.args = []
        for a in range(lib.irx_plan_nargs(self.handle)):
            k, d, n = ctypes.c_int(), ctypes.c_int(), ctypes.c_longlong()
            if lib.irx_plan_arg(self.handle, a, ctypes.byref(k), ctypes.byref(d), ctypes.byref(n)):
                _irx._raise()
            name, shape, stride = args[a]
            shape = (n.value,) if shape is None else shape
            self.args.append(OpArg(a, name, _irx._KIND[k.value], _irx._DT[d.value], n.value, shape, stride or _packed(shape)))

    def workspace(self):
        """A zeroed workspace on the current CUDA device, for the plan's last argument. Launches that
        may run at the same time need one each."""
        import torch
        if self.args[-1].kind != "work":
            _refuse(93, f"a workspace of a {self.family} plan, which needs none")
        return torch.zeros(self.args[-1].elems, dtype=torch.uint8, device="cuda")

    def _ptrs(self, args):
        if isinstance(args, _irx.Bound):
            if args.plan is not self:
                _refuse(93, "arguments bound to another plan")
            return args.arr
        if len(args) != len(self.args):
            _refuse(93, f"a launch with {len(args)} args; the plan has {len(self.args)}")
        out, device = [], None
        for a, x in zip(self.args, args):
            if isinstance(x, int):
                out.append(x)
                continue
            if device is None and x.is_cuda:
                import torch
                device = torch.cuda.current_device()
            if not x.is_cuda or x.get_device() != device:
                _refuse(93, f"arg {a.name}: a tensor on {x.device}, not on the current GPU")
            if str(x.dtype) != _TORCH[a.dtype]:
                _refuse(93, f"arg {a.name}: dtype {x.dtype}, the plan says {a.dtype}")
            if tuple(x.shape) != a.shape:
                _refuse(93, f"arg {a.name}: shape {tuple(x.shape)}, the plan says {a.shape}")
            if any(n > 1 and s != w for n, s, w in zip(x.shape, x.stride(), a.stride)):
                _refuse(93, f"arg {a.name}: strides {tuple(x.stride())}, the plan says {a.stride}")
            out.append(x.data_ptr())
        return (ctypes.c_void_p * len(out))(*out)


def decode(cache: KvCache, heads: int, scale: float | None = None, window: int = 0, sinks: int = 0, lse: bool = False,
           q_stride: int = 0) -> OpPlan:
    """Attention of each sequence's newest token over its cache: [q, k_pool, v_pool, table, lens, out,
    (lse,) workspace]. ``scale`` defaults to head_dim ** -0.5; ``window`` keys are visible (0: all)
    and, before them, the first ``sinks``. A sequence of length 0 gives zeros and an lse of -inf."""
    d = cache._desc()
    heads, b = _int("heads", heads), cache.batch
    scale = 1.0 / math.sqrt(max(1, cache.head_dim)) if scale is None else float(scale)
    if not math.isfinite(scale) or abs(scale) > 3.4028234663852886e38:
        _refuse(42, "a scale that is not finite")
    window, sinks, q_stride = _int("window", window), _int("sinks", sinks), _int("q_stride", q_stride, 62)
    row = (b, heads, cache.head_dim)
    args = [("q", row, (q_stride or heads * cache.head_dim, cache.head_dim, 1)),
            ("k", cache.shape, cache.strides + (1,)), ("v", cache.shape, cache.strides + (1,)),
            ("table", (b, cache.table_cols), None), ("lens", (b,), None), ("out", row, None)]
    if lse:
        args.append(("lse", (b, heads), None))
    args.append(("workspace", None, None))
    return OpPlan(lambda lib, p: lib.irx_compile_decode(ctypes.byref(d), heads, q_stride, scale, window, sinks, int(bool(lse)), p),
                  args)


def kv_append(cache: KvCache, tokens: int, stride: int = 0) -> OpPlan:
    """New tokens into their pages: [k, v, seq, pos, table, k_pool, v_pool]. Token i goes to position
    pos[i] of sequence seq[i]; a negative position is padding. ``stride``: elements from one
    token's rows to the next (0: packed), as in a slice of a fused projection."""
    d = cache._desc()
    tokens, stride = _int("tokens", tokens, 62), _int("stride", stride, 62)
    row = (tokens, cache.heads, cache.head_dim)
    new = (stride or cache.heads * cache.head_dim, cache.head_dim, 1)
    args = [("k", row, new), ("v", row, new), ("seq", (tokens,), None), ("pos", (tokens,), None),
            ("table", (cache.batch, cache.table_cols), None),
            ("k_pool", cache.shape, cache.strides + (1,)), ("v_pool", cache.shape, cache.strides + (1,))]
    return OpPlan(lambda lib, p: lib.irx_compile_kv_append(ctypes.byref(d), tokens, stride, p), args)


def kv_copy(cache: KvCache, pairs: int, layers: int = 1, layer_stride: int = 0) -> OpPlan:
    """Page copies (src, dst) in both pools and every layer: [pairs, k_pools, v_pools], the pools with a
    leading layers axis ``layer_stride`` elements apart (0: packed). (-1, -1) is padding; no page
    may be one pair's destination and in another pair."""
    d = cache._desc()
    pairs, layers, layer_stride = _int("pairs", pairs, 62), _int("layers", layers), _int("layer_stride", layer_stride, 62)
    shape, stride = (layers,) + cache.shape, (layer_stride or cache.pages * cache.strides[0],) + cache.strides + (1,)
    args = [("pairs", (pairs, 2), None), ("k_pools", shape, stride), ("v_pools", shape, stride)]
    return OpPlan(lambda lib, p: lib.irx_compile_kv_copy(ctypes.byref(d), pairs, layers, layer_stride, p), args)


def matvec4(m: int, n: int, k: int, group: int = 128, dtype: str = "bf16", scale_dtype: str | None = None,
            zeros: bool = False, x_stride: int = 0, w_stride: int = 0) -> OpPlan:
    """y[m, n] = sum_k x[m, k] s[n, k // group] (q[n, k] - z[n, k // group]): [x, w, scales, (zeros,) y].
    w is uint8 [n, ceil(k / 2)], the even k in the low four bits (:func:`pack4`); z is uint8, 0 to
    15, or 8 everywhere without ``zeros``. Meant for a few tokens: the weights are read again for every 16
    (every 5 with f32 tokens)."""
    m, n, k, group = _int("m", m, 62), _int("n", n, 62), _int("k", k, 62), _int("group", group)
    x_stride, w_stride = _int("x_stride", x_stride, 62), _int("w_stride", w_stride, 62)
    d = _Matvec4Desc(_dtype(dtype), _dtype(scale_dtype or dtype), m, n, k, group, int(bool(zeros)), x_stride, w_stride)
    groups = -(-k // group) if group > 0 else 0
    args = [("x", (m, k), (x_stride or k, 1)), ("w", (n, (k + 1) // 2), (w_stride or (k + 1) // 2, 1)),
            ("scales", (n, groups), None)]
    if zeros:
        args.append(("zeros", (n, groups), None))
    args.append(("y", (m, n), None))
    return OpPlan(lambda lib, p: lib.irx_compile_matvec4(ctypes.byref(d), p), args)


def pack4(q):
    """Weights 0 to 15, an integer torch tensor or numpy array [n, k], into matvec4's bytes [n, ceil(k / 2)]."""
    n, k = q.shape
    odd = k % 2
    if hasattr(q, "detach"):
        import torch
        if q.numel() and (int(q.min()) < 0 or int(q.max()) > 15):
            _refuse(42, "a weight outside 0 to 15")
        if odd:
            q = torch.cat([q, q.new_zeros(n, 1)], 1)
        q = q.to(torch.uint8).reshape(n, -1, 2)
        return (q[:, :, 0] | (q[:, :, 1] << 4)).contiguous()
    import numpy as np
    q = np.asarray(q)
    if q.size and (q.min() < 0 or q.max() > 15):
        _refuse(42, "a weight outside 0 to 15")
    if odd:
        q = np.concatenate([q, np.zeros((n, 1), q.dtype)], 1)
    q = q.astype(np.uint8).reshape(n, -1, 2)
    return np.ascontiguousarray(q[:, :, 0] | (q[:, :, 1] << 4))


class Pages:
    """The host side of a paged cache (``irx_pages_*``): which pages each sequence holds, shared by
    forks and copied when a shared page is written to. It keeps numbers only: a step gathers the (src,
    dst) pairs that its calls return, reads :attr:`table` to upload it, and runs the pairs through
    :func:`kv_copy` before its other launches. The pairs returned between two readings of the table
    may run in one launch or in any order; pages of theirs that nobody holds any more are free again
    once the table has been read. A copy carries what its source holds: queue a sequence's appends
    before its forks are extended."""

    def __init__(self, pages: int, page_size: int, max_seqs: int, table_cols: int):
        self._h = None
        self.pages, self.page_size = _int("pages", pages), _int("page_size", page_size)
        self.max_seqs, self.table_cols = _int("max_seqs", max_seqs), _int("table_cols", table_cols)
        self._h = _irx._lib().irx_pages_new(self.pages, self.page_size, self.max_seqs, self.table_cols)
        if not self._h:
            _irx._raise()

    def __del__(self):
        if getattr(self, "_h", None):
            _irx._lib().irx_pages_delete(self._h)
            self._h = None

    def open(self) -> int:
        """A new, empty sequence: its row of the table."""
        s = _irx._lib().irx_pages_open(self._h)
        if s < 0:
            _irx._raise()
        return s

    def extend(self, seq: int, tokens: int = 1):
        """Room for ``tokens`` more tokens. Returns the (src, dst) page copy that has to run before the
        first of them is written, or None."""
        pair = (ctypes.c_int * 2)()
        if _irx._lib().irx_pages_extend(self._h, _int("seq", seq), _int("tokens", tokens), pair):
            _irx._raise()
        return None if pair[0] < 0 else (pair[0], pair[1])

    def fork(self, seq: int) -> int:
        """A new sequence that shares all of ``seq``'s pages."""
        s = _irx._lib().irx_pages_fork(self._h, _int("seq", seq))
        if s < 0:
            _irx._raise()
        return s

    def close(self, seq: int):
        """End a sequence; the pages that no other holds are free again."""
        if _irx._lib().irx_pages_close(self._h, _int("seq", seq)):
            _irx._raise()

    def compact(self):
        """Move the live pages to the front of the pool: the (src, dst) copies that have to run before
        the table is used again (every destination was free). Pages of pairs returned since the table
        was last read stay where they are: read it first for a pool without holes."""
        buf = (ctypes.c_int * (2 * self.pages))()
        n = _irx._lib().irx_pages_compact(self._h, buf, self.pages)
        if n < 0:
            _irx._raise()
        return [(buf[2 * i], buf[2 * i + 1]) for i in range(n)]

    @property
    def free(self) -> int:
        """Pages that can be handed out now."""
        return int(_irx._lib().irx_pages_free(self._h))

    def length(self, seq: int) -> int:
        """Tokens of a sequence; -1 when it is not open."""
        return int(_irx._lib().irx_pages_len(self._h, _int("seq", seq)))

    @property
    def table(self):
        """A copy of the page table, int32 [max_seqs, table_cols], -1 where nothing is held. Reading it
        ends a step's gathering: the pairs returned before run before those returned after."""
        import numpy as np
        t = _irx._lib().irx_pages_table(self._h)
        return np.ctypeslib.as_array(t, (self.max_seqs, self.table_cols)).astype(np.int32)
