"""Paged caches and 64-bit definitions on the GPU for the serving operators' tests, with bounds on what
the kernels' roundings can add up to."""
import math

DT = {"bf16": "bfloat16", "f32": "float32"}


def tdt(torch, dtype):
    return getattr(torch, DT[dtype])


class Paged:
    """A filled cache: pools whose pages no token reaches hold NaN, a table in random order whose entries
    that no token reaches name no page, queries, a plan and its buffers. shift: elements that the
    pools' first row lies past a 16-byte boundary."""

    def __init__(self, torch, irx, dtype, heads, kv, d, page, lens, order="head", window=0, sinks=0, scale=None, qmul=1.0, shift=0,
                 seed=0):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        need = [-(-n // page) for n in lens]
        pages, cols = sum(need) + 2, max(1, max(need))
        self.cache = irx.KvCache(dtype, kv, d, page, pages, batch=len(lens), table_cols=cols, order=order)
        dt = tdt(torch, dtype)

        def pool():
            flat = torch.full((pages * kv * page * d + shift,), math.nan, dtype=dt, device="cuda")
            return flat[shift:].view(self.cache.shape)

        self.k, self.v = pool(), pool()
        ids = torch.randperm(pages, generator=gen, device="cuda")
        self.table = torch.full((len(lens), cols), 10 ** 9, dtype=torch.int32, device="cuda")
        self.keys, self.values, at = [], [], 0
        for b, n in enumerate(lens):
            mine = ids[at:at + need[b]]
            at += need[b]
            self.table[b, :need[b]] = mine.to(torch.int32)
            pos = torch.arange(n, device="cuda")
            pg, sl = mine[pos // page], pos % page
            for into, keep in ((self.k, self.keys), (self.v, self.values)):
                x = torch.empty(n, kv, d, device="cuda").normal_(generator=gen).to(dt)
                if order == "head":
                    into[pg, :, sl] = x
                else:
                    into[pg, sl] = x
                keep.append(x)
        self.q = (torch.empty(len(lens), heads, d, device="cuda").normal_(generator=gen) * qmul).to(dt)
        self.torch, self.irx, self.dtype, self.heads, self.kv, self.d, self.page = torch, irx, dtype, heads, kv, d, page
        self.lens, self.window, self.sinks, self.order = tuple(lens), window, sinks, order
        self.scale = 1.0 / math.sqrt(d) if scale is None else scale
        self.plan = irx.decode(self.cache, heads, scale=scale, window=window, sinks=sinks, lse=True)
        self.out = torch.full_like(self.q, math.nan)
        self.lse = torch.full((len(lens), heads), math.nan, device="cuda")
        self.args = [self.q, self.k, self.v, self.table, torch.tensor(lens, dtype=torch.int32, device="cuda"), self.out, self.lse,
                     self.plan.workspace()]

    def put_value(self, b, pos, h, x):
        """Values of one key, for a test's own numbers; x: [d]."""
        pg, sl = int(self.table[b, pos // self.page]), pos % self.page
        x = x.to(self.v.dtype)
        if self.order == "head":
            self.v[pg, h, sl] = x
        else:
            self.v[pg, sl, h] = x
        self.values[b][pos, h] = x

    def put_key(self, b, pos, h, x):
        pg, sl = int(self.table[b, pos // self.page]), pos % self.page
        x = x.to(self.k.dtype)
        if self.order == "head":
            self.k[pg, h, sl] = x
        else:
            self.k[pg, sl, h] = x
        self.keys[b][pos, h] = x

    def launch(self):
        self.out.fill_(math.nan)
        self.lse.fill_(math.nan)
        self.plan.launch(self.args)
        return self

    def visible(self, b):
        n = self.lens[b]
        return [j for j in range(n) if not self.window or j >= n - self.window or j < self.sinks]

    def exact(self, b, at=None):
        """Sequence b over the positions `at` (its visible ones): out, lse, sum p |v|, largest sum |q k| of each row."""
        torch = self.torch
        at = torch.tensor(self.visible(b) if at is None else at, device="cuda", dtype=torch.long)
        g = self.heads // self.kv
        k, v = self.keys[b][at].double(), self.values[b][at].double()
        q = self.q[b].double().view(self.kv, g, self.d)
        s = torch.einsum("hgd,nhd->hgn", q, k) * self.scale
        p = torch.softmax(s, -1)
        big = abs(self.scale) * torch.einsum("hgd,nhd->hgn", q.abs(), k.abs()).amax(-1)
        return (torch.einsum("hgn,nhd->hgd", p, v).reshape(self.heads, self.d), torch.logsumexp(s, -1).reshape(-1),
                torch.einsum("hgn,nhd->hgd", p, v.abs()).reshape(self.heads, self.d), big.reshape(-1))

    def weight_err(self, n, big):
        """Relative error of a softmax weight and of its sums: a score's d products and sums and its scale, in
        f32, twice (its maximum's too), the exp's 2^-22 and n sums of f32 numbers that may be truncated."""
        return 2 * (self.d + 4) * 2.0 ** -24 * big + 2.0 ** -21 + (n + 16) * 2.0 ** -23

    def hold(self, b, at=None):
        """bf16 adds the weights' two parts, the first truncated (a rest below 2^-7 of the weight) and the rest
        rounded to 8 significant bits (2^-8): 2^-15; and the output's rounding, 2^-8. The log-sum adds f32
        weights as they are in both types."""
        n = len(self.visible(b) if at is None else at)
        out, lse, spread, big = self.exact(b, at)
        w = self.weight_err(n, big)
        if self.dtype == "bf16":
            tol = (w[:, None] + 2.0 ** -15) * spread * (1 + 2.0 ** -8) + 2.0 ** -8 * out.abs()
        else:
            tol = w[:, None] * spread + 2.0 ** -24 * out.abs()
        err = (self.out[b].double() - out).abs()
        assert bool((err <= tol).all()), f"sequence {b}: {float((err / tol).nan_to_num(9e9).max()):.3g} of the bound"
        assert bool(((self.lse[b].double() - lse).abs() <= w + 2.0 ** -22 * lse.abs()).all()), f"sequence {b}: lse"

    def hold_all(self):
        for b, n in enumerate(self.lens):
            if n:
                self.hold(b)
            else:
                assert bool((self.out[b] == 0).all()) and bool((self.lse[b] == -math.inf).all())


class Packed:
    """4-bit weights, tokens and a plan."""

    def __init__(self, torch, irx, dtype, m, n, k, group, zeros, scale_dtype=None, seed=0, x=None, q=None, s=None):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        groups = -(-k // group)
        self.q = torch.randint(0, 16, (n, k), generator=gen, device="cuda", dtype=torch.uint8) if q is None else q
        self.x = (torch.empty(m, k, device="cuda").normal_(generator=gen) if x is None else x).to(tdt(torch, dtype))
        self.s = ((torch.rand(n, groups, generator=gen, device="cuda") + 0.1) if s is None else s).to(tdt(torch, scale_dtype or dtype))
        self.z = torch.randint(0, 16, (n, groups), generator=gen, device="cuda", dtype=torch.uint8) if zeros else None
        self.y = torch.full((m, n), math.nan, dtype=self.x.dtype, device="cuda")
        self.plan = irx.matvec4(m, n, k, group=group, dtype=dtype, scale_dtype=scale_dtype, zeros=zeros)
        self.args = [self.x, irx.pack4(self.q), self.s] + ([self.z] if zeros else []) + [self.y]
        self.torch, self.dtype, self.m, self.n, self.k, self.group = torch, dtype, m, n, k, group

    def launch(self):
        self.y.fill_(math.nan)
        self.plan.launch(self.args)
        return self

    def exact(self):
        """(y, sum |x w|) in 64 bits, some rows of w at a time."""
        torch, col = self.torch, self.torch.arange(self.k, device="cuda") // self.group
        xd, parts = self.x.double(), []
        for a in range(0, self.n, 2048):
            z = self.z[a:a + 2048].double()[:, col] if self.z is not None else 8.0
            w = (self.q[a:a + 2048].double() - z) * self.s[a:a + 2048].double()[:, col]
            parts.append((xd @ w.T, xd.abs() @ w.abs().T))
        return torch.cat([p[0] for p in parts], 1), torch.cat([p[1] for p in parts], 1)

    def tol(self, y, mag):
        """Products are exact. A group, or a 128-wide piece of it, is summed by eight instructions that add 17
        numbers each, cut to 24 bits at the largest one's place; a piece's sum, times its scale, is one
        rounding more, and joining halves, slices and an f32 token's three parts a dozen. The output rounds
        once: 2^-8 for bf16's 8 significant bits, 2^-24."""
        return (8 * 17 + self.k / 32 + 16) * 2.0 ** -24 * mag + (2.0 ** -8 if self.dtype == "bf16" else 2.0 ** -24) * y.abs() + 1e-30

    def hold(self):
        y, mag = self.exact()
        err, tol = (self.y.double() - y).abs(), self.tol(y, mag)
        assert bool((err <= tol).all()), f"{float((err / tol).nan_to_num(9e9).max()):.3g} of the bound"
