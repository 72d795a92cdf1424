"""Several prompts at once through a small decoder with rotary positions: packed attention over all of them, then a
replayed step that appends, attends and draws each answer's next token by its own settings.

    python examples/serve_prompts.py

The decoder is decode_layers.py's. Prompts of different lengths go through the layers as one packed batch: their
queries and keys are turned in place, their keys and values appended to pages, and irx.prompt attends
sequence by sequence. A step turns and appends in one launch, and irx.sample draws from its logits. The
last logits are held against the same model computed densely in 64 bits, and every drawn token against its definition.
"""
from __future__ import annotations

import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))

import irptx_b200 as irx  # noqa: E402
from decode_layers import BF, Decoder  # noqa: E402


class Server(Decoder):
    def __init__(self, settings, **kw):
        """settings: (temperature, top_k, top_p, min_p) of every slot."""
        super().__init__(**kw)
        self.freqs = irx.rope_freqs(self.dim, base=10000.0, scaling="yarn", factor=4.0, original=4096)
        self.packed = False
        t, k, p, m = zip(*settings)
        self.temperature, self.top_p, self.min_p = (torch.tensor(x, dtype=torch.float32, device="cuda") for x in (t, p, m))
        self.top_k = torch.tensor(k, dtype=torch.int32, device="cuda")
        self.u = torch.zeros(self.slots, device="cuda")
        self.drawn = torch.zeros(self.slots, dtype=torch.int32, device="cuda")
        self.draw = irx.sample(self.slots, self.embed.shape[0], dtype="bf16")

    def plan(self, key, make):
        if key not in self.kir:
            self.kir[key] = make()
        return self.kir[key]

    def append(self, layer, qkv, seq, pos):
        n, h, kv = qkv.shape[0], self.heads, self.kv
        rows = qkv.unflatten(1, (-1, self.dim))
        if self.packed:                                  # the prompt's attention reads the turned keys from the rows themselves
            turn = self.plan(("rope", n), lambda: irx.rope(n, h + kv, self.dim, self.freqs, x_stride=self.width, y_stride=self.width))
            turn.launch([rows[:, :h + kv], pos, rows[:, :h + kv]])
            super().append(layer, qkv, seq, pos)
        else:                                            # a step's only from the pages
            both = self.plan(("rope_append", n), lambda: irx.rope_append(self.cache, n, h, self.freqs, stride=self.width, out_stride=self.width))
            both.launch([rows[:, :h], rows[:, h:h + kv], rows[:, h + kv:], seq, pos, self.table, rows[:, :h], self.k[layer], self.v[layer]])

    def prompts(self, lists):
        """All prompts in one packed batch: their slots and their last tokens' logits."""
        slots, pairs = [], []
        for tokens in lists:
            slots.append(self.pages.open())
            pairs += [p for p in [self.pages.extend(slots[-1], len(tokens))] if p]
        self.copy_pages(pairs)
        lens = [len(t) for t in lists]
        starts = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device="cuda")
        seq = torch.tensor([s for s, t in zip(slots, lists) for _ in t], dtype=torch.int32, device="cuda")
        pos = torch.tensor([i for t in lists for i in range(len(t))], dtype=torch.int32, device="cuda")
        n, h, kv = sum(lens), self.heads, self.kv
        attend = irx.prompt(n, len(lens), h, kv, self.dim, q_stride=self.width, kv_stride=self.width)

        def attention(_, qkv):
            rows = qkv.unflatten(1, (-1, self.dim))
            o = torch.empty(n, h, self.dim, dtype=BF, device="cuda")
            attend.launch([rows[:, :h], rows[:, h:h + kv], rows[:, h + kv:], starts, o])
            return o.reshape(n, -1)

        self.packed = True
        logits = self.forward(self.embed[torch.tensor([x for t in lists for x in t], device="cuda")], seq, pos, attention)
        self.packed = False
        return slots, logits[starts[1:].long() - 1]

    def choose(self, logits):
        self.draw.launch([logits, self.temperature, self.top_k, self.top_p, self.min_p, self.u, self.drawn])
        return self.drawn

    def turned(self, x):
        half = self.dim // 2
        angle = torch.outer(torch.arange(x.shape[1], device="cuda", dtype=torch.float64), torch.tensor(self.freqs, device="cuda", dtype=torch.float64))
        c, s, a, b = angle.cos(), angle.sin(), x[..., :half], x[..., half:]
        return torch.cat([a * c - b * s, a * s + b * c], -1)


def by_definition(logits, temperature, top_k, top_p, min_p, u):
    """The token that irx.sample draws from one row, by lists of indexes in 64 bits."""
    x = logits.double()
    if not temperature > 0:
        return int((x == x.max()).nonzero()[0])
    w = torch.exp((x - x.max()) / temperature)
    kept = torch.argsort(x, descending=True, stable=True)[:top_k or None]
    sums = torch.cumsum(w[kept], 0)
    if top_p < 1:
        kept = kept[:int((sums < top_p * sums[-1]).sum()) + 1]
    kept = torch.sort(kept[w[kept] >= min_p]).values
    sums = torch.cumsum(w[kept], 0)
    return int(kept[int((sums <= u * sums[-1]).sum())])


def main(steps=12, out=print):
    """(the largest relative error of the last logits against the dense model's, infinity when one is not a number; how many
    drawn tokens are not their definition's)"""
    settings = [(0.0, 0, 1.0, 0.0), (0.75, 40, 1.0, 0.0), (1.0, 0, 0.875, 0.0), (0.5, 100, 0.9375, 0.03125)]
    m = Server(settings)
    gen = torch.Generator(device="cuda").manual_seed(7)
    lists = [[(17 * i * i + 5 * i + 3 + s) % m.embed.shape[0] for i in range(n)] for s, n in enumerate((37, 5, 91, 64))]
    slots, logits = m.prompts(lists)
    answers = {s: list(t) for s, t in zip(slots, lists)}
    out(f"{len(lists)} prompts of {', '.join(str(len(t)) for t in lists)} tokens in one batch")
    worst = 0.0

    def compare(rows):
        nonlocal worst
        for s, row in rows:
            want = m.dense(answers[s])
            off = float((row.double() - want).abs().max() / want.abs().max())
            worst = max(worst, off if math.isfinite(off) else math.inf)

    compare(zip(slots, logits))
    for s, l in zip(slots, logits):
        answers[s].append(int(l.float().argmax()))
    token = torch.zeros(m.slots, dtype=torch.long, device="cuda")
    pos = torch.full((m.slots,), -1, dtype=torch.int32, device="cuda")
    for s, t in zip(slots, lists):
        token[s], pos[s] = answers[s][-1], len(t)
    m.start((token, pos))
    wrong = 0
    for i in range(steps):
        m.u.copy_(torch.rand(m.slots, generator=gen, device="cuda"))
        logits = m.step()
        irx.check()
        if i in (0, steps - 1):
            compare((s, logits[s]) for s in slots)
        for s in slots:
            wrong += int(m.token[s]) != by_definition(logits[s], *settings[s], float(m.u[s]))
            answers[s].append(int(m.token[s]))
    out(f"{steps} steps; the last logits differ from the dense model's by {worst:.4f} of the largest; {wrong} draws are not their definition's")
    del m.step_graph
    return worst, wrong


if __name__ == "__main__":
    off, wrong = main()
    sys.exit(0 if off < 0.05 and not wrong else 1)
