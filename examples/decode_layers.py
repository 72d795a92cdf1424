"""A small decoder that generates tokens with this package's plans: KIR graphs for the norms, the
activations and the prompt's attention, and the serving operators for everything that a
token-by-token step needs, 4-bit projections, the paged cache and attention over it.

    python examples/decode_layers.py

It prefills one prompt, forks it into several answers that share the prompt's pages, decodes them
together as one replayed CUDA graph, ends one answer, compacts the pool and goes on. Every
answer's last logits are then held against the same model computed densely in 64 bits. The weights
are random.
"""
from __future__ import annotations

import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import irptx_b200 as irx  # noqa: E402
from irptx_b200 import kir_author as ka  # noqa: E402

BF = torch.bfloat16


class Linear4:
    """A projection with 4-bit weights, groups of 64 along k, with zero points."""

    def __init__(self, n, k, gen, group=64):
        self.n, self.k, self.group = n, k, group
        q = torch.randint(0, 16, (n, k), generator=gen, device="cuda")
        self.w = irx.pack4(q)
        self.scales = (torch.rand(n, k // group, generator=gen, device="cuda") * 0.4 + 0.8).div(4.6 * math.sqrt(k)).to(BF)
        self.zeros = torch.randint(6, 10, (n, k // group), generator=gen, device="cuda", dtype=torch.uint8)
        g = torch.arange(k, device="cuda") // group
        self.dense = (q - self.zeros.long()[:, g]).double() * self.scales.double()[:, g]     # for the check only
        self.plans = {}

    def __call__(self, x):
        m = x.shape[0]
        if m not in self.plans:
            self.plans[m] = irx.matvec4(m, self.n, self.k, group=self.group, zeros=True)
        y = torch.empty(m, self.n, dtype=BF, device="cuda")
        self.plans[m].launch([x, self.w, self.scales, self.zeros, y])
        return y


class Decoder:
    def __init__(self, layers=2, hidden=512, heads=8, kv_heads=2, dim=128, ffn=1024, vocab=640, page=16, pages=96, slots=4, cols=24, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.layers, self.hidden, self.heads, self.kv, self.dim, self.slots, self.page = layers, hidden, heads, kv_heads, dim, slots, page
        self.width = (heads + 2 * kv_heads) * dim
        self.embed = torch.empty(vocab, hidden, device="cuda").normal_(generator=g).to(BF)
        self.blocks = [dict(qkv=Linear4(self.width, hidden, g), o=Linear4(hidden, heads * dim, g), up=Linear4(ffn, hidden, g),
                            gate=Linear4(ffn, hidden, g), down=Linear4(hidden, ffn, g),
                            n1=(torch.rand(hidden, generator=g, device="cuda") + 0.5).to(BF),
                            n2=(torch.rand(hidden, generator=g, device="cuda") + 0.5).to(BF)) for _ in range(layers)]
        self.head = Linear4(vocab, hidden, g)
        self.norm_f = torch.ones(hidden, device="cuda", dtype=BF)
        # the cache: every layer's pools in one tensor, so that a page copy serves all layers
        self.cache = irx.KvCache("bf16", kv_heads, dim, page, pages, batch=slots, table_cols=cols)
        self.k = torch.zeros((layers,) + self.cache.shape, dtype=BF, device="cuda")
        self.v = torch.zeros_like(self.k)
        self.pages = irx.Pages(pages, page, slots, cols)
        self.table = torch.zeros(slots, cols, dtype=torch.int32, device="cuda")
        self.attend = irx.decode(self.cache, heads, q_stride=self.width)
        self.work = self.attend.workspace()
        self.kir = {}

    def graph(self, name, text):
        if name not in self.kir:
            self.kir[name] = irx.compile(text())
        return self.kir[name]

    def rmsnorm(self, x, w):
        y = torch.empty_like(x)
        self.graph(("norm", x.shape), lambda: ka.rmsnorm(x.shape[0], x.shape[1])).launch([x, w, y])
        return y

    def pointwise(self, name, ops, *xs):
        y = torch.empty_like(xs[0])
        self.graph((name, y.numel()), lambda: ka.pointwise_chain(y.numel(), ops, d="bf16")).launch(list(xs) + [y])
        return y

    def append(self, layer, qkv, seq, pos):
        n = qkv.shape[0]
        if ("append", n) not in self.kir:
            self.kir["append", n] = irx.kv_append(self.cache, n, stride=self.width)
        rows = qkv.unflatten(1, (-1, self.dim))
        self.kir["append", n].launch([rows[:, self.heads:self.heads + self.kv], rows[:, self.heads + self.kv:], seq, pos,
                                      self.table, self.k[layer], self.v[layer]])

    def forward(self, x, seq, pos, attention):
        """The layers over x [tokens, hidden]; attention(layer, qkv) is the prompt's or a step's."""
        for i, b in enumerate(self.blocks):
            qkv = b["qkv"](self.rmsnorm(x, b["n1"]))
            self.append(i, qkv, seq, pos)
            x = self.pointwise("add", [("y", "add", ["x0", "x1"])], x, b["o"](attention(i, qkv)))
            h = self.rmsnorm(x, b["n2"])
            h = self.pointwise("swiglu", [("a", "silu", ["x0"]), ("y", "multiply", ["a", "x1"])], b["gate"](h), b["up"](h))
            x = self.pointwise("add", [("y", "add", ["x0", "x1"])], x, b["down"](h))
        return self.head(self.rmsnorm(x, self.norm_f))

    # ---- the host's part of a step ----

    def copy_pages(self, pairs):
        """Run the page copies that the manager asked for, and upload its table."""
        if pairs:
            n = -(-len(pairs) // 8) * 8                  # padded, so that a few plans serve every list
            if ("copy", n) not in self.kir:
                self.kir["copy", n] = irx.kv_copy(self.cache, n, layers=self.layers)
            pairs = pairs + [(-1, -1)] * (n - len(pairs))
            self.kir["copy", n].launch([torch.tensor(pairs, dtype=torch.int32, device="cuda"), self.k, self.v])
        self.table.copy_(torch.from_numpy(self.pages.table))

    def prompt(self, tokens):
        """Prefill: the prompt's keys and values go into pages, its attention is a KIR graph."""
        s, n = self.pages.open(), len(tokens)
        self.copy_pages([p for p in [self.pages.extend(s, n)] if p])
        seq = torch.full((n,), s, dtype=torch.int32, device="cuda")
        pos = torch.arange(n, dtype=torch.int32, device="cuda")
        plan = self.graph(("prompt", n), lambda: ka.attention(1, self.heads, n, self.dim, causal=True))

        def attention(_, qkv):
            q, k, v = qkv.unflatten(1, (-1, self.dim)).transpose(0, 1).split([self.heads, self.kv, self.kv])
            g = self.heads // self.kv
            o = torch.empty(self.heads, n, self.dim, dtype=BF, device="cuda")
            plan.launch([t.contiguous().reshape(-1) for t in (q, k.repeat_interleave(g, 0), v.repeat_interleave(g, 0))] + [o.reshape(-1)])
            return o.transpose(0, 1).reshape(n, -1).contiguous()

        return s, self.forward(self.embed[torch.tensor(tokens, device="cuda")], seq, pos, attention)[-1]

    def start(self, state):
        """Record a decoding step over all slots; `state` holds each slot's token and position (-1: none)."""
        self.token, self.pos = state
        self.lens = torch.zeros_like(self.pos)
        self.seq = torch.arange(self.slots, dtype=torch.int32, device="cuda")

        def attention(layer, qkv):
            o = torch.empty(self.slots, self.heads, self.dim, dtype=BF, device="cuda")
            q = qkv.unflatten(1, (-1, self.dim))[:, :self.heads]
            self.attend.launch([q, self.k[layer], self.v[layer], self.table, self.lens, o, self.work])
            return o.reshape(self.slots, -1)

        def step():
            self.lens.copy_(self.pos + 1)
            logits = self.forward(self.embed[self.token.clamp_min(0)], self.seq, self.pos, attention)
            self.token.copy_(logits.float().argmax(-1))
            self.pos.add_((self.pos >= 0).to(torch.int32))
            return logits

        keep = self.token.clone(), self.pos.clone()
        self.pos.fill_(-1)                               # the rehearsal that compiles the plans writes nothing
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        self.step_graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.step_graph):
            self.logits = step()
        self.token.copy_(keep[0])
        self.pos.copy_(keep[1])

    def step(self):
        """Room for every open slot's next token, then one replayed step. Returns the logits."""
        pairs = [p for s in range(self.slots) if self.pages.length(s) >= 0 for p in [self.pages.extend(s)] if p]
        self.copy_pages(pairs)
        self.step_graph.replay()
        return self.logits

    # ---- the check ----

    def dense(self, tokens):
        """The last token's logits of the same model, computed over the whole sequence in 64 bits."""
        def norm(x, w):
            return x / (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
        x, n = self.embed[torch.tensor(tokens, device="cuda")].double(), len(tokens)
        mask = torch.ones(n, n, device="cuda", dtype=torch.bool).tril()
        for b in self.blocks:
            q, k, v = (norm(x, b["n1"]) @ b["qkv"].dense.T).unflatten(1, (-1, self.dim)).transpose(0, 1).split([self.heads, self.kv, self.kv])
            k, v = k.repeat_interleave(self.heads // self.kv, 0), v.repeat_interleave(self.heads // self.kv, 0)
            p = (q @ k.transpose(1, 2) / math.sqrt(self.dim)).masked_fill(~mask, -math.inf).softmax(-1)
            x = x + (p @ v).transpose(0, 1).reshape(n, -1) @ b["o"].dense.T
            h = norm(x, b["n2"])
            x = x + (torch.nn.functional.silu(h @ b["gate"].dense.T) * (h @ b["up"].dense.T)) @ b["down"].dense.T
        return norm(x[-1:], self.norm_f)[0] @ self.head.dense.T


def main(prompt_len=37, steps=21, out=print):
    """Returns the largest relative error of the answers' last logits against the dense model, infinity when
    one of them is not a number."""
    m = Decoder()
    prompt = [(17 * i * i + 5 * i + 3) % m.embed.shape[0] for i in range(prompt_len)]
    first, logits = m.prompt(prompt)
    answers = {first: prompt + [int(logits.argmax())]}
    for t in (7, 211):                                   # two more answers that begin with other tokens
        answers[m.pages.fork(first)] = prompt + [t]
    out(f"{len(answers)} answers share the prompt: {m.pages.pages - m.pages.free} pages held")
    token = torch.zeros(m.slots, dtype=torch.long, device="cuda")
    pos = torch.full((m.slots,), -1, dtype=torch.int32, device="cuda")
    for s, a in answers.items():
        token[s], pos[s] = a[-1], prompt_len
    m.start((token, pos))
    worst, ended = 0.0, None
    for i in range(steps):
        if i == steps // 2:                              # the first answer ends; its pages go back and the rest move together
            ended = first
            m.pages.close(ended)
            m.pos[ended] = -1
            moves = m.pages.compact()
            m.copy_pages(moves)
            out(f"step {i}: answer {ended} ends, {len(moves)} pages move, {m.pages.pages - m.pages.free} held")
        logits = m.step()
        if i in (0, steps - 1):
            irx.check()
            for s, a in answers.items():
                if s != ended:
                    want = m.dense(a)
                    off = float((logits[s].double() - want).abs().max() / want.abs().max())
                    worst = max(worst, off if math.isfinite(off) else math.inf)      # (max would drop a NaN)
        for s in answers:
            if s != ended:
                answers[s].append(int(m.token[s]))
    out(f"{steps} steps; the last logits differ from the dense model's by {worst:.4f} of the largest")
    del m.step_graph
    return worst


if __name__ == "__main__":
    sys.exit(0 if main() < 0.05 else 1)
