"""64-bit definitions of the operators around the cache, for their tests: rotary positions, attention over packed
prompts, the draw of a token; and bounds on what the kernels' roundings can add up to."""
import math

DT = {"bf16": "bfloat16", "f32": "float32"}
HALF = {"bf16": 2.0 ** -8, "f32": 2.0 ** -24}            # half a step of the type, relative


def tdt(torch, dtype):
    return getattr(torch, DT[dtype])


def rope_exact(torch, x, pos, freqs, interleaved=False, amplitude=1.0, backward=False):
    """(y, tol): x [tokens, heads, dim]. tol counts, in units of (|x1| + |x2|) amplitude: sincospi's 2^-23, the
    correction to first order, the amplitude's product and the pair's two products and sum, six roundings of
    2^-24: 2^-21 in all; the 64-bit angle's two roundings, 2 pi turns 2^-52; and the output's rounding."""
    r = 2 * len(freqs)
    f = torch.tensor(freqs, dtype=torch.float64, device=x.device)
    angle = pos.double()[:, None] * f[None, :] * (-1.0 if backward else 1.0)
    c, s = (t[:, None, :] * amplitude for t in (torch.cos(angle), torch.sin(angle)))
    one, two = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    y, tol = x.double().clone(), torch.zeros_like(x, dtype=torch.float64)
    a, b = x.double()[..., one], x.double()[..., two]
    y[..., one], y[..., two] = a * c - b * s, a * s + b * c
    t = (a.abs() + b.abs()) * abs(amplitude) * (2.0 ** -21 + 2.0 ** -52 * angle.abs()[:, None, :])
    half = HALF["bf16" if x.dtype == torch.bfloat16 else "f32"]
    tol[..., one], tol[..., two] = t + half * y[..., one].abs(), t + half * y[..., two].abs()
    return y, tol


def prompt_exact(torch, q, k, v, starts, scale, window=0, sinks=0, matrix=False):
    """(out, tol, lse, lse_tol) by sequences; rows outside them stay NaN (they are not compared). The weights' error:
    the scores', d products and sums and the scale in f32 twice (the maximum's too), the exp's and n sums; bf16
    on the matrix instructions rounds weights to bf16 and takes an exp good to 1e-4; the output's rounding."""
    n, h, d = q.shape
    g = h // k.shape[1]
    out = torch.full((n, h, d), math.nan, dtype=torch.float64, device=q.device)
    tol, lse, ltol = torch.zeros_like(out), out[..., 0].clone(), torch.zeros_like(out[..., 0])
    q, k, v = q.double(), k.double(), v.double()
    for a, b in zip(starts, starts[1:]):
        if b == a:
            continue
        i = torch.arange(b - a, device=q.device)
        seen = i[None, :] <= i[:, None]
        if window:
            seen &= (i[None, :] > i[:, None] - window) | (i[None, :] < sinks)
        for hh in range(h):
            qq, kk, vv = q[a:b, hh], k[a:b, hh // g], v[a:b, hh // g]
            s = torch.where(seen, scale * (qq @ kk.T), -math.inf)
            big = torch.where(seen, abs(scale) * (qq.abs() @ kk.abs().T), 0.0).amax(-1, keepdim=True)
            m = s.amax(-1, keepdim=True)
            p = torch.exp(s - m)
            total = p.sum(-1, keepdim=True)
            p = p / total
            o = p @ torch.where(vv.isfinite(), vv, 0.0)
            spread = p @ torch.where(vv.isfinite(), vv, 0.0).abs()
            bad = ~vv.isfinite()
            if bool(bad.any()):                            # what a row does not see has no effect on it
                for j in bad.any(-1).nonzero()[:, 0].tolist():
                    o += torch.where(seen[:, j:j + 1] & bad[j][None], vv[j][None], 0.0)
            w = 2 * (d + 4) * 2.0 ** -24 * big + 2.0 ** -21 + (b - a + 16) * 2.0 ** -23
            if matrix:
                w = w + 2.0 ** -8 + 1e-4
            out[a:b, hh] = o
            half = HALF["bf16" if matrix else "f32"]
            tol[a:b, hh] = w * spread + half * o.abs() + 1e-30
            lse[a:b, hh] = (m + torch.log(total))[:, 0]
            ltol[a:b, hh] = ((2 * (d + 4) * 2.0 ** -24 * big + 2.0 ** -21 + (b - a + 16) * 2.0 ** -23)[:, 0]
                             + (1e-4 if matrix else 0.0) + 2.0 ** -22 * (m.abs() + torch.log(total).abs())[:, 0])
    return out, tol, lse, ltol


def sample_exact(torch, logits, temperature, top_k, top_p, min_p, u):
    """(token, logprob) of one row, from the definition, on lists of indexes."""
    x = torch.nan_to_num(logits.double(), nan=-math.inf, posinf=math.inf, neginf=-math.inf).cpu()
    top = float(x.max())
    if top == -math.inf:
        return -1, -math.inf
    if not temperature > 0:
        return int((x == top).nonzero()[0]), 0.0
    e = (x == top).double() if top == math.inf else torch.exp((x - top) / temperature)
    e = torch.where(x == -math.inf, 0.0, e)
    kept = torch.argsort(x, descending=True, stable=True)
    if 0 < top_k < len(x):
        kept = kept[:top_k]
    if top_p < 1:
        sums = torch.cumsum(e[kept], 0)
        kept = kept[:int((sums < max(top_p, 0.0) * sums[-1]).sum()) + 1]
    if min_p > 0:
        kept = kept[e[kept] >= min(min_p, 1.0)]
    kept = torch.sort(kept).values
    sums = torch.cumsum(e[kept], 0)
    u = min(max(u, 0.0), 0.99999994) if u == u else 0.0
    j = min(int((sums <= u * sums[-1]).sum()), int(e[kept].nonzero()[-1]))
    return int(kept[j]), float(torch.log(e[kept[j]] / sums[-1]))
