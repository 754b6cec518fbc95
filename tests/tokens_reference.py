"""The operators on token sequences in 64 bits, from their formulas, and how far a result rounded to few bits may be off.

`u` is the unit roundoff of the storage.  A result y = sum_j p_j v_j whose weights are rounded to that type before the
product and which is rounded itself is off by at most u |y| + u sum |p_j v_j|; the gradients accordingly.  `slack` covers the
Float32 arithmetic in between: scores of size s carry an error of about s 2^-22, which is what the weights' relative error
is; 2e-5 leaves room for scores of some tens."""
import math

import torch

UNIT = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SLACK = 2e-5


def visible(i, j, n, left, right, sinks):
    """(queries, keys) truth values; left None: no left end."""
    i, j = i[:, None], j[None]
    near = (j >= i - left) if left is not None else torch.ones_like(j >= i)
    return (i >= 0) & (i < n) & (j >= 0) & (j < n) & (j <= i + right) & (near | (j < sinks))


def attend(q, k, v, mask, scale, dy=None, u=0.0):
    """One head: q (n, D), k, v (m, D), mask (n, m).  Returns {name: (value, bound)} for y and, with dy, dq, dk, dv."""
    zero = torch.zeros((), dtype=torch.float64)
    s = torch.where(mask, q @ k.T * scale, torch.tensor(-math.inf, dtype=torch.float64))
    p = torch.where(mask.any(1, keepdim=True), torch.softmax(s, 1), zero)
    p = torch.where(mask, p, zero)
    y = p @ v
    tiny = 2.0 ** -24 * mask.shape[1] if u == 2.0 ** -11 else 0.0       # weights below the smallest normal half
    ya = p @ v.abs()
    out = {"y": (y, u * y.abs() + (u + SLACK) * ya + tiny * v.abs().amax())}
    if dy is None:
        return out
    dp = dy @ v.T
    delta = (dy * y).sum(1, keepdim=True)
    ds = p * (dp - delta)
    size = p * (dy.abs() @ v.abs().T + (dy * y).abs().sum(1, keepdim=True))     # what dS is the difference of
    off = p * (u * (dy * y).abs().sum(1, keepdim=True))                         # delta comes from the rounded y
    e = u * ds.abs() + SLACK * size + off + tiny * (u > 0)
    dq, dk, dv = ds @ k * scale, ds.T @ q * scale, p.T @ dy
    out["dq"] = (dq, u * dq.abs() + (e @ k.abs()) * scale)
    out["dk"] = (dk, u * dk.abs() + (e.T @ q.abs()) * scale)
    out["dv"] = (dv, u * dv.abs() + (u + SLACK) * (p.T @ dy.abs()) + tiny * dy.abs().sum(0))
    return out


def window(q, k, v, left, right, sinks, lengths, scale=None, dy=None, u=0.0):
    """(D, heads, N, B) tensors in 64 bits on the CPU.  Returns {name: (value, bound)}."""
    D, Hq, N, B = q.shape
    G = Hq // k.shape[1]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    at = torch.arange(N)
    like = {"y": q, "dq": q, "dk": k, "dv": v}
    out = {name: (torch.zeros_like(like[name]), torch.zeros_like(like[name])) for name in (like if dy is not None else ("y",))}
    for b in range(B):
        n = N if lengths is None else lengths[b]
        mask = visible(at, at, n, left, right, sinks)
        for h in range(Hq):
            clean = lambda t, hh: torch.where((at < n)[:, None], t[:, hh, :, b].T, torch.zeros((), dtype=torch.float64))
            got = attend(clean(q, h), clean(k, h // G), clean(v, h // G), mask, scale, None if dy is None else clean(dy, h), u)
            for name, (x, e) in got.items():
                hh = h if name in ("y", "dq") else h // G
                out[name][0][:, hh, :, b] += x.T
                out[name][1][:, hh, :, b] += e.T
    return out


def paged(q, k_pages, v_pages, table, starts, lengths, left, sinks, scale=None, u=0.0):
    """q (D, heads, T), pools (D, page, heads, pages) in 64 bits on the CPU; table, starts, lengths lists.  (y, bound)."""
    D, Hq, T = q.shape
    page, Hkv, pages = k_pages.shape[1:]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    y, bound = torch.zeros_like(q), torch.zeros_like(q)
    for s, n in enumerate(lengths):
        t0, t1 = starts[s], starts[s + 1]
        if t0 == t1:
            continue
        j = torch.arange(n)
        i = torch.arange(n - (t1 - t0), n)
        mask = visible(i, j, n, left, 0, sinks)
        where = torch.tensor([table[s][x // page] if x // page < len(table[s]) else -1 for x in range(n)], dtype=torch.long)
        have = (where >= 0) & (where < pages) & mask.any(0)
        mask = mask & have[None]
        w = where.clamp(0, max(pages - 1, 0))
        for h in range(Hq):
            g = h // (Hq // Hkv)
            kk, vv = (torch.where(have[:, None], p[:, j % page, g, w].T, torch.zeros((), dtype=torch.float64)) for p in (k_pages, v_pages))
            got = attend(q[:, h, t0:t1].T, kk, vv, mask, scale, None, u)["y"]
            y[:, h, t0:t1], bound[:, h, t0:t1] = got[0].T, got[1].T
    return y, bound


def rotary(x, positions, freqs, sections, interleaved, inverse=False):
    """x (D, heads, N, B) in 64 bits, positions (axes, N, B) integers, freqs: radians per position as Python floats."""
    out = x.clone()
    pairs = len(freqs)
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    for p in range(pairs):
        a = positions[axis[p]].double() * freqs[p] * (-1.0 if inverse else 1.0)
        c, s = torch.cos(a)[None], torch.sin(a)[None]
        i, j = (2 * p, 2 * p + 1) if interleaved else (p, p + pairs)
        out[i], out[j] = x[i] * c - x[j] * s, x[i] * s + x[j] * c
    return out


def check(got, want, bound, what=""):
    """|got - want| <= bound for every element, got having the storage's type."""
    got = got.detach().double().cpu()
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} for {tuple(want.shape)}"
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = (got - want).abs() - bound - 1e-30
    worst = int(over.argmax()) if over.numel() else 0
    assert not over.numel() or over.max() <= 0, (f"{what}: off by {float((got - want).abs().flatten()[worst]):.3g}, "
                                                 f"{float(bound.flatten()[worst]):.3g} allowed, value {float(want.flatten()[worst]):.3g}")
