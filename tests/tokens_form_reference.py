"""Attention on token sequences with capped scores, a bias by distance, documents, groups and prefixes, in 64 bits and from the
formulas, with bounds of what rounding may do.

Beside the roundings that tests/tokens_reference.py counts, a score z = cap tanh(raw / cap) - slope |i - j| is off by what its
Float32 arithmetic and the polynomial for tanh make: relative to |z| by `REL` (the polynomials are good to 6.9e-6, 5.9e-7 and
5e-8; three Float32 operations add 2e-7), and by 3e-7 of the cap where the exponential unit is used (1 - 2 / (1 + e), two
roundings of numbers below 2).  A weight's relative error is the error of its own score and the weights' mean error of the row's.
The cap's derivative 1 - tanh^2 is off by twice the error of tanh, absolutely."""
import math

import torch

from tests.tokens_reference import SLACK, UNIT, check  # noqa: F401

REL = {torch.float32: 4e-7, torch.bfloat16: 7.5e-6, torch.float16: 9e-7}


def spans(documents, groups):
    """For each token of one sequence: (first, last) that it sees; documents and groups are lists."""
    n = len(documents)
    out = []
    for i in range(n):
        if documents[i] < 0:
            out.append((i, i - 1))
            continue
        a = i
        while a > 0 and documents[a - 1] == documents[i]:
            a -= 1
        b = i
        if groups is not None and groups[i] > 0:
            while b + 1 < n and documents[b + 1] == documents[i] and groups[b + 1] == groups[i]:
                b += 1
        out.append((a, b))
    return out


def attend(q, k, v, i, mask, scale, cap, slope, dtype, dy=None):
    """One head: q (n, D) at positions i, k, v (m, D) at 0 .. m-1, mask (n, m).  {name: (value, bound)}."""
    u, rel = UNIT[dtype], REL[dtype]
    j = torch.arange(k.shape[0])
    raw = q @ k.T * scale
    t = torch.tanh(raw / cap) if cap else torch.zeros_like(raw)
    bias = slope * (i[:, None] - j[None]).abs().double()
    capped = cap * t if cap else raw
    z = torch.where(mask, capped - bias, torch.tensor(-math.inf, dtype=torch.float64))
    p = torch.where(mask.any(1, keepdim=True), torch.softmax(z, 1), torch.zeros((), dtype=torch.float64))
    p = torch.where(mask, p, torch.zeros((), dtype=torch.float64))
    size = torch.where(mask, rel * (capped.abs() + 2 * bias.abs()) + 3e-7 * (cap or 0.0), torch.zeros((), dtype=torch.float64))
    slack = SLACK + size + (p * size).sum(1, keepdim=True)
    y = p @ v
    tiny = 2.0 ** -24 * mask.shape[1] if dtype is torch.float16 else 0.0
    # a result of half precision is off by up to half of its smallest step, 2^-24, however small it is
    least = 2.0 ** -25 if dtype is torch.float16 else 0.0
    out = {"y": (y, u * y.abs() + ((u + slack) * p) @ v.abs() + tiny * v.abs().amax() + least)}
    if dy is None:
        return out
    inner = 1 - t * t
    dp, delta = dy @ v.T, (dy * y).sum(1, keepdim=True)
    ds = p * (dp - delta) * inner
    parts = p * (dy.abs() @ v.abs().T + (dy * y).abs().sum(1, keepdim=True))       # what dS is the difference of
    off = p * (u * (dy * y).abs().sum(1, keepdim=True))                            # delta comes from the rounded y
    e = u * ds.abs() + (slack * parts + off) * inner + (2.5 * rel + 1e-6) * parts * bool(cap) + tiny * (u > 0)
    dq, dk, dv = ds @ k * scale, ds.T @ q * scale, p.T @ dy
    out["dq"] = (dq, u * dq.abs() + (e @ k.abs()) * abs(scale) + least)
    out["dk"] = (dk, u * dk.abs() + (e.T @ q.abs()) * abs(scale) + least)
    out["dv"] = (dv, u * dv.abs() + ((u + slack) * p).T @ dy.abs() + tiny * dy.abs().sum(0) + least)
    return out


def window(q, k, v, left, right, sinks, lengths, cap, slopes, documents, groups, dy=None, scale=None):
    """(D, heads, N, B) tensors of the storage's type; documents, groups: lists of lists or None.  {name: (value, bound)}."""
    dtype = q.dtype
    q, k, v = q.double(), k.double(), v.double()
    D, Hq, N, B = q.shape
    G = Hq // k.shape[1]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    like = {"y": q, "dq": q, "dk": k, "dv": v}
    out = {name: (torch.zeros_like(like[name]), torch.zeros_like(like[name])) for name in (like if dy is not None else ("y",))}
    i = torch.arange(N)
    for b in range(B):
        n = N if lengths is None else lengths[b]
        if documents is None:
            lo, hi = torch.zeros(N, dtype=torch.long), i + right
        else:
            lo, hi = torch.tensor(spans(documents[b], groups[b] if groups else None)).reshape(N, 2).T
        back = i - left if left is not None else torch.zeros_like(i)
        a, j = i[:, None], i[None]
        mask = (j >= lo[:, None]) & (j <= hi[:, None]) & ((j >= back[:, None]) | (j < sinks)) & (a < n) & (j < n)
        exists = (i < n)[:, None]
        for h in range(Hq):
            clean = lambda t, hh: torch.where(exists, t[:, hh, :, b].T, torch.zeros((), dtype=torch.float64))
            got = attend(clean(q, h), clean(k, h // G), clean(v, h // G), i, mask, scale, cap, slopes[h] if slopes is not None else 0.0, dtype,
                         None if dy is None else clean(dy.double(), h))
            for name, (x, e) in got.items():
                hh = h if name in ("y", "dq") else h // G
                out[name][0][:, hh, :, b] += x.T
                out[name][1][:, hh, :, b] += e.T
    return out


def paged(q, k_pages, v_pages, table, starts, lengths, left, sinks, cap, slopes, prefix):
    """q (D, heads, T), pools (D, page, heads, pages); table[s], starts, lengths, prefix lists.  (y, bound)."""
    dtype = q.dtype
    q, k_pages, v_pages = q.double(), k_pages.double(), v_pages.double()
    D, Hq, T = q.shape
    page, Hkv, pages = k_pages.shape[1:]
    y, bound = torch.zeros_like(q), torch.zeros_like(q)
    zero = torch.zeros((), dtype=torch.float64)
    for s, n in enumerate(lengths):
        t0, t1 = starts[s], starts[s + 1]
        if t0 == t1:
            continue
        j, i = torch.arange(n), torch.arange(n - (t1 - t0), n)
        hi = i if prefix is None else i.clamp(min=prefix[s] - 1)
        a = i[:, None]
        mask = (a >= 0) & (j <= hi[:, None]) & ((j >= (a - left if left is not None else 0)) | (j < sinks))
        where = torch.tensor([table[s][x // page] if x // page < len(table[s]) else -1 for x in range(n)], dtype=torch.long)
        have = (where >= 0) & (where < pages) & mask.any(0)
        mask = mask & have[None]
        w = where.clamp(0, max(pages - 1, 0))
        for h in range(Hq):
            kk, vv = (torch.where(have[:, None], p[:, j % page, h // (Hq // Hkv), w].T, zero) for p in (k_pages, v_pages))
            got = attend(q[:, h, t0:t1].T, kk, vv, i, mask, 1.0 / math.sqrt(D), cap, slopes[h] if slopes is not None else 0.0, dtype)["y"]
            y[:, h, t0:t1], bound[:, h, t0:t1] = got[0].T, got[1].T
    return y, bound
