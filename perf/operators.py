"""Performance cases of the operators on token sequences: rotary positions, attention with a sliding window and first
tokens that stay visible, and the same attention over a paged cache.

A case is a dict of plain values.  `kind` says which operator:

    "rotate"   rotary positions with several axes on q and k, and the gradients of both for given cotangents
    "append"   the serving form: a chunk of new tokens is rotated and its k, v are written into a paged cache
    "window"   y = attention of every token to a window of its neighbours and to the first tokens; with `train` the
               gradients of q, k, v too
    "paged"    attention of a chunk of new tokens (one token per sequence: decoding) to a paged cache

Tensors have the framework's Julia-shaped column-major layout: (D, heads, N, B) of dense ones, (D, heads, T) of the packed
tokens of several sequences, (D, page, heads, pages) of a cache.  `left` = -1 means that the window has no left end."""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}


# ------------------------------------------------------------------------------------------------ cases
def _rotate(dtype, D, Hq, Hkv, N, B, axes, interleaved=False, rot=0, name=None):
    return _named(dict(kind="rotate", dtype=dtype, D=D, Hq=Hq, Hkv=Hkv, N=N, B=B, axes=axes, interleaved=interleaved, rot=rot or D), name)


def _append(dtype, D, Hq, Hkv, S, chunk, history, page, axes=1, interleaved=False, name=None):
    return _named(dict(kind="append", dtype=dtype, D=D, Hq=Hq, Hkv=Hkv, S=S, chunk=chunk, history=history, page=page, axes=axes,
                       interleaved=interleaved), name)


def _window(dtype, D, Hq, Hkv, N, B, left, right, sinks, train, ragged=False, name=None):
    return _named(dict(kind="window", dtype=dtype, D=D, Hq=Hq, Hkv=Hkv, N=N, B=B, left=left, right=right, sinks=sinks, train=train,
                       ragged=ragged), name)


def _paged(dtype, D, Hq, Hkv, S, chunk, history, page, left, sinks, name=None):
    return _named(dict(kind="paged", dtype=dtype, D=D, Hq=Hq, Hkv=Hkv, S=S, chunk=chunk, history=history, page=page, left=left,
                       sinks=sinks), name)


def _named(case, name):
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # One new token for each of a few sequences, a small model: only latency counts.
        _append("bf16", 64, 8, 2, 8, 1, 900, 16, name="append one token"),
        # A batch of prompts of mixed lengths enters the cache.
        _append("f16", 128, 32, 8, 32, 900, 2000, 64, axes=3, interleaved=True, name="append prompts"),
        # The quickstart image's pixels as tokens with two axes, Float32.
        _rotate("f32", 64, 4, 4, 12288, 2, 2, name="rotate image train"),
        # A video clip: time, height and width, shared key heads.
        _rotate("bf16", 128, 16, 4, 16384, 2, 3, interleaved=True, name="rotate video train"),
        # A short prompt in evaluation, odd length.
        _window("bf16", 64, 4, 1, 257, 1, 63, 0, 2, False, name="window short infer"),
        # Records of unequal odd lengths, a centred window like the circulant one but without the wrap.
        _window("f16", 64, 8, 8, 5001, 3, 63, 63, 0, True, ragged=True, name="window records train"),
        # Float32 training.
        _window("f32", 64, 8, 8, 4096, 2, 255, 0, 4, True, name="window f32 train"),
        # The training step of a long-context layer with shared key heads.
        _window("bf16", 128, 16, 4, 16384, 2, 1023, 0, 4, True, name="window long train"),
        # A whole document in evaluation.
        _window("bf16", 128, 16, 2, 65536, 1, 4095, 0, 16, False, name="window document infer"),
        # A few conversations, one token each, the whole history visible.
        _paged("bf16", 128, 16, 4, 4, 1, 3000, 32, -1, 0, name="decode few"),
        # A full serving batch, ragged histories, window and first tokens; pages that left the window are freed.
        _paged("bf16", 128, 32, 8, 64, 1, 30000, 16, 4095, 16, name="decode batch"),
        # Chunks of prompts next to single tokens.
        _paged("f16", 128, 16, 2, 12, 900, 6000, 64, 2047, 4, name="chunks mixed"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _flops(case):
    return work(case)["flops"]


def draw(rng):
    """One more case of the ranges the listed ones stand for."""
    while True:
        kind = rng.choice(("rotate", "append", "window", "window", "window", "paged", "paged", "paged"))
        dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
        D = rng.choice((32, 64, 64, 80, 96, 128, 128))
        Hkv = rng.choice((1, 2, 3, 4, 8))
        Hq = Hkv * rng.choice((1, 1, 2, 3, 4, 8))
        if kind == "rotate":
            axes = rng.choice((1, 2, 3))
            case = _rotate(dtype, D, Hq, Hkv, _log_int(rng, 1, 32768), _log_int(rng, 1, 4), axes, rng.random() < 0.5,
                           rng.choice((D, D, D // 2)))
            if work(case)["bytes"] > 1.5e9:
                continue
            return case
        S = _log_int(rng, 1, 64)
        page = rng.choice((16, 16, 32, 48, 64, 128, 256))
        if kind == "append":
            case = _append(dtype, D, Hq, Hkv, S, 1 if rng.random() < 0.5 else _log_int(rng, 2, 1500), _log_int(rng, 1, 8000), page,
                           rng.choice((1, 2, 3)), rng.random() < 0.5)
            if work(case)["bytes"] > 1.5e9 or S * (case["chunk"] + case["history"]) * Hkv * D > 1e9:
                continue
            return case
        sinks = rng.choice((0, 1, 4, 4, 16, 130))
        if kind == "window":
            N, B = _log_int(rng, 1, 32768), _log_int(rng, 1, 6)
            train = rng.random() < 0.6
            left = -1 if rng.random() < 0.2 else _log_int(rng, 1, 4000)
            right = 0 if rng.random() < 0.7 else _log_int(rng, 1, 500)
            span = (N if left < 0 else min(left, N)) + min(right, N) + 256 + sinks
            case = _window(dtype, D, Hq, Hkv, N, B, left, right, sinks, train, rng.random() < 0.4)
            if B * Hq * N * span > (7e8 if train else 2e9) or _flops(case) > (2e11 if dtype == "f32" else 9e11):
                continue
            return case
        one = rng.random() < 0.5
        chunk, history = 1 if one else _log_int(rng, 2, 1500), _log_int(rng, 1, 60000)
        left = -1 if rng.random() < 0.4 else _log_int(rng, 16, 8000)
        case = _paged(dtype, D, Hq, Hkv, S, chunk, history, page, left, sinks)
        span = min(history + chunk, left + chunk if left >= 0 else history + chunk) + sinks
        if S * Hq * chunk * span > 1.5e9 or S * Hkv * span * D > 1.2e9 or _flops(case) > (2e11 if dtype == "f32" else 9e11):
            continue
        return case


# ------------------------------------------------------------------------------------------------ what a case fixes
def _sections(case):
    """Pairs of features that turn with each axis: time gets the smallest share."""
    pairs, axes = case.get("rot", case["D"]) // 2, case["axes"]
    first = pairs - (axes - 1) * (pairs * 3 // 8) if axes > 1 else pairs
    return (first,) + (pairs * 3 // 8,) * (axes - 1)


def _dense_lengths(case):
    """Tokens of each sequence of a dense batch: all N, or unequal ones."""
    return [case["N"] - (case["N"] * b) // (2 * case["B"]) if case["ragged"] else case["N"] for b in range(case["B"])]


def _chunks(case):
    """(new tokens, tokens in the cache with them) of each sequence: unequal histories, and among larger chunks some
    sequences with a single token and one with none."""
    rng = random.Random(case["S"] * 1000003 + case["history"] * 101 + case["chunk"])
    out = []
    for s in range(case["S"]):
        new = case["chunk"] if case["chunk"] == 1 else (1, rng.randint(1, case["chunk"]), case["chunk"], rng.randint(1, case["chunk"]))[s % 4]
        if case["chunk"] > 1 and s == 6:
            new = 0
        out.append((new, new + rng.randint(case["history"] // 2, case["history"])))
    return out


def _first_visible(case, new, total):
    """First position in the window of the first new token."""
    return 0 if case.get("left", -1) < 0 else max(0, total - new - case["left"])


def _pairs(case):
    """(query, key) pairs that are visible, per query head, and the tokens of the cache that are visible to any query."""
    if case["kind"] == "window":
        seen, keys = 0, 0
        for n in _dense_lengths(case):
            i = torch.arange(n, dtype=torch.float64)
            left, right = (n if case["left"] < 0 else case["left"]), case["right"]
            lo = (i - left).clamp(min=0)
            hi = (i + right).clamp(max=n - 1)
            seen += float((hi - lo + 1 + torch.minimum(lo, torch.tensor(float(case["sinks"])))).sum())
            keys += n
        return seen, keys
    seen, keys = 0, 0
    for new, total in _chunks(case):
        i = torch.arange(total - new, total, dtype=torch.float64)
        lo = (i - (total if case["left"] < 0 else case["left"])).clamp(min=0)
        seen += float((i - lo + 1 + torch.minimum(lo, torch.tensor(float(case["sinks"])))).sum())
        if new:
            first = _first_visible(case, new, total)
            keys += total - first + min(case["sinks"], first)
    return seen, keys


def work(case):
    """Every input read once, every output written once.  Attention: two operations for each visible pair and feature of
    each contraction: two contractions forward and five backward (the scores are not kept)."""
    e, D, Hq, Hkv = BYTES[case["dtype"]], case["D"], case["Hq"], case["Hkv"]
    if case["kind"] == "rotate":
        tokens = case["N"] * case["B"]
        return {"bytes": 4 * tokens * (Hq + Hkv) * D * e + 4 * tokens * case["axes"], "flops": 6 * tokens * (Hq + Hkv) * case["rot"]}
    if case["kind"] == "append":
        tokens = sum(new for new, _ in _chunks(case))
        return {"bytes": 2 * tokens * (Hq + 2 * Hkv) * D * e + 4 * tokens * case["axes"], "flops": 3 * tokens * (Hq + Hkv) * D}
    seen, keys = _pairs(case)
    if case["kind"] == "window":
        tokens = case["N"] * case["B"]
        if case["train"]:   # q, k, v, y's cotangent in; y and three gradients out
            return {"bytes": tokens * (4 * Hq + 4 * Hkv) * D * e, "flops": 14 * seen * Hq * D}
        return {"bytes": tokens * (2 * Hq + 2 * Hkv) * D * e, "flops": 4 * seen * Hq * D}
    tokens = sum(new for new, _ in _chunks(case))
    return {"bytes": (2 * tokens * Hq + 2 * keys * Hkv) * D * e, "flops": 4 * seen * Hq * D}


# ------------------------------------------------------------------------------------------------ inputs
class _State:
    pass


def _julia(shape, dtype, gen, scale=1.0):
    """Standard normal Julia-shaped tensor times `scale`."""
    t = torch.randn(tuple(reversed(shape)), dtype=dtype, device="cuda", generator=gen)
    t = t * scale if scale != 1.0 else t
    return t.permute(tuple(range(len(shape) - 1, -1, -1)))


def _columns(rows, dtype=torch.int32):
    """List of rows (lists) -> Julia-shaped integer tensor whose column s is rows[s]."""
    return torch.tensor(rows, dtype=dtype, device="cuda").t()


def _turns(case, gen=None):
    """Turns per position of each pair, base 10000, as a fraction of 2^64 (64-bit two's complement)."""
    pairs = case.get("rot", case["D"]) // 2
    fixed = [int(round(10000.0 ** (-p / pairs) / (2 * math.pi) * 2.0 ** 64)) for p in range(pairs)]
    return torch.tensor([f - (1 << 64) if f >= (1 << 63) else f for f in fixed], dtype=torch.int64, device="cuda")


def _grid_positions(case, n, start, gen):
    """Positions of n tokens on each axis: a running index; with several axes frames of rows and columns."""
    i = torch.arange(start, start + n, device="cuda", dtype=torch.int32)
    if case["axes"] == 1:
        return i[None]
    width, height = 32, 24
    yx = torch.stack([torch.div(i, width, rounding_mode="floor") % height, i % width])
    return yx if case["axes"] == 2 else torch.cat([torch.div(i, width * height, rounding_mode="floor")[None], yx])


def prepare(case, seed):
    """Normal tensors whose scores spread like those of trained heads (queries a little larger than unit, keys of the
    first tokens larger and alike, so that they draw weight), positions, page tables in random order."""
    gen = torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFFFFFF)
    rng = random.Random(int(seed))
    dtype = DTYPES[case["dtype"]]
    D, Hq, Hkv = case["D"], case["Hq"], case["Hkv"]
    s = _State()
    s.case = case
    if case["kind"] == "rotate":
        N, B = case["N"], case["B"]
        s.q, s.k = _julia((D, Hq, N, B), dtype, gen).requires_grad_(True), _julia((D, Hkv, N, B), dtype, gen).requires_grad_(True)
        s.dq, s.dk = _julia((D, Hq, N, B), dtype, gen), _julia((D, Hkv, N, B), dtype, gen)
        start = rng.randrange(0, 100000)
        pos = torch.stack([_grid_positions(case, N, start + 1000 * b, gen) for b in range(B)])      # (B, axes, N)
        s.positions = pos.permute(0, 2, 1).contiguous().permute(2, 1, 0)                            # (axes, N, B)
        s.turns = _turns(case)
        return s
    if case["kind"] == "window":
        N, B, grad = case["N"], case["B"], case["train"]
        s.q = _julia((D, Hq, N, B), dtype, gen, 1.5)
        s.k = _julia((D, Hkv, N, B), dtype, gen)
        s.v = _julia((D, Hkv, N, B), dtype, gen)
        n = min(case["sinks"], N)
        if n:
            s.k[:, :, :n] = s.k[:, :, :1] * 1.5
        s.q, s.k, s.v = (t.requires_grad_(grad) for t in (s.q, s.k, s.v))
        s.dy = _julia((D, Hq, N, B), dtype, gen) if grad else None
        s.lengths = torch.tensor(_dense_lengths(case), dtype=torch.int32, device="cuda") if case["ragged"] else None
        return s
    # a cache: pages of every sequence in random order, those that no new token sees are freed (-1)
    page, chunks = case["page"], _chunks(case)
    need = []
    for new, total in chunks:
        first = _first_visible(case, new, total)
        live = [p * page + page > first or p * page < case.get("sinks", 0) for p in range(-(-total // page))]
        if case["kind"] == "append":      # only the pages that the new tokens enter
            live = [p * page + page > total - new for p in range(-(-total // page))]
        need.append(live)
    count = sum(sum(live) for live in need) + 3
    free = list(range(count))
    rng.shuffle(free)
    width = max(len(live) for live in need) + 1
    s.table = _columns([[free.pop() if on else -1 for on in live] + [-1] * (width - len(live)) for live in need])
    s.lengths = torch.tensor([total for _, total in chunks], dtype=torch.int32, device="cuda")
    starts = [0]
    for new, _ in chunks:
        starts.append(starts[-1] + new)
    s.starts = torch.tensor(starts, dtype=torch.int32, device="cuda")
    T = starts[-1]
    s.k_pages, s.v_pages = _julia((D, page, Hkv, count), dtype, gen), _julia((D, page, Hkv, count), dtype, gen)
    s.q = _julia((D, Hq, T), dtype, gen, 1.5)
    if case["kind"] == "append":
        s.k, s.v = _julia((D, Hkv, T), dtype, gen), _julia((D, Hkv, T), dtype, gen)
        parts = [_grid_positions(case, new, total - new, gen) for new, total in chunks]
        s.positions = torch.cat(parts, 1).t().contiguous().t()                                      # (axes, T)
        s.turns = _turns(case)
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _rotate_plain(x, positions, turns, sections, interleaved, sign=1.0):
    """x (D, heads, tokens...); positions (axes, tokens...): each pair turned by position * turns, angles reduced exactly
    in integers."""
    axis = torch.repeat_interleave(torch.arange(len(sections), device=x.device), torch.tensor(sections, device=x.device))
    phase = positions.long()[axis] * turns.reshape((-1,) + (1,) * (positions.ndim - 1))             # mod 2^64 turns
    angle = (phase >> 32).float() * (math.pi / 2.0 ** 31)
    c, s = torch.cos(angle)[:, None], sign * torch.sin(angle)[:, None]
    n = turns.numel()
    f = x.float()
    a, b = (f[0:2 * n:2], f[1:2 * n:2]) if interleaved else (f[:n], f[n:2 * n])
    u, w = a * c - b * s, a * s + b * c
    turned = torch.stack([u, w], 1).reshape((2 * n,) + x.shape[1:]) if interleaved else torch.cat([u, w])
    return torch.cat([turned, f[2 * n:]]).to(x.dtype)


def _token_places(s):
    """Sequence and position in its cache of every packed token."""
    T = s.q.shape[2]
    t = torch.arange(T, device="cuda")
    seq = torch.searchsorted(s.starts.long(), t, right=True) - 1
    position = s.lengths.long()[seq] - s.starts.long()[seq + 1] + t
    return seq, position


def _softmax_times(scores, mask, v):
    """softmax over the visible columns times v; rows that see nothing give zeros."""
    scores = scores.masked_fill(~mask, -math.inf)
    top = scores.amax(-1, keepdim=True).detach()
    p = torch.exp(scores - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    return torch.matmul(p, v) / p.sum(-1, keepdim=True).clamp(min=1e-30)


def _window_plain(q, k, v, left, right, sinks, lengths):
    """Blocks of queries against the keys from the first one's window to the last one's, and the first tokens as further
    columns for the queries whose window does not reach them."""
    D, Hq, N, B = q.shape
    Hkv = k.shape[1]
    G = Hq // Hkv
    left, right, sinks = N if left < 0 else min(left, N), min(right, N), min(sinks, N)
    block = 256
    nb = -(-N // block)
    span, dev = block + left + right, q.device
    pad = torch.nn.functional.pad
    Q = pad(q.permute(3, 1, 2, 0).float(), (0, 0, 0, nb * block - N)) / math.sqrt(D)
    Q = Q.reshape(B, Hkv, G, nb, block, D).transpose(2, 3).reshape(B, Hkv, nb, G * block, D)
    K, V = (t.permute(3, 1, 2, 0).float() for t in (k, v))
    Kb, Vb = (pad(t, (0, 0, left, right + nb * block - N)).unfold(2, span, block) for t in (K, V))   # (B, Hkv, nb, D, span)
    firstK, firstV = (t[:, :, None, :sinks].expand(B, Hkv, nb, sinks, D) for t in (K, V))
    keys, values = torch.cat([Kb.transpose(3, 4), firstK], 3), torch.cat([Vb.transpose(3, 4), firstV], 3)
    scores = torch.matmul(Q, keys.transpose(3, 4))
    n = torch.full((B,), N, device=dev) if lengths is None else lengths.long()
    n = n.reshape(B, 1, 1, 1)
    i = torch.arange(nb * block, device=dev).reshape(1, nb, block, 1)
    j = torch.arange(nb, device=dev).reshape(1, nb, 1, 1) * block - left + torch.arange(span, device=dev)
    near = (j >= 0) & (j < n) & (j >= i - left) & (j <= i + right) & (i < n)
    j = torch.arange(sinks, device=dev)
    first = (j < i - left) & (j < n) & (i < n)
    mask = torch.cat([near, first], 3)[:, None, :, None].expand(B, 1, nb, G, block, span + sinks).reshape(B, 1, nb, G * block, -1)
    y = _softmax_times(scores, mask, values)
    y = y.reshape(B, Hkv, nb, G, block, D).transpose(2, 3).reshape(B, Hq, nb * block, D)[:, :, :N]
    return y.transpose(1, 2).contiguous().to(q.dtype).permute(3, 2, 1, 0)


def _paged_plain(s):
    """Queries padded to the longest chunk, the keys that any of a sequence's queries sees gathered from its pages."""
    case = s.case
    D, Hq, T = s.q.shape
    page, Hkv = s.k_pages.shape[1], s.k_pages.shape[2]
    G, S, dev = Hq // Hkv, s.lengths.numel(), s.q.device
    chunks = _chunks(case)
    most, longest = max(max(new for new, _ in chunks), 1), max(total for _, total in chunks)
    left = longest if case["left"] < 0 else case["left"]
    seq, position = _token_places(s)
    new = (s.starts[1:] - s.starts[:-1]).long()
    row = torch.arange(T, device=dev) - s.starts.long()[seq]
    Q = torch.zeros(S, most, Hq, D, device=dev)
    Q[seq, row] = s.q.permute(2, 1, 0).float() / math.sqrt(D)
    begin = (s.lengths.long() - new - left).clamp(min=0)
    near = begin[:, None] + torch.arange(min(longest, left + most), device=dev)                      # (S, near)
    j = torch.cat([torch.arange(case["sinks"], device=dev).expand(S, -1), near], 1)                  # (S, keys)
    first = torch.arange(j.shape[1], device=dev) < case["sinks"]
    where = s.table.t().long().gather(1, torch.div(j, page, rounding_mode="floor").clamp(max=s.table.shape[0] - 1))
    at = (where.clamp(min=0)[..., None] * Hkv + torch.arange(Hkv, device=dev)) * page + (j % page)[..., None]
    K, V = (t.permute(3, 2, 1, 0).reshape(-1, D)[at.transpose(1, 2)].float() for t in (s.k_pages, s.v_pages))
    Q = Q.reshape(S, most, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(S, Hkv, G * most, D)
    i = (s.lengths.long() - new)[:, None, None] + torch.arange(most, device=dev)[None, :, None]      # (S, most, 1)
    j = j[:, None]
    mask = torch.where(first, j < i - left, (j >= i - left) & (j <= i)) & (j < s.lengths.long()[:, None, None])
    mask = mask[:, None, None].expand(S, 1, G, most, -1).reshape(S, 1, G * most, -1)
    y = _softmax_times(torch.matmul(Q, K.transpose(2, 3)), mask, V)
    y = y.reshape(S, Hkv, G, most, D).permute(0, 3, 1, 2, 4).reshape(S, most, Hq, D)
    return y[seq, row].to(s.q.dtype).permute(2, 1, 0)


# ------------------------------------------------------------------------------------------------ one pass
def _run_plain(s):
    case = s.case
    if case["kind"] == "rotate":
        args = (s.positions, s.turns, _sections(case), case["interleaved"])
        with torch.no_grad():       # the gradient of a rotation is the rotation back
            return {"q": _rotate_plain(s.q, *args), "k": _rotate_plain(s.k, *args),
                    "grads": (_rotate_plain(s.dq, *args, sign=-1.0), _rotate_plain(s.dk, *args, sign=-1.0))}
    if case["kind"] == "append":
        args = (s.positions, s.turns, _sections(case), case["interleaved"])
        seq, position = _token_places(s)
        page = s.k_pages.shape[1]
        where = s.table[torch.div(position, page, rounding_mode="floor"), seq].long()
        k_pages, v_pages = s.k_pages.permute(3, 1, 2, 0), s.v_pages.permute(3, 1, 2, 0)
        k_pages[where, position % page] = _rotate_plain(s.k, *args).permute(2, 1, 0)
        v_pages[where, position % page] = s.v.permute(2, 1, 0)
        return {"q": _rotate_plain(s.q, *args), "k_pages": s.k_pages, "v_pages": s.v_pages}
    if case["kind"] == "window":
        y = _window_plain(s.q, s.k, s.v, case["left"], case["right"], case["sinks"], s.lengths)
        if not case["train"]:
            return {"y": y}
        return {"y": y.detach(), "grads": torch.autograd.grad(y, (s.q, s.k, s.v), s.dy)}
    return {"y": _paged_plain(s)}


def _run_own(s):
    from __graft_entry__ import load_package
    ca = load_package()
    case = s.case
    left = None if case.get("left", -1) < 0 else case["left"]
    if case["kind"] == "rotate":
        q, k = ca.rotary((s.q, s.k), s.positions, s.turns, sections=_sections(case), interleaved=case["interleaved"])
        return {"q": q.detach(), "k": k.detach(), "grads": torch.autograd.grad((q, k), (s.q, s.k), (s.dq, s.dk))}
    if case["kind"] == "append":
        q = ca.rotary_append_(s.q, s.k, s.v, s.k_pages, s.v_pages, s.table, s.starts, s.lengths, s.positions, s.turns,
                              sections=_sections(case), interleaved=case["interleaved"])
        return {"q": q, "k_pages": s.k_pages, "v_pages": s.v_pages}
    if case["kind"] == "window":
        y = ca.window_attention(s.q, s.k, s.v, left, right=case["right"], sinks=case["sinks"], lengths=s.lengths)
        if not case["train"]:
            return {"y": y}
        return {"y": y.detach(), "grads": torch.autograd.grad(y, (s.q, s.k, s.v), s.dy)}
    return {"y": ca.paged_window_attention(s.q, s.k_pages, s.v_pages, s.table, s.starts, s.lengths, left, sinks=case["sinks"])}


def run(s):
    return _run_own(s) if own else _run_plain(s)


# ------------------------------------------------------------------------------------------------ 64 bits
def _rotated64(x, positions, case, sign):
    """Complex multiplication of each pair by exp(i * sign * position * 10000^(-p / pairs))."""
    pairs = case.get("rot", case["D"]) // 2
    x = x.detach().double()
    out = x.clone()
    p0 = 0
    for axis, n in enumerate(_sections(case)):
        for p in range(p0, p0 + n):
            w = torch.polar(torch.ones(positions.shape[1:], dtype=torch.float64, device="cuda"),
                            sign * positions[axis].double() * 10000.0 ** (-p / pairs))[None]
            a, b = (2 * p, 2 * p + 1) if case["interleaved"] else (p, p + pairs)
            z = torch.complex(x[a], x[b]) * w
            out[a], out[b] = z.real, z.imag
        p0 += n
    return out


def _attend64(q, k, v, i, j, n, left, right, sinks, dy=None):
    """One head in 64 bits: queries at positions i, keys at positions j, n tokens; with dy also (dq, dk, dv)."""
    y, dq = torch.zeros_like(q), torch.zeros_like(q)
    dk, dv = torch.zeros_like(k), torch.zeros_like(v)
    for lo in range(0, q.shape[0], 4096):
        rows = slice(lo, lo + 4096)
        a = i[rows, None]
        sees = (j < n) & (a < n) & (j <= a + right) & ((j < sinks) | (j >= a - left))
        cols = sees.any(0).nonzero()[:, 0]
        if not cols.numel():
            continue
        kk, vv, sees = k[cols], v[cols], sees[:, cols]
        w = torch.where(sees, q[rows] @ kk.T * (q.shape[1] ** -0.5), torch.tensor(-math.inf, dtype=q.dtype, device=q.device))
        p = torch.nan_to_num(torch.softmax(w, 1))
        y[rows] = p @ vv
        if dy is not None:
            dp = dy[rows] @ vv.T
            ds = p * (dp - (p * dp).sum(1, keepdim=True)) * (q.shape[1] ** -0.5)
            dq[rows] = ds @ kk
            dk[cols] += ds.T @ q[rows]
            dv[cols] += p.T @ dy[rows]
    return y, dq, dk, dv


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return _exact(case, s)


def _exact(case, s):
    if case["kind"] == "rotate":
        return {"q": _rotated64(s.q, s.positions, case, 1), "k": _rotated64(s.k, s.positions, case, 1),
                "grads": (_rotated64(s.dq, s.positions, case, -1), _rotated64(s.dk, s.positions, case, -1))}
    chunks = None if case["kind"] == "window" else _chunks(case)
    if case["kind"] == "append":
        k, page = _rotated64(s.k, s.positions, case, 1), case["page"]
        k_pages, v_pages = s.k_pages.double(), s.v_pages.double()
        table, t = s.table.tolist(), 0
        for b, (new, total) in enumerate(chunks):
            at = total - new
            while at < total:
                n = min(total, at - at % page + page) - at
                where = table[at // page][b]
                k_pages[:, at % page:at % page + n, :, where] = k[:, :, t:t + n].transpose(1, 2)
                v_pages[:, at % page:at % page + n, :, where] = s.v[:, :, t:t + n].transpose(1, 2).double()
                at, t = at + n, t + n
        return {"q": _rotated64(s.q, s.positions, case, 1), "k_pages": k_pages, "v_pages": v_pages}
    G = case["Hq"] // case["Hkv"]
    far = 1 << 40
    left = far if case["left"] < 0 else case["left"]
    y = torch.zeros(s.q.shape, dtype=torch.float64, device="cuda")
    if case["kind"] == "window":
        i = torch.arange(case["N"], device="cuda")
        dq = torch.zeros_like(y)
        dk, dv = (torch.zeros(s.k.shape, dtype=torch.float64, device="cuda") for _ in range(2))
        for b, n in enumerate(_dense_lengths(case)):
            for h in range(case["Hq"]):
                args = [t[:, hh, :, b].T.double() for t, hh in ((s.q, h), (s.k, h // G), (s.v, h // G))]
                dy = s.dy[:, h, :, b].T.double() if case["train"] else None
                got = _attend64(*args, i, i, n, left, case["right"], case["sinks"], dy)
                y[:, h, :, b], dq[:, h, :, b] = got[0].T, got[1].T
                dk[:, h // G, :, b] += got[2].T
                dv[:, h // G, :, b] += got[3].T
        return {"y": y, "grads": (dq, dk, dv)} if case["train"] else {"y": y}
    page, t = case["page"], 0
    for b, (new, total) in enumerate(chunks):
        if not new:
            continue
        first = _first_visible(case, new, total)
        j = torch.tensor([x for x in range(total) if x >= first or x < case["sinks"]], device="cuda")
        where, off = s.table[j // page, b].long(), j % page
        i = torch.arange(total - new, total, device="cuda")
        for h in range(case["Hq"]):
            kk, vv = (pool[:, off, h // G, where].T.double() for pool in (s.k_pages, s.v_pages))
            y[:, h, t:t + new] = _attend64(s.q[:, h, t:t + new].T.double(), kk, vv, i, j, total, left, 0, case["sinks"])[0].T
        t += new
    return {"y": y}
