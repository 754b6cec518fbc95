"""Attention on token sequences with capped scores, a bias by distance, documents, groups and prefixes: forward and gradients
against the formulas in 64 bits with derived bounds (tests/tokens_form_reference.py), against differences, masked places,
streams, graphs, and a run of the operators together."""
import math
import random

import pytest
import torch

from tests import tokens_form_reference as ref
from tests.test_gpu_tokens_window import make

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def ints(rows):
    return torch.tensor(rows, dtype=torch.int32, device="cuda")


def numbers(N, B, longest, group, seed):
    """Documents of up to `longest` tokens, some padding between and behind, groups at their begin or anywhere."""
    rng, docs, groups = random.Random(seed), [], []
    for _ in range(B):
        d, g = [], []
        while len(d) < N:
            n = min(rng.randint(1, longest), N - len(d))
            d += [-1 if rng.random() < 0.12 else rng.randint(0, 3) * 7] * n        # numbers come back: other documents
            part = [0] * n
            if group:
                at = rng.choice((0, rng.randrange(n)))
                m = min(rng.randint(0, group), n - at)
                part[at:at + m] = [rng.randint(1, 2)] * m
            g += part
        docs.append(d)
        groups.append(g)
    return docs, groups


def slopes_of(heads):
    return torch.tensor([2.0 ** (-6.0 * (h + 1) / heads) for h in range(heads)], dtype=torch.float32)


CASES = [
    # D, Hq, Hkv, N, B, left, right, sinks, lengths, cap, slopes, longest document, longest group
    (64, 1, 1, 1, 1, None, 0, 0, None, 20.0, True, 0, 0),               # one token
    (64, 2, 1, 130, 1, None, 0, 0, None, 20.0, False, 0, 0),
    (128, 4, 2, 300, 1, 99, 0, 4, None, 5.0, False, 0, 0),              # a small cap, first tokens
    (64, 2, 2, 300, 2, 70, 30, 0, [300, 131], None, True, 0, 0),        # both directions
    (128, 3, 1, 260, 1, None, 0, 3, None, 15.0, True, 0, 0),            # three query heads a key head
    (64, 4, 1, 290, 2, None, 0, 0, None, None, False, 60, 0),           # documents
    (64, 1, 1, 1000, 1, None, 0, 0, None, None, False, 9, 0),           # many short ones
    (128, 2, 1, 385, 1, None, 0, 0, None, 30.0, False, 400, 40),        # and groups
    (64, 2, 1, 300, 2, 50, 0, 0, None, 8.0, True, 200, 120),            # window, documents and groups that pass it
    (64, 2, 2, 290, 3, None, 0, 0, [290, 0, 133], 30.0, True, 150, 20), # lengths cut a document
    (72, 6, 2, 333, 1, None, 0, 0, None, 12.0, True, 100, 100),
    (96, 5, 1, 140, 2, 12, 0, 0, None, None, True, 50, 3),
    (8, 1, 1, 100, 1, 30, 2, 0, None, 2.0, True, 0, 0),
    (128, 4, 1, 1500, 1, 700, 0, 6, None, 25.0, True, 0, 0),
    (128, 2, 2, 1300, 1, None, 0, 0, None, 25.0, False, 900, 300),
]


def problem(case, dtype, size=4.0):
    D, Hq, Hkv, N, B, left, right, sinks, lengths, cap, slopes, longest, group = case
    q, k, v, dy = (make(i, (D, h, N, B), dtype, s) for i, h, s in ((0, Hq, size), (1, Hkv, 1.0), (2, Hkv, 1.0), (3, Hq, 1.0)))
    docs, groups = numbers(N, B, longest, group, N + B) if longest else (None, None)
    return q, k, v, dy, slopes_of(Hq) if slopes else None, docs, groups if group else None


def call(ca, case, q, k, v, slopes, docs, groups, **kw):
    D, Hq, Hkv, N, B, left, right, sinks, lengths, cap = case[:10]
    spans = None if docs is None else ca.token_spans(ints(docs).t(), None if groups is None else ints(groups).t())
    return ca.window_attention(q, k, v, left, right=right, sinks=sinks, lengths=None if lengths is None else ints(lengths), cap=cap,
                               slopes=None if slopes is None else slopes.cuda(), spans=spans, **kw)


@pytest.mark.parametrize("N,B,longest,group", [(1, 1, 1, 1), (5, 3, 2, 2), (1023, 2, 40, 9), (1025, 1, 3000, 500), (4099, 2, 700, 90), (20000, 1, 5000, 1)])
def test_spans(ca, N, B, longest, group):
    docs, groups = numbers(N, B, longest, group, N)
    for g in (groups, None):
        got = ca.token_spans(ints(docs).t(), None if g is None else ints(g).t()).cpu()
        assert got.shape == (4, N, B) and got.dtype == torch.int32
        for b in range(B):
            first, last = list(range(N)), list(range(N))
            for i in range(1, N):
                if docs[b][i] == docs[b][i - 1]:
                    first[i] = first[i - 1]
            by = list(range(N))
            for i in range(1, N):
                if g is not None and docs[b][i] == docs[b][i - 1] and g[b][i] == g[b][i - 1] and g[b][i] > 0:
                    by[i] = by[i - 1]
            until = list(range(N))
            for i in range(N - 2, -1, -1):
                if g is not None and by[i + 1] == by[i] and g[b][i] > 0 and docs[b][i] == docs[b][i + 1]:
                    last[i] = last[i + 1]
                if docs[b][i] == docs[b][i + 1]:
                    until[i] = until[i + 1]
            for i in range(N):
                if docs[b][i] < 0:
                    first[i], by[i], last[i], until[i] = i, i, i - 1, i - 1
            assert got[:, :, b].tolist() == [first, by, last, until]


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace(" ", "") for x in c))
def test_attention_and_gradients(ca, case, dtype):
    q, k, v, dy, slopes, docs, groups = problem(case, dtype)
    lengths, cap = case[8], case[9]
    x = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    y = call(ca, case, *x, slopes, docs, groups)
    got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(y, x, dy.cuda())), y=y)
    want = ref.window(q, k, v, *case[5:8], lengths, cap, slopes, docs, groups, dy)
    for name, (value, bound) in want.items():
        ref.check(got[name], value, bound, name)
    if lengths is not None:
        for b, n in enumerate(lengths):
            assert all(not t[:, :, n:, b].any() for t in got.values())
    if docs is not None:                                                    # padding sees nothing and is seen by nothing
        for b in range(case[4]):
            pad = [i for i, d in enumerate(docs[b]) if d < 0]
            assert all(not t[:, :, pad, b].any() for t in got.values())
    with torch.no_grad():                                                   # the forward without gradients is the same call
        assert torch.equal(call(ca, case, *x, slopes, docs, groups), got["y"])


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize("D,Hq,Hkv,N,B,longest,group", [(64, 4, 4, 1500, 10, 1400, 30), (128, 8, 2, 2100, 4, 2000, 0), (64, 3, 1, 5000, 6, 40, 10)])
def test_batches_that_fill_the_chip(ca, D, Hq, Hkv, N, B, longest, group, dtype):
    """Neighbouring row tiles that share key tiles, the one of an old document, the other of a new one: checked for some of the
    heads and sequences."""
    case = (D, Hq, Hkv, N, B, None, 0, 0, None, 20.0, True, longest, group)
    q, k, v, dy, slopes, docs, groups = problem(case, dtype)
    x = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    y = call(ca, case, *x, slopes, docs, groups)
    got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(y, x, dy.cuda())), y=y)
    G = Hq // Hkv
    for b, g in ((0, 0), (B - 1, Hkv - 1)):
        heads, one = slice(g * G, g * G + G), slice(g, g + 1)
        part = [t[:, h, :, b:b + 1] for t, h in ((q, heads), (k, one), (v, one), (dy, heads))]
        want = ref.window(*part[:3], None, 0, 0, None, 20.0, slopes[heads], docs[b:b + 1], groups and groups[b:b + 1], part[3])
        for name, (value, bound) in want.items():
            ref.check(got[name][:, heads if name in ("y", "dq") else one, :, b:b + 1], value, bound, name)


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize("scale", [0.4, -0.3, 0.0])
def test_scale(ca, dtype, scale):
    case = (64, 4, 2, 200, 1, 60, 10, 0, None, 6.0, True, 0, 0)
    q, k, v, dy, slopes, docs, groups = problem(case, dtype, 1.5)
    x = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    y = call(ca, case, *x, slopes, docs, groups, scale=scale)
    got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(y, x, dy.cuda())), y=y)
    for name, (value, bound) in ref.window(q, k, v, 60, 10, 0, None, 6.0, slopes, None, None, dy, scale).items():
        ref.check(got[name], value, bound, name)


@pytest.mark.parametrize("size,cap", [(0.5, 50.0), (60.0, 10.0), (400.0, 30.0)])
@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
def test_far_from_the_cap_and_far_beyond(ca, dtype, size, cap):
    """Scores that the cap leaves alone, and scores that it holds: all of a row's near +cap or -cap."""
    case = (64, 2, 1, 150, 1, None, 0, 0, None, cap, False, 0, 0)
    q, k, v, dy, slopes, docs, groups = problem(case, dtype, size)
    x = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    y = call(ca, case, *x, slopes, docs, groups)
    got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(y, x, dy.cuda())), y=y)
    for name, (value, bound) in ref.window(q, k, v, None, 0, 0, None, cap, None, None, None, dy).items():
        ref.check(got[name], value, bound, name)


def test_gradients_against_differences(ca):
    case = (16, 2, 1, 40, 1, None, 0, 0, None, 3.0, True, 25, 10)
    q, k, v, dy, slopes, docs, groups = problem(case, torch.float32, 2.0)
    x = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    w = dy.cuda()
    grads = torch.autograd.grad(call(ca, case, *x, slopes, docs, groups), x, w)
    # a step of 2^-7 along a direction; the central difference is off by h^2 / 6 of a third derivative and by the rounding of y
    # (2^-21 of the sum of |y w|, about 500 terms of size one: 3e-4 / h = 0.03 of derivatives of size 20)
    for t, g in zip(x, grads):
        d = torch.randn(t.shape, generator=torch.Generator().manual_seed(9)).cuda()
        h = 2.0 ** -7
        with torch.no_grad():
            ends = []
            for sign in (1, -1):
                moved = [a + sign * h * d if a is t else a for a in x]
                ends.append((call(ca, case, *moved, slopes, docs, groups).double() * w.double()).sum())
        slope = float((ends[0] - ends[1]) / (2 * h))
        assert abs(slope - float((g.double() * d.double()).sum())) < 0.02 * (abs(slope) + 5.0)


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
def test_what_no_token_sees_has_no_effect(ca, dtype):
    """Padding between documents, and what lies behind the length, may hold anything."""
    case = (64, 4, 2, 300, 1, None, 0, 0, [280], 20.0, True, 60, 20)
    q, k, v, dy, slopes, docs, groups = problem(case, dtype)
    docs[0][100:120] = [-1] * 20
    hidden = [i for i in range(300) if docs[0][i] < 0 or i >= 280]

    def run(q, k, v, dy):
        x = [t.cuda().requires_grad_(True) for t in (q, k, v)]
        y = call(ca, case, *x, slopes, docs, groups)
        return [y, *torch.autograd.grad(y, x, dy.cuda())]
    plain = run(q, k, v, dy)
    behind = list(range(280, 300))
    for junk in (math.nan, math.inf, torch.finfo(dtype).min):
        other = [t.clone() for t in (q, k, v, dy)]
        for t in other:
            t[:, :, behind, 0] = junk
        assert all(torch.equal(a, b) for a, b in zip(plain, run(*other)))
    for junk in (3.0, math.nan, math.inf, torch.finfo(dtype).min, torch.finfo(dtype).max):     # in padding too
        other = [t.clone() for t in (q, k, v, dy)]
        for t in other:
            t[:, :, hidden, 0] = junk
        assert all(torch.equal(a, b) for a, b in zip(plain, run(*other))), junk


def test_without_effect_as_without(ca):
    """One document without groups is the causal window (16-bit types divide by another sum, of the rounded weights)."""
    case = (64, 4, 2, 333, 2, 100, 0, 0, None, None, False, 0, 0)
    q, k, v, dy, *_ = problem(case, torch.float32)
    x = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    spans = ca.token_spans(torch.zeros(2, 333, dtype=torch.int32, device="cuda").t())
    y0, y1 = ca.window_attention(*x, 100), ca.window_attention(*x, 100, spans=spans)
    g0, g1 = (torch.autograd.grad(y, x, dy.cuda()) for y in (y0, y1))
    assert torch.equal(y0, y1) and all(torch.equal(a, b) for a, b in zip(g0, g1))


def cache(D, Hkv, page, chunks, dtype, seed=5, holes=True):
    """Pools and a table in random order for (new, total) tokens of each sequence."""
    rng = random.Random(seed)
    need = [-(-total // page) for _, total in chunks]
    pages = sum(need) + 2
    free = list(range(pages))
    rng.shuffle(free)
    width = max(need) + 1
    table = [[free.pop() for _ in range(n)] + [-1] * (width - n) for n in need]
    if holes:
        for row, n in zip(table, need):
            if n > 6:
                row[n // 3] = -1
    starts = [0]
    for new, _ in chunks:
        starts.append(starts[-1] + new)
    return make(seed, (D, page, Hkv, pages), dtype), make(seed + 1, (D, page, Hkv, pages), dtype), table, starts, [t for _, t in chunks]


PAGED = [
    # D, Hq, Hkv, page, (new, total) ..., left, sinks, cap, slopes, prefix
    (64, 4, 2, 16, [(1, 1)], None, 0, 20.0, True, None),
    (128, 8, 2, 16, [(1, 300), (1, 17), (0, 40), (1, 700)], None, 0, 20.0, False, None),
    (64, 6, 2, 32, [(1, 333), (3, 90), (1, 1)], 100, 4, 10.0, True, None),
    (128, 8, 1, 64, [(1, 1000)], None, 0, None, True, None),
    (64, 2, 1, 16, [(40, 40), (17, 60), (1, 90), (33, 33)], None, 0, None, False, [30, 50, 90, 0]),
    (128, 4, 2, 48, [(200, 300), (150, 150), (1, 77)], None, 0, 15.0, True, [250, 150, 3]),
    (64, 4, 1, 64, [(300, 500), (260, 261)], 90, 2, 15.0, False, [420, 10 ** 6]),
    (96, 3, 1, 16, [(130, 400), (5, 5)], 64, 0, None, True, [395, 4]),
    (128, 16, 2, 16, [(8, 200), (7, 150)], None, 0, 25.0, True, [198, 149]),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize("case", PAGED, ids=lambda c: "-".join(str(x).replace(" ", "") for x in c))
def test_over_a_cache(ca, case, dtype):
    D, Hq, Hkv, page, chunks, left, sinks, cap, slopes, prefix = case
    kp, vp, table, starts, lengths = cache(D, Hkv, page, chunks, dtype)
    q = make(1, (D, Hq, starts[-1]), dtype, 4.0)
    slopes = slopes_of(Hq) if slopes else None
    got = ca.paged_window_attention(q.cuda(), kp.cuda(), vp.cuda(), ints(table).t(), ints(starts), ints(lengths), left, sinks=sinks, cap=cap,
                                    slopes=None if slopes is None else slopes.cuda(), prefix=None if prefix is None else ints(prefix))
    ref.check(got, *ref.paged(q, kp, vp, table, starts, lengths, left, sinks, cap, slopes, prefix))


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
def test_a_model_is_served_as_it_is_trained(ca, dtype):
    """A prompt with a prefix in one call, then chunks and single tokens over a cache: the results of the dense call."""
    D, Hq, Hkv, N, page, prefix = 64, 4, 2, 230, 16, 70
    q, k, v = (make(i, (D, h, N, 1), dtype, s).cuda() for i, h, s in ((0, Hq, 4.0), (1, Hkv, 1.0), (2, Hkv, 1.0)))
    slopes = slopes_of(Hq).cuda()
    groups = (torch.arange(N) < prefix).int().cuda()
    spans = ca.token_spans(torch.zeros(N, dtype=torch.int32, device="cuda"), groups)
    with torch.no_grad():
        whole = ca.window_attention(q, k, v, None, cap=20.0, slopes=slopes, spans=spans)
    table = ints([list(range(N // page + 1))]).t()
    kp, vp = (torch.zeros(N // page + 1, Hkv, page, D, dtype=dtype, device="cuda").permute(3, 2, 1, 0) for _ in range(2))
    turns, at = ca.rotary_turns(D // 2), 0
    want, bound = whole.double().cpu(), None
    u = ref.UNIT[dtype] + 2e-5
    mean = (v.abs().amax()).item()
    for n in [90, 33, 1, 1, 64, 1, 17, 1, 22]:
        piece = [t[:, :, at:at + n, 0] for t in (q, k, v)]
        where = (table, ints([0, n]), ints([at + n]))
        ca.rotary_append_(*piece, kp, vp, *where, torch.zeros(1, n, dtype=torch.int32, device="cuda"), turns)     # position 0: not turned
        y = ca.paged_window_attention(piece[0], kp, vp, *where, cap=20.0, slopes=slopes, prefix=ints([prefix]))
        # two roundings of weights and one of the result on each side
        off = (y.double().cpu() - want[:, :, at:at + n, 0]).abs().max()
        assert off <= 4 * u * mean, (at, n, float(off))
        at += n
    assert at == N


def test_other_streams_and_graphs(ca):
    """Replayed on other inputs, and on a stream of its own: the same as an eager call."""
    case = (64, 4, 2, 300, 2, None, 0, 0, None, 20.0, True, 120, 30)
    q, k, v, dy, slopes, docs, groups = problem(case, torch.bfloat16)
    x = [t.cuda() for t in (q, k, v)]
    d, g, sl = ints(docs).t(), ints(groups).t(), slopes.cuda()

    def step():
        return ca.window_attention(*x, None, cap=20.0, slopes=sl, spans=ca.token_spans(d, g))
    with torch.no_grad():
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            first = step()
        torch.cuda.current_stream().wait_stream(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graph.replay()
        assert torch.equal(out, first)
        docs2, groups2 = numbers(300, 2, 50, 9, 77)
        d.copy_(ints(docs2).t())
        g.copy_(ints(groups2).t())
        x[0].mul_(0.5)
        graph.replay()
        assert torch.equal(out, step()) and not torch.equal(out, first)


def test_refusals(ca):
    q, k = (torch.zeros(1, 50, h, 64, device="cuda").permute(3, 2, 1, 0) for h in (4, 2))
    spans = ca.token_spans(torch.zeros(50, dtype=torch.int32, device="cuda"))
    slopes = torch.ones(4, device="cuda")
    with pytest.raises(AssertionError, match="cap .* must be positive"):
        ca.window_attention(q, k, k, 5, cap=0.0)
    with pytest.raises(AssertionError, match="cap .* must be positive"):
        ca.window_attention(q, k, k, 5, cap=math.nan)
    with pytest.raises(ca.CircAttError, match="cap must be positive"):
        ca.window_attention(q, k, k, 5, cap=math.inf)
    with pytest.raises(AssertionError, match="one for each of the 4 query heads"):
        ca.window_attention(q, k, k, 5, slopes=slopes[:2])
    with pytest.raises(TypeError, match="slopes must be Float"):
        ca.window_attention(q, k, k, 5, slopes=slopes.half())
    with pytest.raises(NotImplementedError, match="no gradient"):
        ca.window_attention(q, k, k, 5, slopes=slopes.clone().requires_grad_(True))
    with pytest.raises(AssertionError, match="those of token_spans for 50 tokens"):
        ca.window_attention(q, k, k, 5, spans=spans[:, :49])
    with pytest.raises(TypeError, match="spans must be Int"):
        ca.window_attention(q, k, k, 5, spans=spans.long())
    with pytest.raises(ca.CircAttError, match="spans say what a token sees"):
        ca.window_attention(q, k, k, 5, right=1, spans=spans)
    with pytest.raises(ca.CircAttError, match="spans say what a token sees"):
        ca.window_attention(q, k, k, 5, sinks=1, spans=spans)
    with pytest.raises(RuntimeError, match="slopes is on cpu|only CUDA"):
        ca.window_attention(q, k, k, 5, slopes=slopes.cpu())
    with pytest.raises(AssertionError, match="groups of size"):
        ca.token_spans(torch.zeros(50, dtype=torch.int32, device="cuda"), torch.zeros(49, dtype=torch.int32, device="cuda"))
    with pytest.raises(TypeError, match="documents must be Int"):
        ca.token_spans(torch.zeros(50, device="cuda"))
    pool = torch.zeros(4, 2, 16, 64, device="cuda").permute(3, 2, 1, 0)
    with pytest.raises(AssertionError, match="one for each sequence"):
        ca.paged_window_attention(q[..., 0], pool, pool, ints([[0, 1, 2, 3]]).t(), ints([0, 50]), ints([50]), prefix=ints([1, 2]))


def test_empty(ca):
    q = torch.zeros(1, 0, 2, 64, device="cuda").permute(3, 2, 1, 0)
    assert ca.token_spans(torch.zeros(0, 1, dtype=torch.int32, device="cuda")).shape == (4, 0, 1)
    assert ca.window_attention(q, q, q, None, cap=3.0, spans=ca.token_spans(torch.zeros(0, 1, dtype=torch.int32, device="cuda"))).shape == (64, 2, 0, 1)
