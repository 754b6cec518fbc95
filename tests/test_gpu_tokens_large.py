"""Attention and rotary positions on token sequences at sizes that fill the chip, where kernels take two row tiles, or several
tokens, at a time; and the scale, which small and large calls apply in different places."""
import math
import random

import pytest
import torch

from tests import tokens_reference as ref
from tests.test_gpu_tokens_paged import cache, call, ints
from tests.test_gpu_tokens_window import DTYPES, compare, make, problem, run

pytestmark = pytest.mark.gpu


def name_of(dtype):
    return str(dtype)[6:]


def sm_count():
    return torch.cuda.get_device_properties(0).multi_processor_count


WINDOW = [
    # D, Hq, Hkv, N, B, left, right, sinks, lengths
    (64, 16, 16, 300, 5, 40, 0, 4, None),
    (128, 16, 16, 300, 5, None, 0, 0, [300, 0, 1, 257, 129]),
    (64, 24, 8, 300, 5, 63, 5, 130, None),                       # three query heads a key head: rows copied by threads
    (128, 24, 6, 300, 5, 100, 0, 0, [300, 171, 64, 0, 299]),
    (72, 32, 16, 260, 5, 0, 0, 2, None),
    (128, 16, 16, 385, 5, 200, 20, 4, None),                     # the last row tile of two has one row
    (64, 10, 10, 1100, 4, 127, 127, 0, None),
    (128, 8, 8, 1500, 4, 300, 0, 200, None),                     # first tokens, then a gap, then the window
]


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
@pytest.mark.parametrize("case", WINDOW, ids=lambda c: "-".join(str(x).replace(" ", "") for x in c))
def test_window_attention_of_many_rows(ca, case, dtype):
    D, Hq, Hkv, N, B, left, right, sinks, lengths = case
    assert -(-N * Hq // Hkv // 256) * Hkv * B >= sm_count()      # two row tiles a block
    q, k, v, dy = problem(D, Hq, Hkv, N, B, dtype)
    got = run(ca, q, k, v, dy, left, right, sinks, lengths)
    compare(got, q, k, v, dy, left, right, sinks, lengths)
    for b, n in enumerate(lengths or ()):
        assert all(not t[:, :, n:, b].any() for t in got.values())
    again = run(ca, q, k, v, dy, left, right, sinks, lengths)
    assert all(torch.equal(got[n], again[n]) for n in got)


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
@pytest.mark.parametrize("D,Hq,Hkv,S,new,left,sinks,page", [
    (64, 2, 2, 80, 150, None, 0, 16),
    (128, 6, 2, 40, 100, 90, 4, 48),
    (128, 8, 2, 40, 75, 60, 130, 64),
])
def test_paged_attention_of_many_rows(ca, D, Hq, Hkv, S, new, left, sinks, page, dtype):
    """Chunks of unequal size, single tokens and sequences without new ones among them; pages that are missing inside the
    window."""
    rng = random.Random(5)
    news = [rng.choice((new, new + 31, 2 * new, 1 if s % 8 == 3 else new, 0 if s % 16 == 5 else new)) for s in range(S)]
    chunks = [(n, n + rng.randrange(0, 400)) for n in news]
    T, G = sum(news), Hq // Hkv
    assert (T * G // 256 + S) * Hkv >= sm_count() and T * G > 128 * S
    q = make(9, (D, Hq, T), dtype, 1.5)
    kp, vp, table = cache(D, Hkv, page, chunks, dtype, left, sinks)
    for s in range(0, S, 3):
        table[s][rng.randrange(len(table[s]))] = rng.choice((-1, 10 ** 6))
    y = call(ca, q, kp, vp, table, chunks, left, sinks)
    assert torch.equal(y, call(ca, q, kp, vp, table, chunks, left, sinks))


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
@pytest.mark.parametrize("scale", [-0.2, 0.0, 0.05])
@pytest.mark.parametrize("D,Hq,Hkv,N,B", [(64, 2, 2, 200, 2), (128, 6, 2, 200, 1), (64, 16, 16, 300, 5)])
def test_scale(ca, D, Hq, Hkv, N, B, scale, dtype):
    """Negative scales, and zero: every visible key has the same weight, and q and k have no gradient."""
    q, k, v, dy = problem(D, Hq, Hkv, N, B, dtype)
    got = run(ca, q, k, v, dy, 70, 0, 4, None, scale)
    sign = math.copysign(1.0, scale)                             # the bounds want a positive scale: the sign goes to q
    want = ref.window(sign * q.double(), k.double(), v.double(), 70, 0, 4, None, abs(scale), dy.double(), ref.UNIT[dtype])
    for name, (x, e) in want.items():
        ref.check(got[name], sign * x if name == "dq" else x, e, name)


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
@pytest.mark.parametrize("scale", [-0.2, 0.0, 0.05])
@pytest.mark.parametrize("chunks", [[(1, 90), (1, 300)], [(100, 150), (130, 400)]], ids=["few", "many"])
@pytest.mark.parametrize("D,Hq", [(64, 2), (128, 6)])
def test_scale_over_a_cache(ca, D, Hq, chunks, scale, dtype):
    T, sign = sum(n for n, _ in chunks), math.copysign(1.0, scale)
    q = make(9, (D, Hq, T), dtype, 1.5)
    kp, vp, table = cache(D, 2, 16, chunks, dtype, 70, 4)
    starts, lengths = [0, chunks[0][0], T], [t for _, t in chunks]
    y = ca.paged_window_attention(q.cuda(), kp.cuda(), vp.cuda(), ints(table).t(), ints(starts), ints(lengths), 70, sinks=4, scale=scale)
    want, bound = ref.paged(sign * q.double(), kp.double(), vp.double(), table, starts, lengths, 70, 4, abs(scale), ref.UNIT[dtype])
    ref.check(y, want, bound)


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
@pytest.mark.parametrize("D,heads,N,B,sections,interleaved", [
    (64, (3, 1), 2501, 2, (32,), True),
    (80, (5, 2), 3334, 3, (16, 12, 12), False),
    (128, (2, 1), 20001, 1, (16, 24, 24), True),
    (96, (1,), 9999, 2, (24,), False),
    (72, (2, 2), 20001, 1, (0, 35), False),
])
def test_rotary_of_many_tokens(ca, D, heads, N, B, sections, interleaved, dtype):
    """From 4736 tokens on a block takes several; the same bits as from short calls, in which it takes one."""
    assert N * B >= 4736
    g = torch.Generator().manual_seed(4)
    pos = torch.randint(-2 ** 31, 2 ** 31 - 1, (len(sections), N, B), generator=g, dtype=torch.int32).cuda()
    x = tuple(make(i, (D, h, N, B), dtype).cuda() for i, h in enumerate(heads))
    turns = ca.rotary_turns(sum(sections))

    def turn(x, pos):
        y = ca.rotary(x if len(x) == 2 else x[0], pos, turns, sections=sections, interleaved=interleaved)
        return y if len(x) == 2 else (y,)
    whole = turn(x, pos)
    for b in range(B):
        for n in range(0, N, 1777):
            cut = slice(n, min(n + 1777, N))
            for part, y in zip(turn(tuple(t[:, :, cut, b:b + 1] for t in x), pos[:, cut, b:b + 1]), whole):
                assert torch.equal(part, y[:, :, cut, b:b + 1])


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
def test_rotary_append_of_many_tokens(ca, dtype):
    D, Hq, Hkv, page = 64, 3, 2, 48
    rng = random.Random(6)
    chunks = [(n, n + rng.randrange(0, 100)) for n in (rng.choice((0, 1, 1, 700, 33)) for _ in range(60))]
    T = sum(n for n, _ in chunks)
    assert T >= 4736
    q, k, v = (make(i, (D, h, T), dtype).cuda() for i, h in enumerate((Hq, Hkv, Hkv)))
    kp, vp, table = cache(D, Hkv, page, [(t, t) for _, t in chunks], dtype, None, 0, junk=0.5)
    kp, vp = kp.cuda(), vp.cuda()
    want_k, want_v = kp.clone(), vp.clone()
    starts, seq, at = [0], [], []
    for s, (n, total) in enumerate(chunks):
        starts.append(starts[-1] + n)
        seq += [s] * n
        at += range(total - n, total)
    pos = torch.randint(0, 9000, (1, T), dtype=torch.int32, device="cuda")
    turns = ca.rotary_turns(D // 2)
    got = ca.rotary_append_(q, k, v, kp, vp, ints(table).t(), ints(starts), ints([t for _, t in chunks]), pos, turns)
    turned_q, turned_k = ca.rotary((q, k), pos, turns)
    where = torch.tensor([table[s][j // page] for s, j in zip(seq, at)], device="cuda")
    off = torch.tensor(at, device="cuda") % page
    want_k.permute(3, 1, 2, 0)[where, off] = turned_k.permute(2, 1, 0)
    want_v.permute(3, 1, 2, 0)[where, off] = v.permute(2, 1, 0)
    assert torch.equal(got, turned_q) and torch.equal(kp, want_k) and torch.equal(vp, want_v)
