"""Attention of chunks of new tokens over a paged cache, rotary positions, and the two chained with the cache write:
against the formulas in 64 bits (tests/tokens_reference.py)."""
import math
import random

import pytest
import torch

from tests import tokens_reference as ref

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(seed, shape, dtype, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    t = torch.randn(tuple(reversed(shape)), generator=g, dtype=torch.float64) * scale
    return t.to(dtype).permute(tuple(range(len(shape) - 1, -1, -1)))


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def cache(D, Hkv, page, chunks, dtype, left, sinks, seed=0, junk=math.nan):
    """Pools whose every slot that no query sees holds `junk`, and a table whose every page behind the window is -1 or some
    page number."""
    rng = random.Random(seed)
    width = max([-(-total // page) for _, total in chunks] + [1]) + 1
    count = sum(-(-total // page) for _, total in chunks) + 2
    free = list(range(count))
    rng.shuffle(free)
    pools = [make(seed + i, (D, page, Hkv, count), dtype) for i in range(2)]
    seen = torch.zeros(page, count, dtype=torch.bool)
    table = []
    for new, total in chunks:
        row = []
        first = 0 if left is None else max(0, total - new - left)
        for p in range(-(-total // page)):
            slots = [j for j in range(p * page, min(total, p * page + page)) if new and (j >= first or j < sinks)]
            if slots:
                row.append(free.pop())
                for j in slots:
                    seen[j % page, row[-1]] = True
            else:
                row.append(rng.choice((-1, rng.randrange(count), count, 2 ** 31 - 1)))
        table.append(row + [rng.choice((-1, rng.randrange(count))) for _ in range(width - len(row))])
    for pool in pools:
        pool.permute(1, 3, 0, 2)[~seen] = junk
    return pools[0], pools[1], table


def call(ca, q, kp, vp, table, chunks, left, sinks, scale=None):
    starts = [0]
    for new, _ in chunks:
        starts.append(starts[-1] + new)
    lengths = [total for _, total in chunks]
    y = ca.paged_window_attention(q.cuda(), kp.cuda(), vp.cuda(), ints(table).t(), ints(starts), ints(lengths), left, sinks=sinks, scale=scale)
    want, bound = ref.paged(q.double(), kp.double(), vp.double(), table, starts, lengths, left, sinks, scale, ref.UNIT[q.dtype])
    ref.check(y, want, bound, "y")
    return y


CASES = [
    # D, Hq, Hkv, page, left, sinks, [(new tokens, tokens with them)]
    (64, 1, 1, 16, None, 0, [(1, 1)]),                                          # the very first token
    (64, 4, 1, 16, None, 0, [(1, 15), (1, 16), (1, 17), (1, 128), (1, 129)]),
    (128, 8, 2, 32, 100, 0, [(1, 500), (1, 90), (1, 101), (1, 102)]),
    (128, 8, 1, 16, 63, 4, [(1, 700), (1, 3), (1, 69), (1, 200)]),
    (128, 4, 4, 48, 200, 1, [(1, 1000), (1, 479)]),                             # pages that end inside a tile
    (64, 6, 2, 256, None, 0, [(1, 5000), (1, 4999), (1, 1)]),                   # split over a long axis
    (128, 2, 2, 64, 2000, 130, [(1, 6000)]),
    (64, 4, 2, 16, None, 0, [(0, 0), (1, 40), (0, 33), (7, 7), (0, 0)]),        # sequences without new tokens
    (64, 4, 2, 16, 40, 2, [(130, 130), (1, 300), (65, 400), (2, 2), (33, 90)]),
    (128, 3, 1, 64, 128, 4, [(200, 1000), (129, 129), (1, 513)]),               # three query heads a key head
    (128, 16, 2, 128, 300, 4, [(300, 900), (5, 2000)]),
    (96, 5, 1, 16, 77, 3, [(50, 333), (1, 90)]),
    (72, 2, 1, 80, None, 0, [(64, 500)]),
    (8, 1, 1, 16, 20, 1, [(10, 100)]),
    (64, 2, 1, 16, 0, 0, [(40, 100), (1, 50)]),                                 # each token sees itself only
    (64, 2, 1, 16, 10, 500, [(40, 300)]),                                       # more first tokens than tokens
    (128, 64, 1, 32, 90, 4, [(1, 300), (3, 100)]),                              # 64 query heads a key head
]


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace(" ", "") for x in c))
def test_paged_attention(ca, case, dtype):
    D, Hq, Hkv, page, left, sinks, chunks = case
    q = make(9, (D, Hq, sum(new for new, _ in chunks)), dtype, 1.5)
    kp, vp, table = cache(D, Hkv, page, chunks, dtype, left, sinks)
    y = call(ca, q, kp, vp, table, chunks, left, sinks)
    assert torch.equal(y, call(ca, q, kp, vp, table, chunks, left, sinks))
    ca.ops.check_status()


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize("new", [1, 70])
def test_many_sequences(ca, dtype, new):
    rng = random.Random(3)
    chunks = [(rng.choice((0, new, 1)), 0) for _ in range(70)]
    chunks = [(n, n + rng.randrange(0, 300)) for n, _ in chunks]
    q = make(9, (64, 2, sum(n for n, _ in chunks)), dtype, 1.5)
    kp, vp, table = cache(64, 1, 16, chunks, dtype, 100, 2)
    call(ca, q, kp, vp, table, chunks, 100, 2)


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
def test_missing_pages_and_impossible_lengths(ca, dtype):
    """Missing pages inside the window are skipped; a row that sees nothing at all gives zeros, also where more tokens are
    new than the cache is said to hold."""
    chunks = [(1, 100), (1, 40), (60, 200), (5, 3)]
    q = make(9, (64, 4, 67), dtype, 1.5)
    kp, vp, table = cache(64, 2, 16, chunks, dtype, None, 0)
    table[0][2] = -1
    table[1] = [-1] * len(table[1])
    table[2][3] = table[2][12] = 10 ** 6
    y = call(ca, q, kp, vp, table, chunks, None, 0)
    assert not y[:, :, 1].any() and not y[:, :, 62:64].any() and y[:, :, 64:].any()


@pytest.mark.parametrize("new", [1, 150])
@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
def test_lengths_beyond_the_table(ca, dtype, new):
    """Tokens for which the table has no place count as missing pages: the rows still see what there is, also where a length
    is absurd, and where the window holds nothing that exists."""
    chunks = [(new, 200), (new, 160)]
    q = make(9, (64, 4, 3 * new), dtype, 1.5)
    kp, vp, table = cache(64, 2, 16, chunks, dtype, None, 0, junk=0.25)
    table = [row[:7] for row in table] + [[0] * 7]                     # places for 112 tokens each
    starts, lengths = [0, new, 2 * new, 3 * new], [200, 160, 2 ** 31 - 1]
    for left, sinks in ((None, 0), (60, 20)):
        y = ca.paged_window_attention(q.cuda(), kp.cuda(), vp.cuda(), ints(table).t(), ints(starts), ints(lengths), left, sinks=sinks)
        for s in (0, 1):
            cut = slice(starts[s], starts[s + 1])
            want, bound = ref.paged(q[:, :, cut].double(), kp.double(), vp.double(), [table[s]], [0, new], [lengths[s]], left, sinks, u=ref.UNIT[dtype])
            ref.check(y[:, :, cut], want, bound)
        assert torch.isfinite(y).all() and (left is None or sinks or not y[:, :, 2 * new:].any())
    ca.ops.check_status()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=lambda d: str(d)[6:])
def test_offsets_beyond_32_bits(ca, dtype):
    """A cache of more than 2^32 elements: the pages in use are its last ones."""
    D, Hkv, page = 128, 2, 64
    count = (2 ** 32) // (D * Hkv * page) + 40
    if torch.cuda.mem_get_info()[0] < 2.5 * count * D * Hkv * page * dtype.itemsize:
        pytest.skip("not enough device memory")
    kp, vp = (torch.empty(count, Hkv, page, D, dtype=dtype, device="cuda").permute(3, 2, 1, 0) for _ in range(2))
    small = [make(i, (D, page, Hkv, 8), dtype) for i in range(2)]
    kp[..., -8:], vp[..., -8:] = small[0].cuda(), small[1].cuda()
    for chunks in ([(1, 500)], [(140, 500)]):
        q = make(9, (D, 4, chunks[0][0]), dtype, 1.5)
        y = ca.paged_window_attention(q.cuda(), kp, vp, ints([list(range(count - 8, count))]).t(), ints([0, chunks[0][0]]), ints([500]))
        want, bound = ref.paged(q.double(), small[0].double(), small[1].double(), [list(range(8))], [0, chunks[0][0]], [500], None, 0, u=ref.UNIT[dtype])
        ref.check(y, want, bound)
    k, v = make(20, (D, Hkv, 3), dtype), make(21, (D, Hkv, 3), dtype)
    turns = ca.rotary_turns(64)
    pos = torch.zeros(1, 3, dtype=torch.int32, device="cuda")
    ca.rotary_append_(q[:, :, :3].cuda(), k.cuda(), v.cuda(), kp, vp, ints([list(range(count - 8, count))]).t(), ints([0, 3]), ints([512]), pos, turns)
    assert torch.equal(vp[:, -3:, :, -1].cpu(), v.permute(0, 2, 1)) and torch.equal(kp[:, -3:, :, -1].cpu(), k.permute(0, 2, 1))


def test_cache_views(ca):
    """k and v as two halves of one pool, and a cache whose heads lie inside its tokens."""
    D, Hkv, page, chunks = 64, 2, 16, [(3, 50), (1, 20)]
    q = make(9, (D, 4, 4), torch.bfloat16, 1.5)
    kp, vp, table = cache(D, Hkv, page, chunks, torch.bfloat16, None, 0, junk=1.0)
    base = call(ca, q, kp, vp, table, chunks, None, 0)
    count = kp.shape[3]
    both = torch.empty(count, 2, Hkv, page, D, dtype=torch.bfloat16, device="cuda")
    both[:, 0], both[:, 1] = kp.permute(3, 2, 1, 0).cuda(), vp.permute(3, 2, 1, 0).cuda()
    args = (ints(table).t(), ints([0, 3, 4]), ints([50, 20]))
    assert torch.equal(base, ca.paged_window_attention(q.cuda(), both[:, 0].permute(3, 2, 1, 0), both[:, 1].permute(3, 2, 1, 0), *args))
    inner = [t.permute(3, 1, 2, 0).contiguous().permute(3, 1, 2, 0).cuda() for t in (kp, vp)]
    inner = [t.cuda().permute(3, 1, 2, 0).contiguous().permute(3, 1, 2, 0) for t in (kp, vp)]
    assert torch.equal(base, ca.paged_window_attention(q.cuda(), *inner, *args))
    wide = torch.empty(8, 4, 2 * D, dtype=torch.bfloat16, device="cuda")[:4, :, :D].permute(2, 1, 0)   # q: a slice
    wide.copy_(q)
    assert torch.equal(base, ca.paged_window_attention(wide, kp.cuda(), vp.cuda(), *args))


# ------------------------------------------------------------------------------------------------ rotary positions
def freqs(pairs, base=10000.0):
    return [base ** (-p / pairs) for p in range(pairs)]


ROTARY = [
    # D, heads, second heads, N, B, pairs, sections
    (64, 4, 2, 100, 2, 32, (32,)),
    (128, 8, 1, 33, 1, 64, (16, 24, 24)),
    (64, 1, None, 1, 1, 32, (12, 20)),
    (80, 3, 3, 50, 3, 40, (16, 12, 12)),
    (96, 2, 1, 20, 1, 24, (24,)),                  # half of the features pass
    (80, 2, 1, 20, 2, 20, (4, 8, 8)),              # 8-byte pieces
    (72, 2, 1, 20, 1, 35, (0, 35)),                # single elements, an axis without pairs
    (8, 1, 1, 5, 1, 1, (1,)),
    (256, 1, None, 17, 1, 128, (32, 32, 32, 32)),
    (512, 2, None, 3, 1, 255, (255,)),
]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize("case", ROTARY, ids=lambda c: "-".join(str(x).replace(" ", "") for x in c))
def test_rotary_and_gradient(ca, case, dtype, interleaved):
    D, h1, h2, N, B, pairs, sections = case
    g = torch.Generator().manual_seed(4)
    pos = torch.randint(0, 200000, (len(sections), N, B), generator=g, dtype=torch.int32)
    pos[:, 0] = torch.tensor([0, 1, 2 ** 31 - 1][:B], dtype=torch.int32)
    if N > 2:
        pos[:, 1], pos[:, 2] = -7, -2 ** 31
    xs = [make(i, (D, h, N, B), dtype) for i, h in enumerate((h1, h2)) if h]
    dys = [make(10 + i, x.shape, dtype) for i, x in enumerate(xs)]
    turns = ca.rotary_turns(pairs)
    dev = [x.cuda().requires_grad_(True) for x in xs]
    out = ca.rotary(tuple(dev) if h2 else dev[0], pos.cuda(), turns, sections=sections, interleaved=interleaved)
    out = out if h2 else (out,)
    grads = torch.autograd.grad(out, dev, [d.cuda() for d in dys])
    f = freqs(pairs)
    u = ref.UNIT[dtype]
    for inputs, got, inverse in ((xs, out, False), (dys, grads, True)):
        for x, y in zip(inputs, got):
            want = ref.rotary(x.double(), pos[:, :, :].double()[:, :, :], f, sections, interleaved, inverse)
            size = ref.rotary(x.double().abs(), pos.double() * 0, f, sections, interleaved) * 0
            i = torch.arange(2 * pairs)
            other = (i ^ 1) if interleaved else (i + pairs) % (2 * pairs)
            size[:2 * pairs] = x.double().abs()[:2 * pairs] + x.double().abs()[other]
            # a phase rounded to 2^-24 half turns, sincospi's and the products' last bits; 64-bit angles of 2^31 * 1 rad
            # are themselves off by 2^-22
            ref.check(y, want, u * want.abs() + 2.0 ** -20 * size, "rotary")
            assert torch.equal(y[2 * pairs:].cpu(), x[2 * pairs:])


def test_rotary_forms(ca):
    """Packed tokens, positions shared by the batch, strided inputs, one of two gradients, own ladders per axis."""
    turns = ca.rotary_turns(32)
    x = make(0, (64, 4, 10, 3), torch.bfloat16).cuda()
    pos = torch.randint(0, 5000, (2, 10), dtype=torch.int32, device="cuda")
    full = pos[:, :, None].expand(2, 10, 3)
    base = ca.rotary(x, full.contiguous(), turns, sections=(10, 22))
    assert torch.equal(base, ca.rotary(x, pos, turns, sections=(10, 22)))
    assert torch.equal(base, ca.rotary(x, full, turns, sections=(10, 22)))
    assert torch.equal(base[..., 1], ca.rotary(x[..., 1], pos, turns, sections=(10, 22)))
    assert torch.equal(base, ca.rotary(x.contiguous(), pos.t().contiguous().t(), turns, sections=(10, 22)))
    k = x[:, :1].clone().requires_grad_(True)
    a, b = ca.rotary((x, k), pos, turns, sections=(10, 22))
    assert torch.equal(b, base[:, :1]) and torch.equal(a, base)
    (g,) = torch.autograd.grad(b, (k,), b)
    assert torch.allclose(g.float(), k.detach().float(), atol=2 ** -6)
    own = ca.rotary_turns(32, sections=(10, 22))
    assert own[0] == own[10] == turns[0] and len(own) == 32
    assert ca.rotary(x[:, :, :0], pos[:, :0], turns, sections=(10, 22)).shape == (64, 4, 0, 3)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize("D,pairs,page,chunks", [
    (64, 32, 16, [(1, 1), (1, 16), (1, 17), (0, 5), (1, 40)]),
    (128, 64, 48, [(70, 90), (1, 300), (49, 49)]),
    (80, 20, 32, [(3, 2), (5, 33)]),                # two tokens more than the cache is said to hold: the first is dropped
])
def test_rotary_append(ca, D, pairs, page, chunks, dtype, interleaved):
    Hq, Hkv = 4, 2
    T = sum(n for n, _ in chunks)
    q, k, v = make(0, (D, Hq, T), dtype).cuda(), make(1, (D, Hkv, T), dtype).cuda(), make(2, (D, Hkv, T), dtype).cuda()
    kp, vp, table = cache(D, Hkv, page, [(total, total) for _, total in chunks], dtype, None, 0, junk=0.5)
    kp, vp = kp.cuda(), vp.cuda()
    table[-1][0] = -1 if chunks[-1][1] - chunks[-1][0] < page else table[-1][0]      # a page that is gone
    want_k, want_v = kp.clone(), vp.clone()
    starts = [0]
    for n, _ in chunks:
        starts.append(starts[-1] + n)
    pos = torch.randint(0, 9000, (1, T), dtype=torch.int32, device="cuda")
    turns = ca.rotary_turns(pairs)
    got = ca.rotary_append_(q, k, v, kp, vp, ints(table).t(), ints(starts), ints([t for _, t in chunks]), pos, turns, interleaved=interleaved)
    turned_q, turned_k = ca.rotary((q, k), pos, turns, interleaved=interleaved)
    assert torch.equal(got, turned_q)
    for s, (new, total) in enumerate(chunks):
        for i in range(new):
            j = total - new + i
            if j >= 0 and 0 <= table[s][j // page] < kp.shape[3]:
                want_k[:, j % page, :, table[s][j // page]] = turned_k[:, :, starts[s] + i]
                want_v[:, j % page, :, table[s][j // page]] = v[:, :, starts[s] + i]
    assert torch.equal(kp, want_k) and torch.equal(vp, want_v)


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
def test_serving_agrees_with_training(ca, dtype):
    """A sequence in one call, and the same sequence from the cache in chunks of unequal size."""
    D, Hq, Hkv, N, page, left, sinks = 64, 4, 2, 300, 16, 70, 3
    q, k, v = (make(i, (D, h, N, 1), dtype).cuda() for i, h in enumerate((Hq, Hkv, Hkv)))
    pos = torch.arange(N, dtype=torch.int32, device="cuda")[None]
    turns = ca.rotary_turns(D // 2)
    y = ca.window_attention(*ca.rotary((q, k), pos, turns), v, left, sinks=sinks)
    kp, vp = (torch.full((25, Hkv, page, D), math.nan, dtype=dtype, device="cuda").permute(3, 2, 1, 0) for _ in range(2))
    table = ints([random.Random(0).sample(range(25), 20)]).t()
    at, parts = 0, []
    for n in (1, 1, 130, 7, 1, 100, 60):
        x = [t[:, :, at:at + n, 0] for t in (q, k, v)]
        where = (table, ints([0, n]), ints([at + n]))
        turned = ca.rotary_append_(*x, kp, vp, *where, pos[:, at:at + n], turns)
        parts.append(ca.paged_window_attention(turned, kp, vp, *where, left, sinks=sinks))
        at += n
    got = torch.cat(parts, 2)
    # both are within the same distance of the exact result; twice that between them
    kk, qq = ca.rotary((k, q), pos, turns)
    want = ref.window(*(t.double().cpu() for t in (qq, kk, v)), left, 0, sinks, None, u=ref.UNIT[dtype])["y"]
    ref.check(got[..., None], want[0], want[1])
    ref.check(y, want[0], want[1])


def test_refusals(ca):
    q = torch.zeros(64, 4, 10, device="cuda")
    pool = torch.zeros(7, 2, 16, 64, device="cuda").permute(3, 2, 1, 0)
    table, starts, lengths = ints([[0, 1], [2, 3]]).t(), ints([0, 4, 10]), ints([4, 6])
    at = ca.paged_window_attention
    at(q, pool, pool, table, starts, lengths)
    with pytest.raises(RuntimeError, match="only CUDA compatible"):
        at(q.cpu(), pool, pool, table, starts, lengths)
    with pytest.raises(TypeError, match="k_pages is Half"):
        at(q, pool.half(), pool.half(), table, starts, lengths)
    with pytest.raises(AssertionError, match=r"\(D, heads, T\) expected"):
        at(q[..., None], pool, pool, table, starts, lengths)
    with pytest.raises(AssertionError, match="differ in size"):
        at(q, pool, pool[..., :6], table, starts, lengths)
    with pytest.raises(AssertionError, match="features must be contiguous"):
        at(q, pool.contiguous(), pool.contiguous(), table, starts, lengths)
    with pytest.raises(AssertionError, match=r"\(width, S\), \(S \+ 1\) and \(S\) expected"):
        at(q, pool, pool, table, starts[:2], lengths)
    with pytest.raises(TypeError, match="table must be Int"):
        at(q, pool, pool, table.long(), starts, lengths)
    with pytest.raises(ca.CircAttError, match="multiples of 16 tokens"):
        at(q, pool[:, :8], pool[:, :8], table, starts, lengths)
    with pytest.raises(ca.CircAttError, match="positive multiple"):
        at(q[:, :3], pool, pool, table, starts, lengths)
    x = torch.zeros(64, 4, 10, 2, device="cuda")
    pos, turns = torch.zeros(2, 10, dtype=torch.int32, device="cuda"), ca.rotary_turns(32)
    with pytest.raises(AssertionError, match="2 axes, but 1 sections"):
        ca.rotary(x, pos, turns)
    with pytest.raises(ca.CircAttError, match="sections hold 31 pairs"):
        ca.rotary(x, pos, turns, sections=(10, 21))
    with pytest.raises(ca.CircAttError, match="do not fit"):
        ca.rotary(x, pos[:1], ca.rotary_turns(40))
    with pytest.raises(TypeError, match="positions must be Int"):
        ca.rotary(x, pos.long(), turns, sections=(10, 22))
    with pytest.raises(TypeError, match="turns must be Long"):
        ca.rotary(x, pos, turns.int(), sections=(10, 22))
    with pytest.raises(AssertionError, match="do not fit"):
        ca.rotary(x, pos[:, :9], turns, sections=(10, 22))
    with pytest.raises(AssertionError, match="more than their heads"):
        ca.rotary((x, x[:, :, :5]), pos, turns, sections=(10, 22))
    with pytest.raises(TypeError, match="one tensor or two"):
        ca.rotary((x, x, x), pos, turns, sections=(10, 22))
    with pytest.raises(AssertionError, match="a cache of 2 heads, but k has 4"):
        ca.rotary_append_(q, q, q, pool, pool, table, starts, lengths, pos, turns, sections=(10, 22))
