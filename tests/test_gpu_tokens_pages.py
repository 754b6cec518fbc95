"""The pages of a cache: steps, forks and compaction against plain bookkeeping on lists, with states that share pages, run out of
them, hold entries that are no pages; captured; and a run of all of them with the attention over the cache."""
import random

import pytest
import torch

from tests import tokens_form_reference as ref
from tests.test_gpu_tokens_window import make

pytestmark = pytest.mark.gpu


def ints(rows):
    return torch.tensor(rows, dtype=torch.int32, device="cuda")


def columns(rows, width):
    return torch.tensor(rows, dtype=torch.int32, device="cuda").reshape(len(rows), width).t()


class State:
    """Rows of pages, their counts and lengths as lists."""

    def __init__(self, rows, pages, lengths, page):
        self.rows, self.lengths, self.page, self.width = [list(r) for r in rows], list(lengths), page, len(rows[0]) if rows else 0
        self.refs = [0] * pages
        for row in rows:
            for e in row:
                if 0 <= e < pages:
                    self.refs[e] += 1

    def on_device(self):
        return columns(self.rows, self.width), ints(self.refs), ints(self.lengths)

    def is_page(self, e):
        return 0 <= e < len(self.refs)

    def take(self, wanted):
        """The lowest free pages for the places wanted; returns those that got none."""
        free = [p for p, r in enumerate(self.refs) if r <= 0]
        for (s, c), p in zip(wanted, free):
            self.rows[s][c] = p
            self.refs[p] = 1
        return wanted[len(free):]

    def advance(self, starts, left, sinks):
        wanted = []
        for s, row in enumerate(self.rows):
            n = max(self.lengths[s], 0)
            new = starts[s + 1] - starts[s]
            for c in range(self.width):
                tokens = [t for t in range(c * self.page, (c + 1) * self.page) if t < n]
                # a partly filled page is seen as long as the window reaches any of its places: the next token enters it
                stays = bool(tokens) and (left is None or (c + 1) * self.page > n - new - left or tokens[0] < sinks)
                if self.is_page(row[c]) and not stays:
                    self.refs[row[c]] -= 1
                if not self.is_page(row[c]) or not stays:
                    row[c] = -1
                if row[c] < 0 and any(t >= n - new for t in tokens):
                    wanted.append((s, c))
        return len(self.take(wanted))

    def fork(self, parents):
        old, lengths, S = [list(r) for r in self.rows], list(self.lengths), len(self.rows)
        keeper = {}
        for s, p in reversed(list(enumerate(parents))):
            if 0 <= p < S:
                keeper[p] = s
        for p in keeper:
            if parents[p] == p:
                keeper[p] = p
        wanted, source = [], {}
        for s, p in enumerate(parents):
            if p == s:
                continue
            for e in old[s]:
                if self.is_page(e):
                    self.refs[e] -= 1
            self.rows[s] = [-1] * self.width
            self.lengths[s] = lengths[p] if 0 <= p < S else 0
            n = min(max(self.lengths[s], 0), self.width * self.page) if 0 <= p < S else 0
            for c in range(-(-n // self.page)):
                e = old[p][c]
                if not self.is_page(e):
                    continue
                if (c + 1) * self.page <= n or keeper[p] == s:
                    self.rows[s][c] = e
                    self.refs[e] += 1
                else:
                    wanted.append((s, c))
                    source[s, c] = e
        missing = self.take(wanted)
        return len(missing), [(source[w], self.rows[w[0]][w[1]]) for w in wanted if w not in missing]

    def compact(self):
        used = [p for p, r in enumerate(self.refs) if r > 0]
        L = len(used)
        holes = iter([p for p in range(L) if self.refs[p] <= 0])
        to = {p: p if p < L else next(holes) for p in used}
        refs = [0] * len(self.refs)
        for p in used:
            refs[to[p]] = self.refs[p]
        self.refs = refs
        self.rows = [[to.get(e, -1) for e in row] for row in self.rows]
        return L, [(p, to[p]) for p in used if to[p] != p]


def random_state(seed, S, width, pages, page, fill=0.5, shared=0.2, odd=0.05):
    rng = random.Random(seed)
    free = list(range(pages))
    rng.shuffle(free)
    rows, lengths = [], []
    for s in range(S):
        n = rng.choice((0, rng.randint(0, width * page), rng.randint(0, width * page), -3 if rng.random() < 0.1 else width * page))
        row = [-1] * width
        for c in range(min(width, -(-max(n, 0) // page) + rng.randint(0, 1))):
            x = rng.random()
            if x < odd:
                row[c] = rng.choice((-1, -7, pages, pages + 100, 2 ** 31 - 1))
            elif x < odd + shared and s and rows[s - 1][c] >= 0:
                row[c] = rows[s - 1][c]
            elif free and x < odd + shared + fill:
                row[c] = free.pop()
        rows.append(row)
        lengths.append(n)
    return State(rows, pages, lengths, page), rng


def same(got, state):
    table, refs = got
    assert table.shape == (state.width, len(state.rows)) and table.t().tolist() == state.rows
    assert refs.tolist() == state.refs


SIZES = [(1, 1, 1), (1, 3, 8), (5, 4, 40), (33, 7, 100), (64, 200, 3000), (7, 1500, 20000), (1200, 3, 2500), (3, 0, 5), (2, 5, 0), (70, 40, 9)]


@pytest.mark.parametrize("left,sinks", [(None, 0), (0, 0), (37, 4), (100, 33), (10 ** 6, 10 ** 6)])
@pytest.mark.parametrize("S,width,pages", SIZES)
def test_advance(ca, S, width, pages, left, sinks):
    state, rng = random_state(S + width, S, width, pages, 16, fill=0.9)
    lengths, starts = [], [0]
    for n in state.lengths:
        new = rng.choice((0, 1, 1, rng.randint(0, 60)))
        n = max(0, min(n, width * 16)) + new if rng.random() < 0.8 else 0            # beyond the table too
        lengths.append(n)
        starts.append(starts[-1] + (new if n or rng.random() < 0.5 else 0))
    state.lengths = lengths
    table, refs, n = state.on_device()
    before = table.clone(), refs.clone()
    got = ca.advance_pages(table, refs, ints(starts), n, 16, left, sinks)
    assert torch.equal(table, before[0]) and torch.equal(refs, before[1])           # the old state stays
    missing = state.advance(starts, left, sinks)
    same(got[:2], state)
    assert got[2].tolist() == [missing]


def pools_for(pages, page, kinds=((64, 2, torch.int16), (64, 2, torch.int16), (20, 3, torch.int32), (128, 1, torch.uint8))):
    out = []
    for i, (D, heads, dtype) in enumerate(kinds):
        g = torch.Generator(device="cuda").manual_seed(i)
        t = torch.randint(0, 255, (pages, heads, page, D * dtype.itemsize), dtype=torch.uint8, device="cuda", generator=g)
        out.append(t.view(dtype).permute(3, 2, 1, 0))           # whole numbers: any bits, and none that is not a number
    return out


def moved(pools, copies):
    out = [t.clone() for t in pools]
    for t, old in zip(out, pools):
        for a, b in copies:
            t[..., b] = old[..., a]
    return out


@pytest.mark.parametrize("page", [16, 48])
@pytest.mark.parametrize("S,width,pages", SIZES)
def test_fork(ca, S, width, pages, page):
    for seed in range(3):
        state, rng = random_state(seed + S, S, width, pages, page, fill=(0.3, 0.5, 0.95)[seed])
        parents = [rng.choice((s, rng.randrange(S), rng.randrange(S), -1, S, -2 ** 31)) for s in range(S)]
        if seed == 1:
            parents = [s // 4 * 4 for s in range(S)]
        table, refs, n = state.on_device()
        pools = pools_for(pages, page)
        before = [t.clone() for t in (table, refs, n)]
        kept = [t.clone() for t in pools]
        got = ca.fork_pages(pools, table, refs, n, ints(parents))
        assert all(torch.equal(a, b) for a, b in zip(before, (table, refs, n)))
        missing, copies = state.fork(parents)
        same(got[:2], state)
        assert got[2].tolist() == state.lengths and got[3].tolist() == [missing]
        assert all(torch.equal(a, b) for a, b in zip(pools, moved(kept, copies)))


@pytest.mark.parametrize("S,width,pages", SIZES)
def test_compact(ca, S, width, pages):
    for seed in range(3):
        state, _ = random_state(seed + 10 * S, S, width, pages, 16, fill=(0.1, 0.5, 0.95)[seed])
        table, refs, _ = state.on_device()
        pools = pools_for(pages, 16)
        kept = [t.clone() for t in pools]
        got = ca.compact_pages(pools, table, refs)
        live, copies = state.compact()
        same(got[:2], state)
        assert got[2].tolist() == [live]
        assert all(torch.equal(a, b) for a, b in zip(pools, moved(kept, copies)))


def test_many_pools_and_strides(ca):
    """More pools than one launch takes; pools that are slices, with heads or tokens further apart, pages in another order."""
    state, _ = random_state(4, 20, 6, 90, 16)
    whole = torch.randint(0, 255, (45, 90, 3, 16, 128), dtype=torch.uint8, device="cuda")
    pools = [t.permute(3, 2, 1, 0)[:64] for t in whole]                               # half of the features
    pools += [whole[0, :, 1:2].permute(3, 2, 1, 0)[64:], torch.randint(0, 255, (90, 16, 5, 32), dtype=torch.uint8, device="cuda").permute(3, 1, 2, 0)]
    state.fork([s // 5 * 5 for s in range(20)])
    table, refs, n = state.on_device()
    before, kept = whole.clone(), [t.clone() for t in pools]
    ca.compact_pages(pools[:45] + pools[46:], table, refs)
    live, copies = state.compact()
    assert copies
    want = moved(kept, copies)
    assert all(torch.equal(a, b) for a, b in zip(pools[:45] + pools[46:], want[:45] + want[46:]))
    assert torch.equal(whole[..., 64:], before[..., 64:])                             # the other half is not touched


def test_captured_steps(ca):
    """A step in a graph, replayed on the state that it left; on a stream of its own."""
    page, S, width, pages = 16, 6, 20, 100
    state = State([[-1] * width for _ in range(S)], pages, [0] * S, page)
    table, refs, n = state.on_device()
    starts = ints([0] * (S + 1))
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    missing = []

    def step():
        t, r, m = ca.advance_pages(table, refs, starts, n, page, 60, 5)
        table.copy_(t)
        refs.copy_(r)
        return m
    with torch.cuda.graph(graph, stream=stream):
        m = step()
    rng = random.Random(3)
    for _ in range(12):
        new = [rng.choice((0, 1, 30)) for _ in range(S)]
        at = [0]
        for s, k in enumerate(new):
            state.lengths[s] = 0 if rng.random() < 0.1 else state.lengths[s] + k
            at.append(at[-1] + (k if state.lengths[s] else 0))
        n.copy_(ints(state.lengths))
        starts.copy_(ints(at))
        graph.replay()
        missing.append(state.advance(at, 60, 5))
        same((table, refs), state)
        assert m.tolist() == missing[-1:]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=lambda d: str(d)[6:])
def test_serving(ca, dtype):
    """Prompts, answers that fork from them, a beam that takes another's place, a compaction in between: each sequence's attention
    is that of its own tokens."""
    D, Hq, Hkv, page, S, width, pages, left, sinks, cap = 64, 4, 2, 16, 6, 14, 40, 45, 3, 10.0
    g = torch.Generator().manual_seed(0)
    pools = [torch.full((pages, Hkv, page, D), float("nan"), dtype=dtype, device="cuda").permute(3, 2, 1, 0) for _ in range(2)]
    table, refs, lengths = columns([[-1] * width for _ in range(S)], width), ints([0] * pages), ints([0] * S)
    turns, tokens = ca.rotary_turns(D // 2), [[] for _ in range(S)]               # the (k, v) of each sequence's tokens

    def step(new):
        """new[s] tokens for sequence s; checks y of all of them."""
        nonlocal table, refs, lengths
        T = sum(new)
        starts = [0]
        for k in new:
            starts.append(starts[-1] + k)
        q, k, v = (torch.randn(T, h, D, generator=g, dtype=torch.float64).to(dtype) * f for h, f in ((Hq, 3.0), (Hkv, 1.0), (Hkv, 1.0)))
        lengths = lengths + ints(new)
        table, refs, missing = ca.advance_pages(table, refs, ints(starts), lengths, page, left, sinks)
        assert missing.item() == 0
        where = (table, ints(starts), lengths)
        dev = [t.permute(2, 1, 0).cuda() for t in (q, k, v)]
        ca.rotary_append_(*dev, *pools, *where, torch.zeros(1, T, dtype=torch.int32, device="cuda"), turns)     # position 0: not turned
        y = ca.paged_window_attention(dev[0], *pools, *where, left, sinks=sinks, cap=cap)
        for s in range(S):
            a, b = starts[s], starts[s + 1]
            tokens[s] += [(k[t], v[t]) for t in range(a, b)]
            if a == b:
                continue
            K, V = (torch.stack([t[i] for t in tokens[s]]).double() for i in (0, 1))
            n = len(tokens[s])
            i, j = torch.arange(n - (b - a), n), torch.arange(n)
            mask = (j <= i[:, None]) & ((j >= i[:, None] - left) | (j < sinks))
            for h in range(Hq):
                want, bound = ref.attend(q[a:b, h].double(), K[:, h // 2], V[:, h // 2], i, mask, D ** -0.5, cap, 0.0, dtype)["y"]
                ref.check(y[:, h, a:b].permute(1, 0), want, bound, f"sequence {s}")

    def fork(parents):
        nonlocal table, refs, lengths, tokens
        table, refs, lengths, missing = ca.fork_pages(pools, table, refs, lengths, ints(parents))
        tokens = [list(tokens[p]) if p >= 0 else [] for p in parents]
        assert missing.item() == 0

    step([37, 0, 0, 50, 0, 0])
    step([5, 0, 0, 0, 0, 0])
    fork([0, 0, 0, 3, 3, 3])
    for _ in range(20):
        step([1] * S)
    fork([1, 1, 0, -1, 5, 4])                        # 0 and 2 change places with others, 3 ends
    assert lengths.tolist() == [len(t) for t in tokens]
    step([1, 2, 1, 0, 1, 30])
    table, refs, live = ca.compact_pages(pools, table, refs)
    assert live.item() == int((refs > 0).sum()) == len({e for row in table.t().tolist() for e in row if e >= 0})
    assert max(e for row in table.t().tolist() for e in row) < live.item()
    for pool in pools:
        pool[..., live.item():] = float("nan")       # what lies behind is free
    step([1, 2, 1, 17, 1, 1])
    fork([-1] * S)
    assert not refs.any() and (table == -1).all() and not lengths.any()


def test_refusals(ca):
    table, refs, n = columns([[0, 1], [2, -1]], 2), ints([1] * 4), ints([20, 3])
    pool = torch.zeros(4, 2, 16, 64, device="cuda").permute(3, 2, 1, 0)
    starts, parents = ints([0, 1, 2]), ints([0, 0])
    with pytest.raises(ca.CircAttError, match="multiples of 16 tokens"):
        ca.advance_pages(table, refs, starts, n, 8)
    with pytest.raises(ca.CircAttError, match="sinks=-1"):
        ca.advance_pages(table, refs, starts, n, 16, sinks=-1)
    with pytest.raises(AssertionError, match="left"):
        ca.advance_pages(table, refs, starts, n, 16, -2)
    with pytest.raises(AssertionError, match=r"\(S \+ 1\) expected"):
        ca.advance_pages(table, refs, n, n, 16)
    with pytest.raises(TypeError, match="table must be Int"):
        ca.advance_pages(table.long(), refs, starts, n, 16)
    with pytest.raises(AssertionError, match="table column-major"):
        ca.advance_pages(table.t().contiguous(), refs, starts, n, 16)
    with pytest.raises(AssertionError, match="no pools"):
        ca.fork_pages([], table, refs, n, parents)
    with pytest.raises(AssertionError, match="with 4 pages expected"):
        ca.fork_pages([pool[..., :3]], table, refs, n, parents)
    with pytest.raises(AssertionError, match="multiples of 16 bytes"):
        ca.fork_pages([pool[:63]], table, refs, n, parents)
    with pytest.raises(AssertionError, match="multiples of 16 bytes"):
        ca.compact_pages([pool.permute(1, 0, 2, 3)], table, refs)
    with pytest.raises(AssertionError, match="pages of 16 and 8 tokens"):
        ca.compact_pages([pool, pool[:, :8]], table, refs)
    with pytest.raises(ca.CircAttError, match="multiples of 16 tokens"):
        ca.compact_pages([pool[:, :8]], table, refs)
    with pytest.raises(AssertionError, match="parents of size"):
        ca.fork_pages([pool], table, refs, n, starts)
    with pytest.raises(RuntimeError, match="on cpu"):
        ca.compact_pages([pool.cpu()], table, refs)
