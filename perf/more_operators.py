"""Performance cases of attention with other scores and masks (a cap, a bias that falls with distance, documents, prefixes),
dense and over a paged cache, and of the pages of such a cache: taking and freeing, forking, compacting.

A case is a dict of plain values.  `kind` says which operator:

    "window"   attention of a batch; spans of documents and groups are made from their numbers in the same pass; with
               `train` the gradients of q, k, v too
    "paged"    attention of new tokens to a paged cache
    "advance"  the pages of a serving step: those behind the windows go back, new tokens get theirs
    "fork"     sequences continue as copies of others: samples of a prompt, beams, sequences that end
    "compact"  the pages in use move to the lowest numbers

Tensors have the framework's Julia-shaped column-major layout: (D, heads, N, B) of dense ones, (D, heads, T) of the packed
tokens of several sequences, (D, page, heads, pages) of a cache, (width, S) of a page table.  `left` = -1 means that the
window has no left end, `cap` = 0 that scores are not capped, `longest` = 0 that there is one document, `group` = 0 that no
tokens see each other both ways."""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}


# ------------------------------------------------------------------------------------------------ cases
def _named(case, name):
    if name:
        case["name"] = name
    return case


def _window(dtype, D, Hq, Hkv, N, B, left, right, train, cap=0.0, slopes=False, longest=0, group=0, ragged=False, name=None):
    return _named(dict(kind="window", dtype=dtype, D=D, Hq=Hq, Hkv=Hkv, N=N, B=B, left=left, right=right, train=train, cap=cap,
                       slopes=slopes, longest=longest, group=group, ragged=ragged), name)


def _paged(dtype, D, Hq, Hkv, S, chunk, history, page, left, sinks, cap=0.0, slopes=False, prefix=False, name=None):
    return _named(dict(kind="paged", dtype=dtype, D=D, Hq=Hq, Hkv=Hkv, S=S, chunk=chunk, history=history, page=page, left=left,
                       sinks=sinks, cap=cap, slopes=slopes, prefix=prefix), name)


def _advance(S, chunk, history, page, left, sinks, name=None):
    return _named(dict(kind="advance", S=S, chunk=chunk, history=history, page=page, left=left, sinks=sinks), name)


def _fork(dtype, D, Hkv, pools, S, group, history, page, beams, name=None):
    return _named(dict(kind="fork", dtype=dtype, D=D, Hkv=Hkv, pools=pools, S=S, group=group, history=history, page=page,
                       beams=beams), name)


def _compact(dtype, D, Hkv, pools, S, pages, live, page, name=None):
    return _named(dict(kind="compact", dtype=dtype, D=D, Hkv=Hkv, pools=pools, S=S, pages=pages, live=live, page=page), name)


def listed():
    return [
        # A short prompt whose first part sees itself both ways, in evaluation: only latency counts.
        _window("bf16", 64, 4, 1, 300, 1, -1, 0, False, group=120, name="window prefix infer"),
        # A training batch packed with documents of unequal lengths, shared key heads, capped scores.
        _window("bf16", 128, 16, 4, 16384, 1, -1, 0, True, cap=30.0, longest=4096, name="window packed train"),
        # Records of unequal odd lengths, read in both directions, with a bias by distance in place of positions.
        _window("f16", 64, 8, 8, 5001, 3, 127, 127, True, slopes=True, ragged=True, name="window sloped train"),
        # Float32, everything at once: documents with groups (pictures between text), cap and bias.
        _window("f32", 64, 8, 8, 4096, 2, -1, 0, True, cap=30.0, slopes=True, longest=1024, group=100, name="window f32 train"),
        # A full serving batch, one token each, window and first tokens, capped scores.
        _paged("bf16", 128, 32, 8, 64, 1, 30000, 16, 4095, 16, cap=50.0, name="decode capped"),
        # Chunks of prompts whose prefix sees itself both ways, next to single tokens; bias by distance.
        _paged("f16", 128, 16, 2, 12, 900, 2000, 64, -1, 0, slopes=True, prefix=True, name="chunks prefix"),
        # One token for each sequence of a serving batch: few pages change.
        _advance(64, 1, 30000, 16, 4095, 16, name="advance one token"),
        # Chunks of prompts for many sequences, no window: many pages are taken.
        _advance(256, 900, 8000, 16, -1, 0, name="advance prompts"),
        # Beams of a small model's two requests, one new token ago.
        _fork("bf16", 64, 2, 4, 8, 4, 900, 16, True, name="fork beams"),
        # Sixteen answers to each of eight prompts, eight layers.
        _fork("bf16", 128, 8, 16, 128, 16, 2000, 64, False, name="fork samples"),
        # A small cache after a few requests.
        _compact("f16", 64, 2, 4, 8, 300, 0.4, 16, name="compact small"),
        # Half of a large cache's pages in use, four layers.
        _compact("bf16", 128, 8, 8, 64, 2000, 0.5, 64, name="compact large"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the ranges the listed ones stand for."""
    while True:
        kind = rng.choice(("window", "window", "window", "paged", "paged", "advance", "fork", "compact"))
        dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
        D = rng.choice((32, 64, 64, 80, 96, 128, 128))
        Hkv = rng.choice((1, 2, 3, 4, 8))
        Hq = Hkv * rng.choice((1, 1, 2, 3, 4, 8))
        page = rng.choice((16, 16, 32, 48, 64, 128))
        cap, slopes = rng.choice((0.0, 20.0, 30.0, 50.0)), rng.random() < 0.5
        if kind == "advance":
            S = _log_int(rng, 1, 256)
            case = _advance(S, 1 if rng.random() < 0.5 else _log_int(rng, 2, 1500), _log_int(rng, 1, 30000), page,
                            -1 if rng.random() < 0.4 else _log_int(rng, 1, 8000), rng.choice((0, 4, 16, 130)))
            if S * (case["history"] + 2 * case["chunk"]) > 3.3e6:
                continue
            return case
        if kind == "fork":
            group = rng.choice((1, 2, 4, 8, 16))
            case = _fork(dtype, D, Hkv, rng.choice((1, 2, 4, 6, 16)), group * _log_int(rng, 1, 16), group, _log_int(rng, 1, 4000), page,
                         rng.random() < 0.5)
            if case["S"] * (1 + case["history"] / page) * case["pools"] * _page_bytes(case) > 4e9 or work(case)["bytes"] > 1e9:
                continue
            return case
        if kind == "compact":
            case = _compact(dtype, D, Hkv, rng.choice((1, 2, 4, 6, 16)), _log_int(rng, 1, 100), _log_int(rng, 4, 4000),
                            rng.choice((0.1, 0.3, 0.5, 0.7, 0.9, 0.99)), page)
            if case["pages"] * case["pools"] * _page_bytes(case) > 4e9 or work(case)["bytes"] > 1e9:
                continue
            return case
        if kind == "window":
            train = rng.random() < 0.6
            N, B = _log_int(rng, 2 if train else 1, 20000), _log_int(rng, 1, 4)     # the gradients of a single token are zeros
            spans = rng.random() < 0.5
            left = -1 if rng.random() < 0.5 else _log_int(rng, 1, 3000)
            right = 0 if spans or rng.random() < 0.7 else _log_int(rng, 1, 500)
            longest = (_log_int(rng, 32, 4000) if rng.random() < 0.8 else 0) if spans else 0
            group = _log_int(rng, 1, 400) if spans and (not longest or rng.random() < 0.5) else 0
            case = _window(dtype, D, Hq, Hkv, N, B, left, right, train, cap, slopes, longest, group, not spans and rng.random() < 0.4)
            span = sum(_reach(case)) + 256
            if B * Hq * N * span > (6e8 if case["train"] else 1.2e9) or work(case)["flops"] > (1e11 if dtype == "f32" else 4e11):
                continue
            return case
        S = _log_int(rng, 1, 64)
        chunk, history = 1 if rng.random() < 0.5 else _log_int(rng, 2, 1500), _log_int(rng, 1, 30000)
        left = -1 if rng.random() < 0.4 else _log_int(rng, 16, 8000)
        case = _paged(dtype, D, Hq, Hkv, S, chunk, history, page, left, rng.choice((0, 1, 4, 16, 130)), cap, slopes,
                      chunk > 1 and rng.random() < 0.5)
        keys = history + chunk if left < 0 else min(history + chunk, left + 2 * chunk)
        if S * Hq * chunk * keys > 1.2e9 or S * Hkv * keys * D > 1.2e9 or work(case)["flops"] > (1e11 if dtype == "f32" else 4e11):
            continue
        return case


# ------------------------------------------------------------------------------------------------ what a case fixes
def _rng_of(case):
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _spanned(case):
    return bool(case["longest"] or case["group"])


def _lengths(case):
    """Tokens of each sequence of a dense batch: all N, or unequal ones."""
    return [case["N"] - (case["N"] * b) // (2 * case["B"]) if case["ragged"] else case["N"] for b in range(case["B"])]


def _documents(case):
    """For each of the batch the documents' numbers and the groups' numbers of its tokens.  Documents of unequal lengths
    fill the sequence, a short rest is padding (-1); a document begins with a group and has another one in its middle."""
    rng, N, out = _rng_of(case), case["N"], []
    for _ in range(case["B"]):
        documents, groups, number, run = [], [], 0, 0
        while len(documents) < N:
            n = _log_int(rng, max(1, case["longest"] // 16), case["longest"]) if case["longest"] else N
            if len(documents) + n > N:
                n = N - len(documents)
                if case["longest"] and n < case["longest"] // 16:
                    documents += [-1] * n
                    groups += [0] * n
                    break
            part = [0] * n
            if case["group"]:
                for at in (0, n // 2):
                    g = min(rng.randint(0, case["group"]), n // 2)
                    run += 1
                    part[at:at + g] = [run] * g
            documents += [number] * n
            groups += part
            number += 1
        out.append((documents, groups))
    return out


def _runs(documents, groups):
    """First and last token that each token sees, by its document and group; (i, i - 1) of padding."""
    n = len(documents)
    first, last = list(range(n)), list(range(n))
    for i in range(1, n):
        if documents[i] == documents[i - 1] and documents[i] >= 0:
            first[i] = first[i - 1]
    for i in range(n - 2, -1, -1):
        if documents[i] == documents[i + 1] and documents[i] >= 0 and groups[i] > 0 and groups[i] == groups[i + 1]:
            last[i] = last[i + 1]
    for i in range(n):
        if documents[i] < 0:
            last[i] = i - 1
    return first, last


def _reach(case):
    """Tokens back and ahead that any token sees at most."""
    back = case["longest"] or case["N"]
    ahead = case["group"] if _spanned(case) else case["right"]
    return min(case["N"], back if case["left"] < 0 else min(back, case["left"])), min(case["N"], ahead)


def _chunks(case):
    """(new tokens, tokens with them) of each sequence: unequal histories, and among larger chunks some sequences with a
    single token and one with none."""
    rng, out = _rng_of(case), []
    for s in range(case["S"]):
        chunk = case["chunk"]
        new = chunk if chunk == 1 else (1, rng.randint(1, chunk), chunk, rng.randint(1, chunk))[s % 4]
        if chunk > 1 and s == 6:
            new = 0
        out.append((new, new + rng.randint(case["history"] // 2, case["history"])))
    return out


def _prefixes(case):
    """Tokens of each sequence that all of it sees: into the new ones, or short of them."""
    rng = _rng_of(case)
    return [max(0, total - rng.randint(0, max(1, 2 * new))) for new, total in _chunks(case)]


def _page_bytes(case):
    return case["D"] * case["page"] * case["Hkv"] * BYTES[case["dtype"]]


def _parents(case):
    """Which sequence each one continues: every sample the first of its group, or beams at random; a group of beams ends."""
    rng, S, g = _rng_of(case), case["S"], case["group"]
    if not case["beams"]:
        return [s - s % g for s in range(S)]
    parents = [s - s % g + rng.randrange(g) for s in range(S)]
    return [-1] * g + parents[g:] if S > 2 * g else parents


def _fork_lengths(case):
    """Tokens of each sequence before: only the prompts, or all beams of a group the same."""
    rng, S, g = _rng_of(case), case["S"], case["group"]
    per = [rng.randint(max(1, case["history"] // 2), case["history"]) for _ in range(S // g)]
    return [per[s // g] if case["beams"] or s % g == 0 else 0 for s in range(S)]


def _copied(case):
    """Pages that a fork copies in each pool: partly filled ones of parents that several sequences continue."""
    parents, lengths = _parents(case), _fork_lengths(case)
    takers = {}
    for s, p in enumerate(parents):
        if p >= 0 and lengths[p] % case["page"]:
            takers[p] = takers.get(p, 0) + 1
    return sum(n - 1 for n in takers.values())


def _width(case):
    """Places of the page table of a sequence."""
    if case["kind"] == "fork":
        return -(-case["history"] // case["page"]) + 2
    if case["kind"] == "compact":
        return -(-int(2 * case["pages"] * case["live"]) // case["S"]) + 2
    return -(-max(total for _, total in _chunks(case)) // case["page"]) + 1


def work(case):
    """Every input read once, every output written once.  Attention: two operations for each visible pair and feature of
    each contraction: two contractions forward and five backward (the scores are not kept)."""
    kind = case["kind"]
    if kind in ("advance", "fork", "compact"):
        table = _width(case) * case["S"]
        if kind == "advance":
            pages = table                     # about as many pages as places
            return {"bytes": 8 * table + 8 * pages, "flops": 4 * table}
        if kind == "fork":
            return {"bytes": 2 * _copied(case) * case["pools"] * _page_bytes(case) + 8 * table, "flops": 4 * table}
        live = int(case["pages"] * case["live"])
        moved = live * (1 - live / case["pages"])
        return {"bytes": int(2 * moved * case["pools"] * _page_bytes(case)) + 8 * table + 8 * case["pages"], "flops": 4 * table}
    e, D, Hq, Hkv = BYTES[case["dtype"]], case["D"], case["Hq"], case["Hkv"]
    seen, keys = 0, 0
    if kind == "window":
        for b, n in enumerate(_lengths(case)):
            i = torch.arange(n, dtype=torch.float64)
            if _spanned(case):
                first, last = (torch.tensor(x, dtype=torch.float64) for x in _runs(*_documents(case)[b]))
            else:
                first, last = torch.zeros_like(i), (i + case["right"]).clamp(max=n - 1)
            if case["left"] >= 0:
                first = torch.maximum(first, i - case["left"])
            seen += float((last - first + 1).clamp(min=0).sum())
        tokens = case["N"] * case["B"]
        if case["train"]:   # q, k, v, y's cotangent in; y and three gradients out
            return {"bytes": tokens * (4 * Hq + 4 * Hkv) * D * e, "flops": 14 * seen * Hq * D}
        return {"bytes": tokens * (2 * Hq + 2 * Hkv) * D * e, "flops": 4 * seen * Hq * D}
    tokens, prefixes = 0, _prefixes(case) if case["prefix"] else [0] * case["S"]
    for (new, total), prefix in zip(_chunks(case), prefixes):
        i = torch.arange(total - new, total, dtype=torch.float64)
        lo = (i - (total if case["left"] < 0 else case["left"])).clamp(min=0)
        hi = i.clamp(min=min(prefix, total) - 1)
        seen += float((hi - lo + 1 + torch.minimum(lo, torch.tensor(float(case["sinks"])))).sum())
        if new:
            first = _first_visible(case, new, total)
            keys += total - first + min(case["sinks"], first)
        tokens += new
    return {"bytes": (2 * tokens * Hq + 2 * keys * Hkv) * D * e, "flops": 4 * seen * Hq * D}


def _first_visible(case, new, total):
    """First position in the window of the first new token."""
    return 0 if case["left"] < 0 else max(0, total - new - case["left"])


# ------------------------------------------------------------------------------------------------ inputs
class _State:
    pass


def _julia(shape, dtype, gen, scale=1.0):
    """Standard normal Julia-shaped tensor times `scale`."""
    t = torch.randn(tuple(reversed(shape)), dtype=dtype, device="cuda", generator=gen)
    t = t * scale if scale != 1.0 else t
    return t.permute(tuple(range(len(shape) - 1, -1, -1)))


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _columns(rows):
    """List of rows (lists) -> Julia-shaped integer tensor whose column s is rows[s]."""
    return _ints(rows).t()


def _slopes(case):
    """One slope for each query head, a falling geometric row."""
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / case["Hq"]) for h in range(case["Hq"])], dtype=torch.float32, device="cuda")


def prepare(case, seed):
    """Normal tensors; where scores are capped, queries so large that the cap matters (scores of standard deviation 8, the
    largest beyond the cap), else scores as those of trained heads.  Page tables in random order."""
    gen = torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFFFFFF)
    rng = random.Random(int(seed))
    s = _State()
    s.case, s.page = case, case.get("page")
    if case["kind"] in ("window", "paged"):
        dtype, D, Hq, Hkv = DTYPES[case["dtype"]], case["D"], case["Hq"], case["Hkv"]
        size = 8.0 if case["cap"] else 1.5
        s.slopes = _slopes(case) if case["slopes"] else None
        s.cap = case["cap"] or None
    if case["kind"] == "window":
        N, B, grad = case["N"], case["B"], case["train"]
        s.q = _julia((D, Hq, N, B), dtype, gen, size).requires_grad_(grad)
        s.k = _julia((D, Hkv, N, B), dtype, gen).requires_grad_(grad)
        s.v = _julia((D, Hkv, N, B), dtype, gen).requires_grad_(grad)
        s.dy = _julia((D, Hq, N, B), dtype, gen) if grad else None
        s.lengths = _ints(_lengths(case)) if case["ragged"] else None
        s.documents = s.groups = None
        if _spanned(case):
            both = _documents(case)
            s.documents = _columns([d for d, _ in both])
            s.groups = _columns([g for _, g in both]) if case["group"] else None
        return s
    if case["kind"] == "paged":
        chunks, page = _chunks(case), case["page"]
        live = []
        for new, total in chunks:
            first = _first_visible(case, new, total)
            live.append([p * page + page > first or p * page < case["sinks"] for p in range(-(-total // page))])
        count = sum(sum(x) for x in live) + 3
        free = list(range(count))
        rng.shuffle(free)
        width = _width(case)
        s.table = _columns([[free.pop() if on else -1 for on in x] + [-1] * (width - len(x)) for x in live])
        s.lengths = _ints([total for _, total in chunks])
        s.starts = _starts(chunks)
        s.prefix = _ints(_prefixes(case)) if case["prefix"] else None
        s.k_pages, s.v_pages = _julia((D, page, Hkv, count), dtype, gen), _julia((D, page, Hkv, count), dtype, gen)
        s.q = _julia((D, Hq, sum(new for new, _ in chunks)), dtype, gen, size)
        return s
    return _prepare_pages(s, case, gen, rng)


def _starts(chunks):
    starts = [0]
    for new, _ in chunks:
        starts.append(starts[-1] + new)
    return _ints(starts)


def _prepare_pages(s, case, gen, rng):
    S, page, width = case["S"], case["page"], _width(case)
    rows = [[-1] * width for _ in range(S)]
    if case["kind"] == "advance":
        # The step before brought as many tokens; its window's pages are there.  Some sequences are at their end.
        chunks = [(0, 0) if i % 9 == 8 else c for i, c in enumerate(_chunks(case))]
        old = []
        for i, (new, total) in enumerate(_chunks(case)):
            have = total - new
            first = 0 if case["left"] < 0 else max(0, have - new - case["left"])
            old.append([c for c in range(-(-have // page)) if c * page + page > first or c * page < case["sinks"]])
        need = sum(-(-total // page) - (total - new) // page + 1 for new, total in chunks)
        pages = sum(len(x) for x in old) + need
        free = list(range(pages))
        rng.shuffle(free)
        refs = [0] * pages
        for i, x in enumerate(old):
            for c in x:
                shared = i % 2 and c < len(old[i]) // 4 and rows[i - 1][c] >= 0      # pairs share their prompts' pages
                rows[i][c] = rows[i - 1][c] if shared else free.pop()
                refs[rows[i][c]] += 1
        s.lengths, s.starts = _ints([total for _, total in chunks]), _starts(chunks)
    elif case["kind"] == "fork":
        g, lengths = case["group"], _fork_lengths(case)
        pages = sum(-(-n // page) + 1 for n in lengths) + S
        free = list(range(pages))
        rng.shuffle(free)
        refs = [0] * pages
        for i, n in enumerate(lengths):
            for c in range(-(-n // page) + (1 if n else 0)):                          # one page is there in advance
                shared = case["beams"] and i % g and c < n // page // 2               # beams share the prompt's pages
                rows[i][c] = rows[i - i % g][c] if shared else free.pop()
                refs[rows[i][c]] += 1
        s.lengths, s.parents = _ints(lengths), _ints(_parents(case))
    else:
        pages = case["pages"]
        used = rng.sample(range(pages), int(pages * case["live"]))
        refs, at = [0] * pages, 0
        for p in used + [rng.choice(used) for _ in range(len(used) // 4)] if used else []:   # some are shared
            rows[at % S][at // S] = p
            refs[p] += 1
            at += 1
    s.table, s.refs = _columns(rows), _ints(refs)
    if case["kind"] != "advance":
        s.pools = tuple(_julia((case["D"], page, case["Hkv"], pages), DTYPES[case["dtype"]], gen) for _ in range(case["pools"]))
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _formed(scores, distance, cap, slope):
    """cap tanh(score / cap), less slope times distance."""
    if cap:
        scores = cap * torch.tanh(scores / cap)
    return scores if slope is None else scores - slope * distance


def _softmax_times(scores, mask, v):
    """softmax over the visible columns times v; rows that see nothing give zeros."""
    scores = scores.masked_fill(~mask, -math.inf)
    top = scores.amax(-1, keepdim=True).detach()
    p = torch.exp(scores - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    return torch.matmul(p, v) / p.sum(-1, keepdim=True).clamp(min=1e-30)


def _run_numbers(s):
    """Running numbers of the documents and of the groups (0: none) of every token, (B, N)."""
    documents = s.documents.t().long()
    N = documents.shape[1]
    new = torch.ones_like(documents, dtype=torch.bool)
    new[:, 1:] = documents[:, 1:] != documents[:, :-1]
    run = torch.where(documents >= 0, torch.cumsum(new, 1), torch.zeros_like(documents))
    if s.groups is None:
        return run, torch.zeros_like(run)
    groups = s.groups.t().long()
    other = new.clone()
    other[:, 1:] |= groups[:, 1:] != groups[:, :-1]
    return run, torch.where(groups > 0, torch.cumsum(other, 1), torch.zeros_like(groups))


def _window_plain(s):
    """Blocks of queries against the keys from the furthest that the first one sees to the furthest of the last."""
    q, k, v, case = s.q, s.k, s.v, s.case
    D, Hq, N, B = q.shape
    Hkv = k.shape[1]
    G = Hq // Hkv
    back, ahead = _reach(case)
    block = 256
    nb = -(-N // block)
    rest, span, dev = nb * block - N, block + back + ahead, q.device
    pad = torch.nn.functional.pad
    Q = pad(q.permute(3, 1, 2, 0).float(), (0, 0, 0, rest)) / math.sqrt(D)
    Q = Q.reshape(B, Hkv, G, nb, block, D).transpose(2, 3).reshape(B, Hkv, nb, G * block, D)
    keys, values = (pad(t.permute(3, 1, 2, 0).float(), (0, 0, back, ahead + rest)).unfold(2, span, block) for t in (k, v))
    scores = torch.matmul(Q, keys).reshape(B, Hkv, nb, G, block, span)
    i = torch.arange(nb * block, device=dev).reshape(1, nb, block, 1)
    j = torch.arange(nb, device=dev).reshape(1, nb, 1, 1) * block - back + torch.arange(span, device=dev)
    n = torch.full((B, 1, 1, 1), N, device=dev) if s.lengths is None else s.lengths.long().reshape(B, 1, 1, 1)
    mask = (j >= 0) & (j < n) & (i < n)
    if case["left"] >= 0:
        mask = mask & (j >= i - case["left"])
    if s.documents is None:
        mask = mask & (j <= i + case["right"])
    else:
        run, group = _run_numbers(s)
        rows = [pad(t, (0, rest)).reshape(B, nb, block, 1) for t in (run, group)]
        cols = [pad(t, (back, ahead + rest)).unfold(1, span, block).unsqueeze(2) for t in (run, group)]
        mask = mask & (rows[0] == cols[0]) & (rows[0] > 0) & ((j <= i) | ((rows[1] == cols[1]) & (rows[1] > 0)))
    slope = None if s.slopes is None else s.slopes.reshape(1, Hkv, 1, G, 1, 1)
    scores = _formed(scores, (i - j).abs().float().unsqueeze(2).unsqueeze(1), s.cap, slope)
    mask = mask.unsqueeze(2).unsqueeze(1).expand(B, 1, nb, G, block, span).reshape(B, 1, nb, G * block, span)
    y = _softmax_times(scores.reshape(B, Hkv, nb, G * block, span), mask, values.transpose(3, 4))
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
    total, new = s.lengths.long(), (s.starts[1:] - s.starts[:-1]).long()
    t = torch.arange(T, device=dev)
    seq = torch.searchsorted(s.starts.long(), t, right=True) - 1
    row = t - s.starts.long()[seq]
    Q = torch.zeros(S, most, Hq, D, device=dev)
    Q[seq, row] = s.q.permute(2, 1, 0).float() / math.sqrt(D)
    begin = (total - new - left).clamp(min=0)
    near = begin[:, None] + torch.arange(min(longest, left + 2 * most), device=dev)                  # (S, near)
    j = torch.cat([torch.arange(case["sinks"], device=dev).expand(S, -1), near], 1)                  # (S, keys)
    first = torch.arange(j.shape[1], device=dev) < case["sinks"]
    where = s.table.t().long().gather(1, torch.div(j, page, rounding_mode="floor").clamp(max=s.table.shape[0] - 1))
    at = (where.clamp(min=0)[..., None] * Hkv + torch.arange(Hkv, device=dev)) * page + (j % page)[..., None]
    K, V = (x.permute(3, 2, 1, 0).reshape(-1, D)[at.transpose(1, 2)].float() for x in (s.k_pages, s.v_pages))
    Q = Q.reshape(S, most, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(S, Hkv, G * most, D)
    i = (total - new)[:, None, None] + torch.arange(most, device=dev)[None, :, None]                 # (S, most, 1)
    j, total = j[:, None], total[:, None, None]
    ahead = i if s.prefix is None else torch.maximum(i, s.prefix.long()[:, None, None] - 1)
    mask = torch.where(first, j < i - left, j >= i - left) & (j <= ahead) & (j < total)
    scores = torch.matmul(Q, K.transpose(2, 3)).reshape(S, Hkv, G, most, -1)
    slope = None if s.slopes is None else s.slopes.reshape(1, Hkv, G, 1, 1)
    scores = _formed(scores, (i - j).abs().float()[:, None, None], s.cap, slope)
    mask = mask[:, None, None].expand(S, 1, G, most, -1).reshape(S, 1, G * most, -1)
    y = _softmax_times(scores.reshape(S, Hkv, G * most, -1), mask, V)
    y = y.reshape(S, Hkv, G, most, D).permute(0, 3, 1, 2, 4).reshape(S, most, Hq, D)
    return y[seq, row].to(s.q.dtype).permute(2, 1, 0)


def _take(refs, wanted):
    """Gives the places of `wanted` (S, width) the lowest pages without users, sequence by sequence.  Returns the pages
    (S, width; -1 where none is wanted or left), the new counts and how many were wanting."""
    flat = wanted.reshape(-1)
    free = torch.sort((refs > 0).int(), stable=True).indices.int()
    rank = torch.cumsum(flat, 0) - 1
    have = (refs <= 0).sum()
    got = flat & (rank < have)
    pages = torch.where(got, free[rank.clamp(0, refs.numel() - 1)], torch.full_like(rank, -1, dtype=torch.int32))
    number = torch.arange(refs.numel(), device=refs.device)
    taken = torch.minimum(flat.sum(), have)
    refs = refs.clone()
    refs[free.long()] = torch.where(number < taken, torch.ones_like(refs), refs[free.long()])
    return pages.reshape(wanted.shape), refs, (flat.sum() - taken).int().reshape(1)


def _count(refs, table, on, sign):
    """refs plus `sign` for every entry of the table (S, width) where `on`."""
    return refs.index_add(0, torch.where(on, table, torch.zeros_like(table)).reshape(-1).long(), (sign * on.int()).reshape(-1).int())


def _advance_plain(s):
    case, page, pages = s.case, s.page, s.refs.numel()
    table, n = s.table.t(), s.lengths.long()[:, None]
    new = (s.starts[1:] - s.starts[:-1]).long()[:, None]
    at = torch.arange(table.shape[1], device=table.device)[None] * page                # first token of each place
    begin = n - new                                                                     # position of the first new token
    first = torch.zeros_like(begin) if case["left"] < 0 else (begin - case["left"]).clamp(min=0)
    stays = ((at + page > first) & (at < n)) | (at < n.clamp(max=case["sinks"]))
    there = (table >= 0) & (table < pages)
    refs = _count(s.refs, table, there & ~stays, -1)
    kept = torch.where(there & stays, table, torch.full_like(table, -1))
    wanted = (kept < 0) & (new > 0) & (at + page > begin) & (at < n)
    got, refs, missing = _take(refs, wanted)
    return {"table": torch.where(wanted, got, kept).t(), "refs": refs, "missing": missing}


def _move_plain(pools, source, target):
    for pool in pools:
        by_page = pool.permute(3, 2, 1, 0)
        by_page[target] = by_page[source]


def _fork_plain(s):
    page, pages, S = s.page, s.refs.numel(), s.parents.numel()
    table, me = s.table.t(), torch.arange(S, device=s.refs.device)
    parent = s.parents.long()
    known = (parent >= 0) & (parent < S)
    p = parent.clamp(0, S - 1)
    n = torch.where(known, s.lengths.long()[p], torch.zeros_like(p))
    full, part = torch.div(n, page, rounding_mode="floor"), n % page > 0
    # who keeps the partly filled page: the parent itself, else the first that continues it
    keeper = torch.full((S,), S, device=me.device).scatter_reduce(0, p, torch.where(known, torch.where(p == me, -1, me), S), "amin")
    same, keeps = known & (p == me), keeper[p] == me
    c = torch.arange(table.shape[1], device=me.device)[None]
    there = (table >= 0) & (table < pages)
    theirs, on = table[p], there[p] & known[:, None]
    shared = on & ((c < full[:, None]) | ((c == full[:, None]) & (part & keeps)[:, None])) & ~same[:, None]
    wanted = on & (c == full[:, None]) & (part & ~keeps & ~same)[:, None]
    refs = _count(_count(s.refs, table, there & ~same[:, None], -1), theirs, shared, 1)
    got, refs, missing = _take(refs, wanted)
    out = torch.where(same[:, None], table, torch.where(shared, theirs, got))
    moved = wanted & (got >= 0)
    _move_plain(s.pools, theirs[moved].long(), got[moved].long())
    return {"table": out.t(), "refs": refs, "lengths": n.int(), "missing": missing, "pools": s.pools}


def _compact_plain(s):
    pages, table = s.refs.numel(), s.table.t()
    live = s.refs > 0
    count = live.sum()
    number = torch.arange(pages, device=table.device)
    high, low = live & (number >= count), ~live & (number < count)
    source, target = number[high], number[low]
    where = torch.where(live, number, torch.full_like(number, -1))
    where[source] = target
    there = (table >= 0) & (table < pages)
    out = torch.where(there, where[table.clamp(0, pages - 1).long()], torch.full_like(number[:1], -1)).int()
    refs = torch.where(live & ~high, s.refs, torch.zeros_like(s.refs))
    refs[target] = s.refs[source]
    _move_plain(s.pools, source, target)
    return {"table": out.t(), "refs": refs, "live": count.int().reshape(1), "pools": s.pools}


# ------------------------------------------------------------------------------------------------ one pass
def _run_plain(s):
    kind = s.case["kind"]
    if kind == "window":
        y = _window_plain(s)
        if not s.case["train"]:
            return {"y": y}
        return {"y": y.detach(), "grads": torch.autograd.grad(y, (s.q, s.k, s.v), s.dy)}
    return {"y": _paged_plain(s)} if kind == "paged" else {"advance": _advance_plain, "fork": _fork_plain, "compact": _compact_plain}[kind](s)


def _run_own(s):
    from __graft_entry__ import load_package
    ca = load_package()
    case, kind = s.case, s.case["kind"]
    left = None if case.get("left", -1) < 0 else case["left"]
    if kind == "window":
        spans = None if s.documents is None else ca.token_spans(s.documents, s.groups)
        y = ca.window_attention(s.q, s.k, s.v, left, right=case["right"], lengths=s.lengths, cap=s.cap, slopes=s.slopes, spans=spans)
        if not case["train"]:
            return {"y": y}
        return {"y": y.detach(), "grads": torch.autograd.grad(y, (s.q, s.k, s.v), s.dy)}
    if kind == "paged":
        return {"y": ca.paged_window_attention(s.q, s.k_pages, s.v_pages, s.table, s.starts, s.lengths, left, sinks=case["sinks"],
                                               cap=s.cap, slopes=s.slopes, prefix=s.prefix)}
    if kind == "advance":
        table, refs, missing = ca.advance_pages(s.table, s.refs, s.starts, s.lengths, s.page, left, sinks=case["sinks"])
        return {"table": table, "refs": refs, "missing": missing}
    if kind == "fork":
        table, refs, lengths, missing = ca.fork_pages(s.pools, s.table, s.refs, s.lengths, s.parents)
        return {"table": table, "refs": refs, "lengths": lengths, "missing": missing, "pools": s.pools}
    table, refs, live = ca.compact_pages(s.pools, s.table, s.refs)
    return {"table": table, "refs": refs, "live": live, "pools": s.pools}


def run(s):
    return _run_own(s) if own else _run_plain(s)


# ------------------------------------------------------------------------------------------------ 64 bits
def _attend64(q, k, v, i, first, last, cap, slope, sinks=0, dy=None):
    """One head in 64 bits: queries at positions i, which see the keys first..last and those below `sinks` up to last;
    with dy also (dq, dk, dv)."""
    y, dq, dk, dv = (torch.zeros_like(t) for t in (q, q, k, v))
    j, scale = torch.arange(k.shape[0], device=k.device), q.shape[1] ** -0.5
    for lo in range(0, q.shape[0], 2048):
        rows = slice(lo, lo + 2048)
        a, b = first[rows, None], last[rows, None]
        sees = (j <= b) & ((j >= a) | (j < sinks))
        cols = sees.any(0).nonzero()[:, 0]
        if not cols.numel():
            continue
        kk, vv, sees = k[cols], v[cols], sees[:, cols]
        z = (q[rows] @ kk.T) * scale
        t = torch.tanh(z / cap) if cap else torch.zeros_like(z)
        z = cap * t if cap else z
        z = z - slope * (i[rows, None] - cols).abs().double()
        z = torch.where(sees, z, torch.tensor(-math.inf, dtype=z.dtype, device=z.device))
        p = torch.nan_to_num(torch.softmax(z, 1))
        y[rows] = p @ vv
        if dy is not None:
            dp = dy[rows] @ vv.T
            ds = p * (dp - (p * dp).sum(1, keepdim=True)) * (1 - t * t) * scale
            dq[rows] = ds @ kk
            dk[cols] += ds.T @ q[rows]
            dv[cols] += p.T @ dy[rows]
    return y, dq, dk, dv


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"window": _exact_window, "paged": _exact_paged, "advance": _exact_advance, "fork": _exact_fork, "compact": _exact_compact}[case["kind"]](s, case)


def _exact_window(s, case):
    Hq, Hkv, N = case["Hq"], case["Hkv"], case["N"]
    i = torch.arange(N, device="cuda")
    y, dq = (torch.zeros(s.q.shape, dtype=torch.float64, device="cuda") for _ in range(2))
    dk, dv = (torch.zeros(s.k.shape, dtype=torch.float64, device="cuda") for _ in range(2))
    slopes = s.slopes.tolist() if case["slopes"] else [0.0] * Hq
    for b, n in enumerate(_lengths(case)):
        if _spanned(case):
            first, last = (torch.tensor(x, device="cuda") for x in _runs(*_documents(case)[b]))
        else:
            first, last = torch.zeros_like(i), i + case["right"]
        if case["left"] >= 0:
            first = torch.maximum(first, i - case["left"])
        last = torch.where(i < n, last.clamp(max=n - 1), -1)
        for h in range(Hq):
            g = h // (Hq // Hkv)
            args = [t[:, hh, :, b].T.double() for t, hh in ((s.q, h), (s.k, g), (s.v, g))]
            dy = s.dy[:, h, :, b].T.double() if case["train"] else None
            got = _attend64(*args, i, first, last, case["cap"], slopes[h], 0, dy)
            y[:, h, :, b], dq[:, h, :, b] = got[0].T, got[1].T
            dk[:, g, :, b] += got[2].T
            dv[:, g, :, b] += got[3].T
    return {"y": y, "grads": (dq, dk, dv)} if case["train"] else {"y": y}


def _exact_paged(s, case):
    page, t, Hq = case["page"], 0, case["Hq"]
    G = Hq // case["Hkv"]
    y = torch.zeros(s.q.shape, dtype=torch.float64, device="cuda")
    slopes = s.slopes.tolist() if case["slopes"] else [0.0] * Hq
    prefixes = _prefixes(case) if case["prefix"] else [0] * case["S"]
    for b, (new, total) in enumerate(_chunks(case)):
        if not new:
            continue
        j = torch.arange(total, device="cuda")
        where, off = s.table[j // page, b].long(), j % page
        i = torch.arange(total - new, total, device="cuda")
        first = torch.zeros_like(i) if case["left"] < 0 else i - case["left"]
        last = i.clamp(min=prefixes[b] - 1)
        there = (where >= 0)[:, None]
        for h in range(Hq):
            kk, vv = (torch.where(there, pool[:, off, h // G, where.clamp(min=0)].T.double(), 0.0) for pool in (s.k_pages, s.v_pages))
            y[:, h, t:t + new] = _attend64(s.q[:, h, t:t + new].T.double(), kk, vv, i, first, last, case["cap"], slopes[h], case["sinks"])[0].T
        t += new
    return {"y": y}


def _lowest(refs):
    """Numbers of pages without users, lowest first; follows changes of refs as long as they only take pages."""
    at = 0
    while at < len(refs):
        if refs[at] <= 0:
            yield at
        at += 1


def _exact_advance(s, case):
    page, left, sinks = case["page"], case["left"], case["sinks"]
    rows, refs, starts = s.table.t().tolist(), s.refs.tolist(), s.starts.tolist()
    want, missing = [], 0
    for b, n in enumerate(s.lengths.tolist()):
        begin = n - (starts[b + 1] - starts[b])
        first = 0 if left < 0 else max(0, begin - left)
        for c, e in enumerate(rows[b]):
            tokens = range(c * page, min(c * page + page, n))
            stays = len(tokens) > 0 and (tokens[-1] >= first or tokens[0] < sinks)
            if e >= 0 and not stays:
                refs[e] -= 1
                rows[b][c] = -1
            elif e < 0 and len(tokens) and tokens[-1] >= begin:
                want.append((b, c))
    free = _lowest(refs)
    for b, c in want:
        p = next(free, None)
        if p is None:
            missing += 1
        else:
            rows[b][c], refs[p] = p, 1
    return {"table": _columns(rows), "refs": _ints(refs), "missing": _ints([missing])}


def _exact_fork(s, case):
    page, old, refs = case["page"], s.table.t().tolist(), s.refs.tolist()
    lengths, parents = s.lengths.tolist(), s.parents.tolist()
    width, rows, out, want = len(old[0]), [], [], []
    owner = {}
    for b, p in enumerate(parents):
        if p >= 0:
            owner[p] = p if parents[p] == p else min(owner.get(p, b), b)
    for b, p in enumerate(parents):
        out.append(lengths[p] if p >= 0 else 0)
        if p == b:
            rows.append(list(old[b]))
            continue
        for e in old[b]:
            if e >= 0:
                refs[e] -= 1
        row = [-1] * width
        for c in range(-(-out[b] // page)):
            whole = c * page + page <= out[b]
            if old[p][c] >= 0 and (whole or owner[p] == b):
                row[c] = old[p][c]
                refs[row[c]] += 1
            elif old[p][c] >= 0:
                want.append((b, c, old[p][c]))
        rows.append(row)
    free, missing, source, target = _lowest(refs), 0, [], []
    for b, c, e in want:
        f = next(free, None)
        if f is None:
            missing += 1
        else:
            rows[b][c], refs[f] = f, 1
            source.append(e)
            target.append(f)
    return {"table": _columns(rows), "refs": _ints(refs), "lengths": _ints(out), "missing": _ints([missing]), "pools": _moved(s.pools, source, target)}


def _exact_compact(s, case):
    rows, refs = s.table.t().tolist(), s.refs.tolist()
    used = [p for p, r in enumerate(refs) if r > 0]
    n = len(used)
    free = (p for p in range(n) if refs[p] <= 0)
    to, counts = {p: p if p < n else next(free) for p in used}, [0] * len(refs)
    for p in used:
        counts[to[p]] = refs[p]
    source = [p for p in used if to[p] != p]
    rows = [[to.get(e, -1) for e in row] for row in rows]
    return {"table": _columns(rows), "refs": _ints(counts), "live": _ints([n]), "pools": _moved(s.pools, source, [to[p] for p in source])}


def _moved(pools, source, target):
    for pool in pools:
        kept = {p: pool[..., p].clone() for p in source}
        for p, f in zip(source, target):
            pool[..., f] = kept[p]
    return pools
