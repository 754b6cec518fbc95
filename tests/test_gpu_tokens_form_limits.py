"""Attention with other scores and masks where calls go to extremes: caps and scales of every size, hidden places that hold
anything, windows behind a table, calls that are not full, sequences of many tiles, strides, streams, threads, graphs, and pools
beyond 32 bits."""
import math
import threading

import pytest
import torch

from tests import tokens_form_reference as ref
from tests.test_gpu_tokens_form import call, ints, numbers, problem, slopes_of
from tests.test_gpu_tokens_window import make

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
types = pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])


def gradients(ca, case, x, dy, *form, **kw):
    x = [t.detach().cuda().requires_grad_(True) for t in x]
    y = call(ca, case, *x, *form, **kw)
    return dict(zip(("dq", "dk", "dv"), torch.autograd.grad(y, x, dy.cuda())), y=y)


@types
@pytest.mark.parametrize("cap,scale,size", [(20.0, -0.3, 1.5), (20.0, 0.0, 1.5), (200.0, None, 100.0), (69.0, None, 60.0), (1e-6, None, 1.0), (1e6, None, 1.0),
                                            (3.0, 1e-7, 1.0), (1e30, None, 2.0)])
def test_caps_and_scales(ca, dtype, cap, scale, size):
    """Those whose scores the exponents of 16-bit weights stand without a reference, and others; polynomials whose coefficients
    hold the factors, and others; scores turned round."""
    case = (64, 2, 1, 140, 1, 90, 0, 2, None, cap, False, 0, 0)
    q, k, v, dy, *form = problem(case, dtype, size)
    got = gradients(ca, case, (q, k, v), dy, *form, scale=scale)
    for name, (value, bound) in ref.window(q, k, v, 90, 0, 2, None, cap, None, None, None, dy, scale).items():
        ref.check(got[name], value, bound, name)


@pytest.mark.parametrize("dtype,cap,large", [(torch.bfloat16, 50.0, 1e25), (torch.bfloat16, 30.0, 1e25), (torch.bfloat16, 60.0, 1e25), (torch.float16, 50.0, 500.0),
                                             (torch.float32, 50.0, 1e25)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_large_values_and_scores_at_the_cap(ca, dtype, cap, large, sign):
    """All of a row's scores near +cap, or near -cap, and values near the type's limits: weights without a reference hold both."""
    case = (64, 2, 1, 260, 1, None, 0, 0, None, cap, False, 0, 0)
    q, k, v, dy, *form = problem(case, dtype)
    q, k = (t.abs() * f for t, f in ((q, 20.0), (k, 5.0 * sign)))           # scores of about 8 * 64 * 80 / 8
    v = (v.float() * large).to(dtype)
    got = gradients(ca, case, (q, k, v), dy, *form)
    for name, (value, bound) in ref.window(q, k, v, None, 0, 0, None, cap, None, None, None, dy).items():
        if name in ("y", "dv"):                                             # the cap's derivative is 0, so dq and dk are what is left of it
            ref.check(got[name], value, bound, name)
        assert torch.isfinite(got[name]).all(), name


@types
def test_only_far_keys(ca, dtype):
    """The near pages are gone: every key is thousands of tokens away, the bias alone is some 17000 in the exponent."""
    D, Hq, Hkv, page, new, n = 64, 2, 1, 16, 150, 6000
    kp, vp = (make(s, (D, page, Hkv, 10), dtype) for s in (2, 3))
    q = make(1, (D, Hq, new), dtype, 2.0)
    table = [[4, 5, 6] + [-1] * 373]
    slopes = torch.tensor([2.0, 0.5])
    for cap in (10.0, None):
        got = ca.paged_window_attention(q.cuda(), kp.cuda(), vp.cuda(), ints(table).t(), ints([0, new]), ints([n]), cap=cap, slopes=slopes.cuda())
        ref.check(got, *ref.paged(q, kp, vp, table, [0, new], [n], None, 0, cap, slopes, None))
        one = ca.paged_window_attention(q[:, :, -1:].cuda(), kp.cuda(), vp.cuda(), ints(table).t(), ints([0, 1]), ints([n]), cap=cap, slopes=slopes.cuda())
        ref.check(one, *ref.paged(q[:, :, -1:], kp, vp, table, [0, 1], [n], None, 0, cap, slopes, None))


@types
@pytest.mark.parametrize("D,Hq,Hkv,N,B,longest,group", [(64, 8, 1, 5001, 2, 900, 20), (128, 1, 1, 17000, 1, 17000, 0)])
def test_many_tiles(ca, D, Hq, Hkv, N, B, longest, group, dtype):
    """More tiles than ranks, the last run of them shorter: the result of the same call for a piece that stands alone."""
    case = (D, Hq, Hkv, N, B, 300, 0, 0, None, 15.0, True, longest, group)
    q, k, v, dy, slopes, docs, groups = problem(case, dtype)
    got = gradients(ca, case, (q, k, v), dy, slopes, docs, groups)
    # the last tokens of the first sequence: what they see, and what sees them, lies in the last 900 of them
    n, keep = 900, 600
    part = [t[:, :, N - n:, :1] for t in (q, k, v, dy)]
    want = ref.window(*part[:3], 300, 0, 0, None, 15.0, slopes, [docs[0][N - n:]], groups and [groups[0][N - n:]], part[3])
    for name, (value, bound) in want.items():
        ref.check(got[name][:, :, N - keep:, :1], value[:, :, n - keep:], bound[:, :, n - keep:], name)


@types
@pytest.mark.parametrize("new", [1, 40, 200])
def test_hidden_places_of_a_cache(ca, dtype, new):
    """Freed pages, places behind a length and behind a prefix's window may hold anything."""
    D, Hq, Hkv, page, width, pages = 64, 4, 2, 16, 30, 80
    lengths, starts, left = [300, new, 410], [0, new, 2 * new, 3 * new], 64
    table = [[3 * c + s for c in range(26)] + [-1] * 4 for s in range(3)]
    q = make(1, (D, Hq, 3 * new), dtype, 4.0).cuda()
    kp, vp = (make(s, (D, page, Hkv, pages), dtype).cuda() for s in (2, 3))
    seen = torch.zeros(pages, page, dtype=torch.bool)
    for s, n in enumerate(lengths):
        for j in range(max(0, n - new - left), n):
            seen[table[s][j // page], j % page] = True
    for form in (dict(cap=9.0), dict(slopes=slopes_of(Hq).cuda()), dict(prefix=ints([290, new, 405])), dict(cap=9.0, slopes=slopes_of(Hq).cuda(), prefix=ints([0, 5, 400]))):
        run = lambda k, v: ca.paged_window_attention(q, k, v, ints(table).t(), ints(starts), ints(lengths), left, **form)
        plain = run(kp, vp)
        for junk in (math.nan, math.inf, torch.finfo(dtype).min):
            k, v = kp.clone(), vp.clone()
            for t in (k, v):
                t.permute(3, 1, 0, 2)[~seen] = junk
            assert torch.equal(run(k, v), plain), (form.keys(), junk)


@types
@pytest.mark.parametrize("new", [1, 90])
def test_calls_that_are_not_full(ca, dtype, new):
    """Packed tokens of no sequence give zeros; sequences without tokens, missing pages, windows behind the table."""
    D, Hq, Hkv, page, T = 128, 4, 2, 16, 2 * new + 60
    kp, vp = (make(s, (D, page, Hkv, 20), dtype).cuda() for s in (2, 3))
    q = make(1, (D, Hq, T), dtype, 4.0).cuda()
    table, starts, lengths = [[1, 2, 3, -1, 5, 6, 7], [8] * 7, [-1] * 7], [7, 7 + new, 7 + new, 7 + 2 * new], [7 * page, 5000, new]
    for form in (dict(cap=9.0), dict(slopes=slopes_of(Hq).cuda()), dict(cap=9.0, slopes=slopes_of(Hq).cuda(), prefix=ints([20, 0, 3]))):
        y = ca.paged_window_attention(q, kp, vp, ints(table).t(), ints(starts), ints(lengths), 50, sinks=3, **form)
        assert not y[:, :, :7].any() and not y[:, :, 7 + new:].any()          # the second has no tokens, the third no pages
        f = dict(cap=form.get("cap"), slopes=slopes_of(Hq) if "slopes" in form else None, prefix=[20] if "prefix" in form else None)
        want = ref.paged(q[:, :, 7:7 + new].cpu(), kp.cpu(), vp.cpu(), table[:1], [0, new], lengths[:1], 50, 3, f["cap"], f["slopes"], f["prefix"])
        ref.check(y[:, :, 7:7 + new], *want)


@types
def test_strides(ca, dtype):
    """Slices of one projection, taken as they lie, and tensors that have to be copied."""
    D, H, N, B = 64, 6, 150, 2
    case = (D, 4, 1, N, B, None, 0, 0, None, 12.0, True, 70, 20)
    slopes, (docs, groups) = slopes_of(4), numbers(N, B, 70, 20, 5)
    packed = make(3, (D, H, N, B), dtype, 2.0).cuda()
    dy = make(4, (D, 4, N, B), dtype)
    parts = packed[:, :4], packed[:, 4:5], packed[:, 5:]
    want = gradients(ca, case, [t.contiguous() for t in parts], dy, slopes, docs, groups)
    for views in (parts, [t.permute(2, 0, 3, 1).contiguous().permute(1, 3, 0, 2) for t in parts]):
        got = {"y": None}
        x = [t.detach().requires_grad_(True) for t in views]
        y = call(ca, case, *x, slopes, docs, groups)
        got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(y, x, dy.cuda())), y=y)
        assert all(torch.equal(got[n], want[n]) for n in want)
    # numbers of documents that lie row by row are copied
    rows = ints(docs).t().contiguous()
    assert torch.equal(ca.token_spans(rows, ints(groups).t()), ca.token_spans(ints(docs).t(), ints(groups).t()))


@types
def test_again_and_at_once(ca, dtype):
    """Repeated calls give the same bits, on two streams and two host threads at once too."""
    case = (128, 4, 2, 900, 2, None, 0, 0, None, 12.0, True, 500, 100)
    q, k, v, dy, *form = problem(case, dtype)
    base = gradients(ca, case, (q, k, v), dy, *form)
    torch.cuda.synchronize()
    got, streams = [[], []], [torch.cuda.Stream(), torch.cuda.Stream()]

    def work(i):
        with torch.cuda.stream(streams[i]):
            for _ in range(5):
                got[i].append(gradients(ca, case, (q, k, v), dy, *form))
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert all(len(g) == 5 for g in got)
    assert all(torch.equal(r[n], base[n]) for g in got for r in g for n in base)
    ca.ops.check_status()


@types
def test_a_step_in_a_graph(ca, dtype):
    """Forward and backward captured, replayed on other numbers of documents and other tensors."""
    case = (64, 4, 2, 400, 1, None, 0, 0, None, 12.0, True, 200, 30)
    q, k, v, dy, slopes, docs, groups = problem(case, dtype)
    x = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    d, g, sl, dy = ints(docs).t(), ints(groups).t(), slopes.cuda(), dy.cuda()

    def step():
        y = ca.window_attention(*x, None, cap=12.0, slopes=sl, spans=ca.token_spans(d, g))
        return [y, *torch.autograd.grad(y, x, dy)]
    graph, got = ca.capture(step)
    docs2, groups2 = numbers(400, 1, 50, 9, 77)
    with torch.no_grad():
        d.copy_(ints(docs2).t())
        g.copy_(ints(groups2).t())
        x[0].mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_spans_that_do_not_belong(ca):
    """Spans of other documents than any: wrong results at most, no memory but the call's own and no wait that runs out."""
    q, k, v, dy = (make(i, (64, 2, 700, 2), torch.bfloat16).cuda().requires_grad_(True) for i in range(4))
    g = torch.Generator(device="cuda").manual_seed(1)
    for low, high in ((0, 700), (-2 ** 31, 2 ** 31 - 1), (0, 1)):
        spans = torch.randint(low, high, (2, 700, 4), dtype=torch.int32, device="cuda", generator=g).permute(2, 1, 0)
        for dtype in DTYPES:
            a, b, c = (t.detach().to(dtype).requires_grad_(True) for t in (q, k, v))
            y = ca.window_attention(a, b, c, None, cap=10.0, spans=spans)
            torch.autograd.grad(y, (a, b, c), dy.detach().to(dtype))
    torch.cuda.synchronize()
    ca.ops.check_status()


def test_pools_beyond_32_bits(ca):
    """Pages whose offsets pass 2^32 elements: moved, and read by attention with a cap."""
    D, heads, page = 128, 8, 64
    pages = 2 ** 32 // (D * heads * page) + 40
    pool = torch.zeros(pages, heads, page, D, dtype=torch.bfloat16, device="cuda").permute(3, 2, 1, 0)
    table, refs = [[pages - 1, 3, pages - 7]], [0] * pages
    for i, e in enumerate(table[0]):
        pool[..., e] = make(i, (D, page, heads), torch.bfloat16).cuda()
        refs[e] = 1
    q = make(9, (D, heads, 5), torch.bfloat16, 3.0).cuda()
    where = (ints([0, 5]), ints([150]))
    before = ca.paged_window_attention(q, pool, pool, ints(table).t(), *where, cap=20.0)
    new, counts, live = ca.compact_pages([pool], ints(table).t(), ints(refs))
    assert live.item() == 3 and sorted(new[:, 0].tolist()) == [0, 1, 2] and int(counts.sum()) == 3
    pool[..., 3:].zero_()
    assert torch.equal(ca.paged_window_attention(q, pool, pool, new, *where, cap=20.0), before) and before.any()
