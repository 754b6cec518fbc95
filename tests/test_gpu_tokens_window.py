"""Attention with a sliding window and first tokens that stay visible: forward and gradients against the formulas in 64
bits, with bounds that follow from the storage's rounding (tests/tokens_reference.py), against differences, and what masked
places, strides, streams and repeated calls must not change."""
import math

import pytest
import torch

from tests import tokens_reference as ref

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(seed, shape, dtype, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    t = torch.randn(tuple(reversed(shape)), generator=g, dtype=torch.float64) * scale
    return t.to(dtype).permute(tuple(range(len(shape) - 1, -1, -1)))


def problem(D, Hq, Hkv, N, B, dtype, seed=0):
    return (make(seed, (D, Hq, N, B), dtype, 1.5), make(seed + 1, (D, Hkv, N, B), dtype), make(seed + 2, (D, Hkv, N, B), dtype),
            make(seed + 3, (D, Hq, N, B), dtype))


def run(ca, q, k, v, dy, left, right=0, sinks=0, lengths=None, scale=None):
    q, k, v = (t.detach().cuda().requires_grad_(True) for t in (q, k, v))
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    y = ca.window_attention(q, k, v, left, right=right, sinks=sinks, lengths=n, scale=scale)
    dq, dk, dv = torch.autograd.grad(y, (q, k, v), dy.cuda())
    return {"y": y, "dq": dq, "dk": dk, "dv": dv}


def compare(got, q, k, v, dy, left, right=0, sinks=0, lengths=None, scale=None):
    want = ref.window(q.double(), k.double(), v.double(), left, right, sinks, lengths, scale, dy.double(), ref.UNIT[q.dtype])
    for name, (x, e) in want.items():
        ref.check(got[name], x, e, name)


CASES = [
    # D, Hq, Hkv, N, B, left, right, sinks, lengths
    (64, 1, 1, 1, 1, None, 0, 0, None),                  # one token
    (64, 2, 1, 2, 1, 0, 0, 0, None),                     # each token sees itself only
    (64, 2, 2, 63, 2, 5, 0, 1, None),
    (64, 4, 1, 129, 1, 64, 0, 4, None),                  # shared key head, one row behind a tile
    (128, 3, 1, 128, 2, 127, 0, 2, None),                # three query heads a key head
    (128, 8, 1, 200, 1, 33, 0, 0, None),                 # eight
    (128, 2, 2, 257, 1, None, 0, 0, None),               # no left end
    (128, 4, 2, 385, 1, 128, 0, 128, None),              # a whole tile of first tokens
    (64, 2, 1, 500, 1, 63, 0, 130, None),                # first tokens that end inside the second tile
    (64, 2, 1, 300, 1, 20, 0, 1000, None),               # more first tokens than tokens
    (64, 1, 1, 300, 2, 10, 7, 0, None),                  # both sides
    (64, 2, 1, 300, 1, 0, 200, 3, None),                 # the future mostly
    (128, 2, 1, 260, 1, 31, 400, 0, None),               # right end beyond the sequence
    (64, 2, 1, 290, 4, 70, 0, 4, [290, 0, 1, 133]),      # unequal lengths, an empty one
    (64, 2, 2, 290, 3, None, 290, 0, [129, 128, 290]),   # everything visible
    (8, 1, 1, 100, 1, 30, 0, 2, None),                   # few features
    (24, 3, 1, 150, 1, 40, 0, 2, None),
    (72, 2, 1, 150, 1, 40, 3, 2, None),
    (96, 6, 2, 333, 2, 100, 0, 5, [333, 200]),
    (120, 5, 1, 140, 1, 12, 0, 1, None),                 # five query heads a key head
    (128, 4, 1, 1500, 1, 700, 0, 6, None),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace(" ", "") for x in c))
def test_window_attention_and_gradients(ca, case, dtype):
    D, Hq, Hkv, N, B, left, right, sinks, lengths = case
    q, k, v, dy = problem(D, Hq, Hkv, N, B, dtype)
    got = run(ca, q, k, v, dy, left, right, sinks, lengths)
    compare(got, q, k, v, dy, left, right, sinks, lengths)
    if lengths is not None:
        for b, n in enumerate(lengths):
            assert all(not t[:, :, n:, b].any() for t in got.values())
    # the forward without gradients is the same call
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    with torch.no_grad():
        y = ca.window_attention(q.cuda(), k.cuda(), v.cuda(), left, right=right, sinks=sinks, lengths=n)
    assert torch.equal(y, got["y"])


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
def test_whatever_lies_behind_the_length_has_no_effect(ca, dtype):
    q, k, v, dy = problem(64, 4, 2, 300, 3, dtype)
    lengths = [300, 131, 0]
    plain = run(ca, q, k, v, dy, 50, 0, 3, lengths)
    for junk in (math.nan, math.inf, torch.finfo(dtype).min):
        qq, kk, vv, dd = (t.clone() for t in (q, k, v, dy))
        for t in (qq, kk, vv, dd):
            for b, n in enumerate(lengths):
                t[:, :, n:, b] = junk
        got = run(ca, qq, kk, vv, dd, 50, 0, 3, lengths)
        for name in plain:
            assert torch.equal(plain[name], got[name]), (name, junk)


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize("D", [64, 128])
def test_what_is_not_a_number_is_not_hidden(ca, dtype, D):
    """A key that is not a number shows in every token that sees it, at whatever place of a tile the key is; tokens of tiles
    further on are not touched."""
    q, k, v, _ = (t.cuda() for t in problem(D, 2, 1, 600, 1, dtype))
    for j in (*range(8, 17), 63, 64, 70, 71, 127, 128, 255):
        bad = k.clone()
        bad[:, 0, j, 0] = math.nan
        with torch.no_grad():
            y = ca.window_attention(q, bad, v, 40)
        assert y[:, :, j : j + 41, 0].isnan().all()
        assert not y[:, :, j + 300 :, 0].isnan().any()


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
def test_empty_sequences_give_zeros_every_time(ca, dtype):
    """Tiles that see no key at all, next to some that do, many times over: nothing that was on its way lands in the results."""
    q, k, v, dy = (t.cuda() for t in problem(128, 4, 2, 300, 4, dtype))
    n = torch.tensor([0, 300, 0, 7], dtype=torch.int32, device="cuda")
    with torch.no_grad():
        for _ in range(100):
            y = ca.window_attention(q, k, v, 50, sinks=3, lengths=n)
            assert not y[..., 0].any() and not y[..., 2].any() and not y[:, :, 7:, 3].any()


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize("size", [1e-3, 40.0])
def test_flat_and_peaked_rows(ca, dtype, size):
    """Scores that all are nearly equal, and scores of some hundreds that grow along the sequence, so that every tile
    raises the row's maximum."""
    D, N = 64, 520
    q, k, v, dy = problem(D, 2, 1, N, 1, torch.float64)
    ramp = torch.linspace(0.1, 1.0, N, dtype=torch.float64)[None, None, :, None]
    q, k = q.abs() * size ** 0.5, k.abs() * ramp * size ** 0.5
    q, k, v, dy = (t.to(dtype) for t in (q, k, v, dy))
    got = run(ca, q, k, v, dy, None)
    peak = float((q.double()[:, 0, :, 0].T @ k.double()[:, 0, :, 0]).abs().max()) / math.sqrt(D)
    # a Float32 score of this size is itself uncertain by peak * 2^-22, which the weights inherit
    u, old = ref.UNIT[dtype], ref.SLACK
    ref.SLACK = max(old, 8 * peak * 2.0 ** -22)
    try:
        compare(got, q, k, v, dy, None)
    finally:
        ref.SLACK = old
    assert u >= 0


@pytest.mark.parametrize("size", [2.0 ** -12, 1.0, 4096.0])
def test_range_of_half_precision(ca, size):
    """Scaled losses and vanishing gradients, and rows whose weights are all below the smallest normal half: the products'
    operands stay inside the type's range."""
    D, N = 64, 900
    q, k, v, dy = problem(D, 2, 1, N, 1, torch.float64)
    q = q * 0.01                                        # flat rows: weights of about 1/900
    v = v * (1.0 / size if size > 1 else 1.0)           # gradients of k and q stay inside the type
    dy = dy * size
    q, k, v, dy = (t.to(torch.float16) for t in (q, k, v, dy))
    got = run(ca, q, k, v, dy, None, 899, 0)
    want = ref.window(q.double(), k.double(), v.double(), None, 899, 0, None, None, dy.double(), ref.UNIT[torch.float16])
    for name, (x, e) in want.items():
        # results below the smallest normal half are rounded to multiples of 2^-24
        ref.check(got[name], x, e + 2.0 ** -24, name)
        norm = float((got[name].double().cpu() - x).norm() / x.norm())
        assert norm < 2.0 ** -11 or float(x.abs().amax()) < 2.0 ** -9, (name, norm)


def test_gradients_against_differences(ca):
    q, k, v, dy = problem(24, 4, 2, 90, 2, torch.float32)
    args = dict(left=17, right=2, sinks=3, lengths=[90, 55])
    grads = run(ca, q, k, v, dy, **args)
    n = torch.tensor(args["lengths"], dtype=torch.int32, device="cuda")

    def loss(*x):
        y = ca.window_attention(*(t.cuda() for t in x), 17, right=2, sinks=3, lengths=n)
        return float((y.double() * dy.cuda().double()).sum())

    for at, name in enumerate(("dq", "dk", "dv")):
        x = [q, k, v]
        d = make(50 + at, x[at].shape, torch.float32)
        h = 1e-2
        up, down = list(x), list(x)
        up[at], down[at] = x[at] + h * d, x[at] - h * d
        numeric = (loss(*up) - loss(*down)) / (2 * h)
        # third derivatives of order |d|^3 h^2 and the Float32 loss: a percent of the size of the sum's terms
        formula = float((grads[name].double().cpu() * d.double()).sum())
        size = float((grads[name].double().cpu() * d.double()).square().sum().sqrt())
        assert abs(numeric - formula) < 0.02 * size + 0.01 * abs(formula), (name, numeric, formula)


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
def test_strides_and_orders(ca, dtype):
    D, Hq, Hkv, N, B = 64, 4, 2, 140, 3
    q, k, v, dy = (t.cuda() for t in problem(D, Hq, Hkv, N, B, dtype))
    base = run(ca, q, k, v, dy, 30, 0, 2)

    def same(*x):
        got = run(ca, *x, 30, 0, 2)
        for name in base:
            assert torch.equal(base[name], got[name]), name

    packed = torch.cat([q, k, v], 1)                                   # one projection, sliced
    packed = packed.permute(3, 2, 1, 0).contiguous().permute(3, 2, 1, 0)
    same(packed[:, :Hq], packed[:, Hq:Hq + Hkv], packed[:, Hq + Hkv:], dy)
    rows = lambda t, order: t.permute(order).contiguous().permute([order.index(i) for i in range(4)])
    same(*(rows(t, (3, 1, 2, 0)) for t in (q, k, v, dy)))              # heads outside tokens
    same(*(rows(t, (2, 3, 1, 0)) for t in (q, k, v, dy)))              # batch inside tokens
    same(*(rows(t, (0, 1, 2, 3)) for t in (q, k, v, dy)))              # features outermost: copied
    wide = [torch.empty(D + 1, t.shape[1], N, B, dtype=dtype, device="cuda") for t in (q, k, v, dy)]
    for w, t in zip(wide, (q, k, v, dy)):
        w[1:] = t
    same(*(w[1:] for w in wide))                                       # features not contiguous, address off by one element
    shared = k[:, :1].expand(D, Hkv, N, B)                             # a broadcast input: its gradient is the sum
    kk = k[:, :1].clone().requires_grad_(True)
    y = ca.window_attention(q, kk.expand(D, Hkv, N, B), v, 30, sinks=2)
    (g,) = torch.autograd.grad(y, (kk,), dy)
    full = run(ca, q, shared, v, dy, 30, 0, 2)
    assert torch.equal(y, full["y"]) and torch.equal(g, full["dk"].sum(1, keepdim=True))
    one = torch.ones((), dtype=dtype, device="cuda")                   # an expanded cotangent
    got = run(ca, q, k, v, one.expand(q.shape), 30, 0, 2)
    want = run(ca, q, k, v, torch.ones_like(q), 30, 0, 2)
    assert all(torch.equal(got[n], want[n]) for n in got)


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
def test_repeated_calls_and_other_streams(ca, dtype):
    q, k, v, dy = (t.cuda() for t in problem(128, 8, 2, 1100, 2, dtype))
    base = run(ca, q, k, v, dy, 200, 0, 4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            got = run(ca, q, k, v, dy, 200, 0, 4)
    torch.cuda.current_stream().wait_stream(side)
    for name in base:
        assert torch.equal(base[name], got[name]), name
    ca.ops.check_status()


def test_a_host_thread_of_its_own(ca):
    """The first CUDA call of a thread: tensor maps are made through the driver, which needs the device's context there."""
    import threading
    q, k, v, dy = (t.cuda() for t in problem(64, 4, 2, 300, 1, torch.bfloat16))
    base = run(ca, q, k, v, dy, 60, 0, 4)["y"].detach()
    got = []

    def work():
        with torch.no_grad():
            got.append(ca.window_attention(q, k, v, 60, sinks=4))
    for _ in range(3):
        t = threading.Thread(target=work)
        t.start()
        t.join()
    assert len(got) == 3 and all(torch.equal(g, base) for g in got)


def test_in_a_graph(ca):
    q, k, v, dy = (t.cuda() for t in problem(64, 4, 2, 300, 1, torch.bfloat16))
    base = run(ca, q, k, v, dy, 60, 0, 4)
    graph, got = ca.capture(lambda: run(ca, q, k, v, dy, 60, 0, 4))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(base[n], got[n]) for n in base)


def test_no_tokens(ca):
    for shape in ((64, 4, 0, 2), (64, 4, 5, 0)):
        q = torch.empty(shape, device="cuda", requires_grad=True)
        y = ca.window_attention(q, q, q, 5)
        assert y.shape == shape
        (g,) = torch.autograd.grad(y.sum(), (q,))
        assert g.shape == shape


def test_refusals(ca):
    q = torch.zeros(64, 4, 10, 2, device="cuda")
    k = torch.zeros(64, 2, 10, 2, device="cuda")
    at = ca.window_attention
    with pytest.raises(RuntimeError, match="only CUDA compatible"):
        at(q.cpu(), k.cpu(), k.cpu(), 3)
    with pytest.raises(TypeError, match="k is BFloat16"):
        at(q, k.bfloat16(), k, 3)
    with pytest.raises(TypeError, match="Float16 are supported"):
        at(q.double(), k.double(), k.double(), 3)
    with pytest.raises(AssertionError, match="expected, k and v alike"):
        at(q, k, k[:, :1], 3)
    with pytest.raises(AssertionError, match="expected, k and v alike"):
        at(q, k[:, :, :9], k[:, :, :9], 3)
    with pytest.raises(AssertionError, match="must not be negative"):
        at(q, k, k, -1)
    with pytest.raises(ca.CircAttError, match="right=-1"):
        at(q, k, k, 3, right=-1)
    with pytest.raises(ca.CircAttError, match="sinks=-2"):
        at(q, k, k, 3, sinks=-2)
    with pytest.raises(ca.CircAttError, match="positive multiple"):
        at(q[:, :3], k, k, 3)
    with pytest.raises(ca.CircAttError, match="multiples of 8 up to 128"):
        at(q[:60], k[:60], k[:60], 3)
    big = torch.zeros(136, 1, 4, 1, device="cuda")
    with pytest.raises(ca.CircAttError, match="multiples of 8 up to 128"):
        at(big, big, big, 3)
    with pytest.raises(TypeError, match="lengths must be Int"):
        at(q, k, k, 3, lengths=torch.tensor([1, 2], device="cuda"))
    with pytest.raises(AssertionError, match="one for each of the batch"):
        at(q, k, k, 3, lengths=torch.tensor([1], device="cuda", dtype=torch.int32))
    with pytest.raises(OverflowError):
        at(q, k, k, 1 << 40)
