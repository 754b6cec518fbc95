"""Capped scores where all that a row sees lies near -cap, and values of every size: the weights' reference has to leave room for
what they multiply, at both ends of the exponents."""
import pytest
import torch

from tests import tokens_form_reference as ref
from tests.test_gpu_tokens_form import ints
from tests.test_gpu_tokens_form_limits import gradients, types
from tests.test_gpu_tokens_window import make

pytestmark = pytest.mark.gpu


def saturated(dtype, N, factor, sign, value, heads=2, B=1):
    """q, k, v, dy with raw scores of about 5.1 * factor * sign, none of the other sign."""
    q, k, v, dy = (make(i, (64, h, N, B), dtype) for i, h in ((0, heads), (1, 1), (2, 1), (3, heads)))
    q, k = (q.float().abs() * factor).to(dtype), (k.float().abs() * sign).to(dtype)
    return q, k, (v.float() * value).to(dtype), dy


def documents(N):
    """One token, two, three and so on: first tokens that see only themselves."""
    out, k = [], 0
    while len(out) < N:
        out += [k] * (k + 1)
        k += 1
    return [out[:N]]


SIZES = [(torch.bfloat16, x) for x in (1e25, 1.0, 1e-2, 1e-4)] + [(torch.float16, x) for x in (500.0, 1.0, 1e-2)] + [(torch.float32, x) for x in (1e25, 1.0, 1e-4)]


@pytest.mark.parametrize("dtype,value", SIZES)
@pytest.mark.parametrize("cap", [20.0, 33.0, 34.0, 45.0, 50.0, 50.6])
@pytest.mark.parametrize("sign", [-1.0, 1.0])
@pytest.mark.parametrize("packed", [False, True])
def test_values_of_rows_at_the_cap(ca, dtype, value, cap, sign, packed):
    """Scores far beyond -cap (or +cap), many keys and one: y and dv element by element.  The cap's derivative is 0 there."""
    q, k, v, dy = saturated(dtype, 260, 100.0, sign, value)
    docs = documents(260) if packed else None
    got = gradients(ca, (64, 2, 1, 260, 1, None, 0, 0, None, cap), (q, k, v), dy, None, docs, None)
    for name, (x, bound) in ref.window(q, k, v, None, 0, 0, None, cap, None, docs, None, dy).items():
        if name in ("y", "dv"):
            ref.check(got[name], x, bound, name)
        assert torch.isfinite(got[name]).all(), name


@types
@pytest.mark.parametrize("cap", [30.0, 50.0])
@pytest.mark.parametrize("value", [1.0, 1e-2])
def test_gradients_of_rows_before_the_cap(ca, dtype, cap, value):
    """Raw scores of about -100: the lowest weights with a derivative left, all gradients."""
    q, k, v, dy = saturated(dtype, 200, 20.0, -1.0, value)
    docs = documents(200)
    got = gradients(ca, (64, 2, 1, 200, 1, None, 0, 0, None, cap), (q, k, v), dy, None, docs, None)
    for name, (x, bound) in ref.window(q, k, v, None, 0, 0, None, cap, None, docs, None, dy).items():
        ref.check(got[name], x, bound, name)


@types
@pytest.mark.parametrize("cap", [33.0, 45.0, 50.0, 50.6])
@pytest.mark.parametrize("factor", [14.0, 20.0, 100.0])
def test_rows_that_see_one_key(ca, dtype, cap, factor):
    """Their result is the key's value, to the bit, whatever its size."""
    q, k, v, _ = saturated(dtype, 300, factor, -1.0, 1.0)
    v = (v.double() * torch.logspace(-3, 0, 300, dtype=torch.float64)[None, None, :, None]).to(dtype)
    y = ca.window_attention(q.cuda(), k.cuda(), v.cuda(), 0, cap=cap)
    assert torch.equal(y.cpu(), v.expand_as(y)) if dtype is not torch.float32 else torch.allclose(y.cpu(), v.expand_as(y), rtol=1e-6, atol=0)


@types
@pytest.mark.parametrize("cap", [33.0, 45.0, 50.0, 50.6])
@pytest.mark.parametrize("value", [1.0, 1e-2, 1e-4])
def test_chunks_as_single_tokens(ca, dtype, cap, value):
    """Over a cache: chunks and single tokens, which other kernels take, are both within the bound."""
    D, page, n, new = 64, 16, 300, 200
    q, k, v, _ = saturated(dtype, n, 100.0, -1.0, value, heads=4)
    pool = lambda t: torch.cat([t[:, 0, :, 0], torch.zeros(D, 20, dtype=dtype)], 1).reshape(D, 20, page).permute(1, 2, 0).contiguous()[:, None].permute(3, 2, 1, 0).cuda()
    kp, vp = pool(k), pool(v)
    qs, table = q[:, :, n - new:, 0].permute(2, 1, 0).contiguous().permute(2, 1, 0), [list(range(20))]
    y = ca.paged_window_attention(qs.cuda(), kp, vp, ints(table).t(), ints([0, new]), ints([n]), 150, cap=cap)
    x, bound = ref.paged(qs, kp.cpu(), vp.cpu(), table, [0, new], [n], 150, 0, cap, None, None)
    ref.check(y, x, bound, "chunk")
    one = ca.paged_window_attention(qs[:, :, -1:].cuda(), kp, vp, ints(table).t(), ints([0, 1]), ints([n]), 150, cap=cap)
    ref.check(one, x[:, :, -1:], bound[:, :, -1:], "one token")


@pytest.mark.parametrize("cap,value", [(33.0, 1e-15), (33.0, 1e25), (50.0, 1e-34), (50.0, 1e34)])
def test_small_and_large_values(ca, cap, value):
    """bfloat16's range.  A reference without a look for the maximum, for caps up to 33, has weights of 2^-64 to 2^32: weighted sums are
    held from 2^-62 (2e-19) on and up to 2^95 by the number of keys; with other caps, as far as Float32 goes."""
    q, k, v, _ = saturated(torch.bfloat16, 260, 100.0, -1.0, value)
    y = ca.window_attention(q.cuda(), k.cuda(), v.cuda(), None, cap=cap)
    x, bound = ref.window(q, k, v, None, 0, 0, None, cap, None, None, None)["y"]
    ref.check(y.double().cpu() / value, x / value, bound / value, "y")          # in units of the values: the check's own slack is 1e-30


@pytest.mark.parametrize("cap", [33.0, 34.0])
@pytest.mark.parametrize("sign", [-1.0, 1.0])
def test_smallest_values(ca, cap, sign):
    """One key a row, with values from 2^-61 on."""
    q, k, v, _ = saturated(torch.bfloat16, 260, 100.0, sign, 1.0)
    v = ((1 + v.float().abs()) * v.float().sign() * 2.0 ** -61).to(torch.bfloat16)
    y = ca.window_attention(q.cuda(), k.cuda(), v.cuda(), 0, cap=cap)
    assert torch.equal(y.cpu(), v.expand_as(y))


@types
@pytest.mark.parametrize("new", [1, 3, 100])
def test_negative_prefixes(ca, dtype, new):
    """No prefix, whatever negative number says so."""
    D, page, n = 64, 16, 150
    kp, vp = (make(s, (D, page, 2, 10), dtype).cuda() for s in (2, 3))
    q = make(1, (D, 4, new), dtype, 2.0).cuda()
    where = (ints([list(range(10))]).t(), ints([0, new]), ints([n]))
    want = ca.paged_window_attention(q, kp, vp, *where, prefix=ints([0]))
    for prefix in (-1, -5, -2 ** 31 + 1, -2 ** 31):
        assert torch.equal(ca.paged_window_attention(q, kp, vp, *where, prefix=ints([prefix])), want), prefix
