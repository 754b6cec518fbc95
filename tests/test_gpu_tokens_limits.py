"""Attention on token sequences where sizes and numbers reach the limits of what the kernels' choices assume: values of unequal
size in half precision, windows behind a cache's table, several devices in
one process, tokens of no sequence, infinities next to rows that see nothing,
many first tokens."""
import math
import random

import pytest
import torch

from tests import tokens_reference as ref
from tests.test_gpu_tokens_paged import cache, ints
from tests.test_gpu_tokens_window import DTYPES, compare, make, problem, run

pytestmark = pytest.mark.gpu


def name_of(dtype):
    return str(dtype)[6:]


def sm_count():
    return torch.cuda.get_device_properties(0).multi_processor_count


@pytest.mark.parametrize("left,sinks", [(None, 0), (150, 4)])
@pytest.mark.parametrize("at", [0, 2, 3])
@pytest.mark.parametrize("ratio", [2.0 ** -8, 2.0 ** -14])
@pytest.mark.parametrize("D", [64, 128])
def test_values_of_unequal_size_in_half_precision(ca, D, ratio, at, left, sinks):
    """128 keys whose values are much smaller than those of the keys next to them: dS of those keys is made of the others'
    values, through the rows' sums."""
    N = 512
    q, k, v, dy = problem(D, 2, 1, N, 1, torch.float64)
    v, dy = 1 + 0.3 * v, 1 + 0.3 * dy
    v[:, :, 128 * at:128 * at + 128] *= ratio
    q, k, v, dy = (t.to(torch.float16) for t in (q, k, v, dy))
    got = run(ca, q, k, v, dy, left, 0, sinks)
    want = ref.window(q.double(), k.double(), v.double(), left, 0, sinks, None, None, dy.double(), ref.UNIT[torch.float16])
    for name, (x, e) in want.items():
        ref.check(got[name], x, e + 2.0 ** -24, name)       # results below the smallest normal half: multiples of 2^-24


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
@pytest.mark.parametrize("left,sinks", [(60, 0), (60, 20), (60, 400), (0, 0), (None, 0)])
@pytest.mark.parametrize("D,G,S,new", [
    (64, 2, 4, 1),                  # few rows a key head
    (64, 4, 4, 150),                # one row tile, two streams over its keys
    (128, 3, 3, 150),
    (64, 1, 80, 150),               # two row tiles that share the key tiles
    (128, 4, 40, 70),
])
def test_windows_behind_the_table(ca, D, G, S, new, left, sinks, dtype):
    """Lengths beyond the places of the table: windows that lie behind it wholly, or those of the last rows only.  Such rows see
    first tokens or nothing at all, and nothing gives zeros."""
    page, width, Hkv = 16, 9, 2                                                          # 144 places: not whole tiles of keys
    lengths = [(1000, 290, 160, 204, 140 + new, 144)[s % 6] for s in range(S)]
    if S > 4:
        assert (S * new * G // 256 + S) * Hkv >= sm_count() and new * G > 128
    order = list(range(S * width))
    random.Random(1).shuffle(order)
    table = [order[width * s:width * s + width] for s in range(S)]
    starts = [new * s for s in range(S + 1)]
    q = make(9, (D, Hkv * G, S * new), dtype, 1.5)
    kp, vp = (make(i, (D, page, Hkv, S * width), dtype) for i in (1, 2))
    args = (q.cuda(), kp.cuda(), vp.cuda(), ints(table).t(), ints(starts), ints(lengths), left)
    want, bound = ref.paged(q.double(), kp.double(), vp.double(), table, starts, lengths, left, sinks, u=ref.UNIT[dtype])
    for _ in range(3):
        y = ca.paged_window_attention(*args, sinks=sinks)
        ref.check(y, want, bound)
        assert y[:, :, :new].any() == (sinks > 0 or left is None)                        # the first sequence's length is 1000
    ca.ops.check_status()


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
def test_decoding_on_every_device(ca, dtype):
    """Few sequences take the largest clusters, which a kernel has to be allowed on each device (two where there are two)."""
    devices = [f"cuda:{i}" for i in range(min(2, torch.cuda.device_count()))]
    page, width, S, Hkv = 16, 64, 4, 4
    table = [list(range(width * s, width * s + width)) for s in range(S)]
    starts, lengths = list(range(S + 1)), [1024, 900, 17, 333]
    q = make(9, (128, 16, S), dtype, 1.5)
    kp, vp = (make(i, (128, page, Hkv, S * width), dtype) for i in (1, 2))
    want, bound = ref.paged(q.double(), kp.double(), vp.double(), table, starts, lengths, None, 0, u=ref.UNIT[dtype])
    for device in devices * 2:
        at = [t.to(device) for t in (q, kp, vp, ints(table).t(), ints(starts), ints(lengths))]
        ref.check(ca.paged_window_attention(*at), want, bound)


@pytest.mark.parametrize("new,S", [(1, 2), (150, 2), (150, 80)])
@pytest.mark.parametrize("D,G", [(64, 1), (64, 3), (128, 4), (24, 2)])
@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
def test_tokens_of_no_sequence(ca, dtype, D, G, new, S):
    """Packed tokens before the first sequence and behind the last, as in a call of fixed size that is not full: zeros,
    whatever the result's memory held."""
    total = max(new, 160)
    kp, vp, table = cache(D, 2, 16, [(new, total)] * S, dtype, 60, 3)
    for lead, tail in ((0, 9), (4, 700), (0, 0)):
        starts, T = [lead + new * s for s in range(S + 1)], lead + new * S + tail
        q = make(9, (D, 2 * G, T), dtype, 1.5)
        torch.full((T, 2 * G, D), math.nan, dtype=dtype, device="cuda")        # freed at once: the result's place
        y = ca.paged_window_attention(q.cuda(), kp.cuda(), vp.cuda(), ints(table).t(), ints(starts), ints([total] * S), 60, sinks=3)
        want, bound = ref.paged(q.double(), kp.double(), vp.double(), table, starts, [total] * S, 60, 3, u=ref.UNIT[dtype])
        ref.check(y, want, bound)
        assert not y[:, :, :lead].any() and not y[:, :, T - tail:].any()


@pytest.mark.parametrize("junk", [math.inf, math.nan])
@pytest.mark.parametrize("which", range(4), ids=("q", "k", "v", "dy"))
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
def test_zeros_behind_the_length_next_to_infinity(ca, dtype, D, which, junk):
    """The last token of a sequence is not finite, and the places behind it share its tiles: they are zeros all the same, and
    the other sequence is not touched."""
    x = list(problem(D, 4, 2, 300, 2, dtype))
    x[which][:, :, 130, 0] = junk
    for left, sinks in ((50, 3), (None, 0)):
        for name, t in run(ca, *x, left, 0, sinks, [131, 300]).items():
            assert not t[:, :, 131:, 0].any(), name
            assert torch.isfinite(t[..., 1]).all(), name


@pytest.mark.parametrize("new", [5, 150])
@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
def test_zeros_of_rows_that_see_nothing_next_to_infinity(ca, dtype, new):
    """More tokens are new than the cache is said to hold: the first two see nothing, the others see values that are infinite."""
    kp, vp, table = cache(64, 2, 16, [(new - 2, new - 2)], dtype, None, 0, junk=0.5)
    vp[..., table[0][0]] = math.inf
    q = make(9, (64, 4, new), dtype, 1.5)
    y = ca.paged_window_attention(q.cuda(), kp.cuda(), vp.cuda(), ints(table).t(), ints([0, new]), ints([new - 2]))
    assert not y[:, :, :2].any() and not torch.isfinite(y[:, :, 2:]).any()


@pytest.mark.parametrize("dtype", DTYPES, ids=name_of)
@pytest.mark.parametrize("D,Hq,Hkv,N,B,left,sinks,lengths", [
    (64, 2, 1, 4000, 1, 31, 4, None),                # one tile's queries, dealt to many CTAs
    (128, 2, 1, 4000, 1, 31, 130, [3001]),
    (64, 8, 8, 1000, 10, 20, 300, None),             # some tiles, to fewer
    (64, 16, 16, 600, 9, 20, 590, None),             # all tiles: each has its CTA
])
def test_many_first_tokens(ca, D, Hq, Hkv, N, B, left, sinks, lengths, dtype):
    q, k, v, dy = problem(D, Hq, Hkv, N, B, dtype)
    got = run(ca, q, k, v, dy, left, 0, sinks, lengths)
    compare(got, q, k, v, dy, left, 0, sinks, lengths)
