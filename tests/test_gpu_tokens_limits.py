"""Attention on token sequences where sizes and numbers reach the limits of what the kernels' choices assume: values of unequal
size in half precision."""
import pytest
import torch

from tests import tokens_reference as ref
from tests.test_gpu_tokens_window import problem, run

pytestmark = pytest.mark.gpu


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
