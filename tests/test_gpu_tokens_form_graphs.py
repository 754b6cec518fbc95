"""Captured calls of attention with other scores, whose kernels may begin under the one before: behind a copy, a fill, nothing at all,
and two streams that join."""
import pytest
import torch

from tests.test_gpu_tokens_form import slopes_of
from tests.test_gpu_tokens_window import make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("before", ["nothing", "copy", "fill", "join"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=lambda d: str(d)[6:])
def test_what_stands_before_a_captured_call(ca, dtype, before):
    q, k, v = (make(i, (64, h, 700, 2), dtype, s).cuda() for i, h, s in ((0, 4, 3.0), (1, 2, 1.0), (2, 2, 1.0)))
    other = make(5, (64, 2, 700, 2), dtype).cuda()
    slopes = slopes_of(4).cuda()
    side = torch.cuda.Stream()

    def attend(x):
        return ca.window_attention(q, x, v, 300, cap=20.0, slopes=slopes)

    def step():
        if before == "copy":
            k.copy_(other)
        elif before == "fill":
            k[..., 1].zero_()
        elif before == "join":
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                x = other * 0.5
            k.mul_(0.5)
            torch.cuda.current_stream().wait_stream(side)
            return attend(x)
        return attend(k)
    start = k.clone()
    want = step()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        got = step()
    for _ in range(3):
        k.copy_(start)
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    ca.ops.check_status()
