"""The example layer on a token stream: it trains, and serving it from a paged cache with freed pages gives what one call
gives."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example(ca):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "token_layer.py")
    spec = importlib.util.spec_from_file_location("token_layer", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=lambda d: str(d)[6:])
def test_serving_gives_what_one_call_gives(example, dtype):
    torch.manual_seed(1)
    layer = example.Layer().cuda()
    turns = layer.turns
    layer = layer.to(dtype)
    layer.turns = turns
    x = torch.randn(420, 256, device="cuda", dtype=dtype).t()
    with torch.no_grad():
        whole = layer(x[..., None])[..., 0].float()
    got = example.serve(layer, x, [200, 1, 1, 90] + [1] * 128).float()
    # both round the same intermediate results once more or less; Float32: sums in another order
    assert float((got - whole).norm() / whole.norm()) < {torch.float32: 1e-5, torch.bfloat16: 2e-2, torch.float16: 2.5e-3}[dtype]


def test_training_goes_down(example):
    torch.manual_seed(2)
    layer = example.Layer().cuda()
    losses = example.train(layer, steps=60, N=300, B=2)
    assert losses[-1] < 0.9 * losses[0]
