"""An attention layer on a token stream, trained and served with the same operators.

    python examples/token_layer.py

The layer is: projections, rotary positions, attention with a sliding window and a few first tokens that stay visible, output
projection.  `train` fits it to the mean of the tokens in its window, `serve` runs it over a paged cache, a prompt in chunks and
then token by token, freeing the pages that the window has left, and the two agree."""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from __graft_entry__ import load_package  # noqa: E402

ca = load_package()

D, HEADS, KEY_HEADS, WINDOW, SINKS, PAGE = 64, 8, 2, 127, 4, 16


class Layer(torch.nn.Module):
    """Tokens (model, N, B) in the package's column-major layout, like every tensor here."""

    def __init__(self, model=256):
        super().__init__()
        self.qkv = torch.nn.Linear(model, (HEADS + 2 * KEY_HEADS) * D, bias=False)
        self.out = torch.nn.Linear(HEADS * D, model, bias=False)
        self.register_buffer("turns", ca.rotary_turns(D // 2))

    def heads(self, x):
        """q, k, v (D, heads, N, B): slices of one projection, taken as they lie."""
        y = self.qkv(x.permute(2, 1, 0)).unflatten(-1, (HEADS + 2 * KEY_HEADS, D)).permute(3, 2, 1, 0)
        return y[:, :HEADS], y[:, HEADS:HEADS + KEY_HEADS], y[:, HEADS + KEY_HEADS:]

    def merge(self, y):
        return self.out(y.permute(*range(y.ndim - 1, -1, -1)).flatten(-2)).permute(*range(y.ndim - 2, -1, -1))

    def forward(self, x, lengths=None):
        q, k, v = self.heads(x)
        positions = torch.arange(x.shape[1], dtype=torch.int32, device=x.device)[None]
        q, k = ca.rotary((q, k), positions, self.turns)
        return self.merge(ca.window_attention(q, k, v, WINDOW, sinks=SINKS, lengths=lengths))

    @torch.no_grad()
    def step(self, x, cache):
        """New tokens (model, T) of one sequence: their keys and values enter the cache, then they attend to it."""
        q, k, v = (t[..., 0] for t in self.heads(x[..., None]))
        positions = cache.grow(x.shape[1])
        where = (cache.table, cache.starts, cache.lengths)
        q = ca.rotary_append_(q, k, v, cache.k, cache.v, *where, positions, self.turns)
        return self.merge(ca.paged_window_attention(q, cache.k, cache.v, *where, WINDOW, sinks=SINKS))


class Cache:
    """Pages for one sequence.  Each step gives back those that the window has left and takes some for the new tokens; where a
    step's pages are is known on the device only."""

    def __init__(self, pages, width, dtype, device="cuda"):
        self.k, self.v = (ca.jl.empty((D, PAGE, KEY_HEADS, pages), dtype, device) for _ in range(2))
        self.table = torch.full((1, width), -1, dtype=torch.int32, device=device).t()
        self.refs = torch.zeros(pages, dtype=torch.int32, device=device)
        self.total, self.device = 0, device

    def grow(self, n):
        at, self.total = self.total, self.total + n
        self.starts = torch.tensor([0, n], dtype=torch.int32, device=self.device)
        self.lengths = torch.tensor([self.total], dtype=torch.int32, device=self.device)
        self.table, self.refs, _ = ca.advance_pages(self.table, self.refs, self.starts, self.lengths, PAGE, WINDOW, sinks=SINKS)
        return torch.arange(at, self.total, dtype=torch.int32, device=self.device)[None]


def train(layer, steps=60, N=500, B=4, device="cuda"):
    """Regression onto the mean of the last WINDOW + 1 tokens (times 8: of about unit size).  Returns the losses."""
    optimizer = torch.optim.Adam(layer.parameters(), lr=5e-3)
    losses = []
    model = layer.qkv.in_features
    for step in range(steps):
        g = torch.Generator(device=device).manual_seed(step)
        x = torch.randn(B, N, model, device=device, dtype=layer.qkv.weight.dtype, generator=g).permute(2, 1, 0)
        total = torch.cumsum(x, 1)
        mean = (total[:, WINDOW + 1:] - total[:, :-WINDOW - 1]) / (WINDOW + 1)
        loss = (layer(x)[:, WINDOW + 1:] - 8 * mean).float().square().mean()
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.item())
    return losses


def serve(layer, x, chunks, pages=40):
    """The outputs of one sequence (model, N) from the cache, `chunks` tokens at a time."""
    cache, parts, at = Cache(pages, -(-x.shape[1] // PAGE), x.dtype, x.device), [], 0
    for n in chunks:
        parts.append(layer.step(x[:, at:at + n], cache))
        at += n
    return torch.cat(parts, 1)


def main():
    torch.manual_seed(0)
    layer = Layer().cuda()
    losses = train(layer)
    print(f"loss {losses[0]:.4f} -> {losses[-1]:.4f}")
    for dtype in (torch.float32, torch.bfloat16):
        served = Layer().cuda().to(dtype)
        served.load_state_dict({k: v for k, v in layer.state_dict().items()})
        served.turns = layer.turns
        x = torch.randn(700, 256, device="cuda", dtype=dtype).t()
        with torch.no_grad():
            whole = served(x[..., None])[..., 0]
        got = serve(served, x, [300, 100, 50] + [1] * 250)
        off = float((got - whole).float().norm() / whole.float().norm())
        print(f"{str(dtype)[6:]}: cache against one call, relative difference {off:.2g}")
        assert off < (1e-5 if dtype is torch.float32 else 2e-2)


if __name__ == "__main__":
    main()
