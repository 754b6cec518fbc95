"""CPU-side checks of the operators on token sequences: the 64-bit formulas against automatic differentiation, the
frequencies, and descriptors that are refused before any device work."""
import ctypes as C
import math

import pytest
import torch

from tests import tokens_reference as ref


@pytest.mark.parametrize("left,right,sinks,lengths", [(3, 0, 0, None), (2, 1, 2, [9, 0]), (None, 0, 0, [12, 5])])
def test_reference_gradients(left, right, sinks, lengths):
    g = torch.Generator().manual_seed(0)
    q, k, v, dy = (torch.randn(6, h, 12, 2, generator=g, dtype=torch.float64) for h in (4, 2, 2, 4))
    x = [t.clone().requires_grad_(True) for t in (q, k, v)]
    at = torch.arange(12)
    y = torch.zeros_like(q)
    for b in range(2):
        mask = ref.visible(at, at, 12 if lengths is None else lengths[b], left, right, sinks)
        for h in range(4):
            s = x[0][:, h, :, b].T @ x[1][:, h // 2, :, b] / math.sqrt(6)
            p = torch.exp(s) * mask
            y[:, h, :, b] = ((p / p.sum(1, keepdim=True).clamp(min=1e-300)) @ x[2][:, h // 2, :, b].T).T
    grads = torch.autograd.grad(y, x, dy)
    want = ref.window(q, k, v, left, right, sinks, lengths, dy=dy)
    for name, t in zip(("y", "dq", "dk", "dv"), (y, *grads)):
        assert torch.allclose(want[name][0], t.detach(), atol=1e-12), name


def test_turns(ca):
    turns = ca.rotary_turns(8, base=500.0, device="cpu")
    for p, t in enumerate(turns.tolist()):
        assert abs((t % 2 ** 64) / 2.0 ** 64 - 500.0 ** (-p / 8) / (2 * math.pi)) < 1e-16
    with pytest.raises(AssertionError, match="do not hold 8 pairs"):
        ca.rotary_turns(8, sections=(3, 4), device="cpu")
    with pytest.raises(AssertionError, match="must be positive"):
        ca.rotary_turns(0, device="cpu")


def _seq(ca, **kw):
    from circatt_b200._lib import ca_seq_desc
    base = dict(dtype=2, dim=64, heads_q=4, heads_kv=2, tokens=10, batch=2, left=3, right=0, sinks=0, scale=0.125)
    base.update(kw)
    return ca_seq_desc(**base)


def _views(ca, n, **kw):
    from circatt_b200._lib import ca_seq_view
    base = dict(data=256, head=64, token=256, batch=2560)       # never dereferenced: validation comes first
    base.update(kw)
    return [ca_seq_view(**base) for _ in range(n)]


@pytest.mark.parametrize("kw,code,msg", [
    (dict(dtype=1), -1, "dtype 1"),
    (dict(dim=60), -1, "multiples of 8 up to 128"),
    (dict(dim=136), -1, "multiples of 8 up to 128"),
    (dict(heads_q=3), -1, "positive multiple"),
    (dict(heads_kv=0), -1, "positive multiple"),
    (dict(tokens=-1), -1, "must not be negative"),
    (dict(right=-1), -1, "must not be negative"),
    (dict(sinks=-1), -1, "must not be negative"),
    (dict(batch=70000), -5, "grid limit"),
    (dict(tokens=2 ** 31 - 1), -5, "2^31 rows"),
])
def test_bad_descriptors(ca, kw, code, msg):
    lib = ca.lib
    assert lib.ca_window_fwd(_seq(ca, **kw), *_views(ca, 3), None, *_views(ca, 1), None, None, None) == code
    assert msg in lib.ca_last_error().decode()
    assert lib.ca_window_bwd_workspace(_seq(ca, **kw)) == 0


def test_bad_views_and_pages(ca):
    from circatt_b200._lib import ca_page_view, ca_pages, ca_rotary_desc
    lib, err = ca.lib, lambda: ca.lib.ca_last_error().decode()
    d = _seq(ca)
    good = _views(ca, 4)
    assert lib.ca_window_fwd(d, None, *good[:2], None, good[3], None, None, None) == -3 and "q is NULL" in err()
    assert lib.ca_window_fwd(d, _views(ca, 1, data=264)[0], *good[:2], None, good[3], None, None, None) == -1 and "16-byte" in err()
    assert lib.ca_window_fwd(d, _views(ca, 1, token=4)[0], *good[:2], None, good[3], None, None, None) == -1 and "stride" in err()
    assert lib.ca_window_fwd(d, _views(ca, 1, token=-256)[0], *good[:2], None, good[3], None, None, None) == -1 and "stride" in err()
    assert lib.ca_window_bwd(d, *_views(ca, 6), None, None, *_views(ca, 3), None, None) == -3 and "lse" in err()
    assert lib.ca_window_fwd(_seq(ca, tokens=0), *good[:3], None, good[3], None, None, None) == 0
    pool = ca_page_view(data=256, token=64, head=1024, page=2048)
    ok = dict(table=256, starts=256, lengths=256, width=4, page=16, pages=9, sequences=2)
    one = _seq(ca, batch=1)

    def paged(desc=one, **kw):
        return lib.ca_paged_window(desc, good[0], pool, pool, ca_pages(**{**ok, **kw}), good[1], None)
    assert paged(d) == -1 and "batch 1" in err()
    assert paged(_seq(ca, batch=1, right=2)) == -1 and "no later tokens" in err()
    assert paged(page=8) == -1 and "multiples of 16" in err()
    assert paged(sequences=0) == -1 and "no sequence" in err()
    assert paged(table=None) == -3 and "NULL" in err()
    assert paged(pages=-1) == -1
    base = dict(dtype=2, dim=64, pairs=32, axes=1, tokens=5, batch=1, positions=256, turns=256)

    def rotary(**kw):
        sections = (C.c_int32 * 4)(*kw.pop("sections", (32,)))
        return lib.ca_rotary(ca_rotary_desc(**{**base, **kw}, sections=sections), good[0], good[1], 4, None, None, 0, None)
    assert rotary(dim=60) == -1 and "multiples of 8" in err()
    assert rotary(pairs=33, sections=(33,)) == -1 and "do not fit" in err()
    assert rotary(axes=5) == -1 and "axes=5" in err()
    assert rotary(sections=(31,)) == -1 and "31 pairs" in err()
    assert rotary(axes=2, sections=(33, -1)) == -1 and "negative" in err()
    assert rotary(positions=None) == -3
    assert rotary(tokens=0) == 0


def test_views_without_data(ca):
    """A view of a call that has something to do holds an address: NULL is refused, not read."""
    from circatt_b200._lib import ca_page_view, ca_pages, ca_rotary_desc
    lib, err = ca.lib, lambda: ca.lib.ca_last_error().decode()
    d, one, good, none = _seq(ca), _seq(ca, batch=1), _views(ca, 9), _views(ca, 1, data=None)[0]
    for i, name in enumerate(("q", "k", "v", "y")):
        x = [none if j == i else good[j] for j in range(4)]
        assert lib.ca_window_fwd(d, *x[:3], None, x[3], None, None, None) == -3 and err().startswith(f"{name} has no data")
    assert lib.ca_window_fwd(_seq(ca, tokens=0), none, none, none, None, none, None, None, None) == 0
    for i, name in enumerate(("q", "k", "v", "y", None, "dy", "dq", "dk", "dv")):
        x = [none if j == i else good[j] for j in range(9)]
        if name:
            assert lib.ca_window_bwd(d, *x[:6], None, 256, *x[6:], 256, None) == -3 and err().startswith(f"{name} has no data")
    assert lib.ca_window_bwd(d, *good[:6], None, 256, *good[6:], 260, None) == -1 and "workspace is not 16-byte" in err()
    pool, gone = (ca_page_view(data=p, token=64, head=1024, page=2048) for p in (256, None))
    pages = ca_pages(table=256, starts=256, lengths=256, width=4, page=16, pages=9, sequences=2)
    for i, name in enumerate(("q", "k_pages", "v_pages", "y")):
        x = [good[0], pool, pool, good[1]]
        x[i] = gone if "pages" in name else none
        assert lib.ca_paged_window(one, *x[:3], pages, x[3], None) == -3 and err().startswith(f"{name} has no data")
    r = ca_rotary_desc(dtype=2, dim=64, pairs=32, axes=1, tokens=5, batch=1, positions=256, turns=256, sections=(C.c_int32 * 4)(32))
    for i, name in enumerate(("x1", "y1", "x2", "y2")):
        x = [none if j == i else good[j] for j in range(4)]
        assert lib.ca_rotary(r, *x[:2], 4, *x[2:], 2, None) == -3 and err().startswith(f"{name} has no data")
    for i, name in enumerate(("q", "q_out", "k", "v", "k_pages", "v_pages")):
        x = [*good[:4], pool, pool]
        x[i] = gone if "pages" in name else none
        assert lib.ca_rotary_append(r, *x[:2], 4, *x[2:4], 2, *x[4:], pages, None) == -3 and err().startswith(f"{name} has no data")


@pytest.mark.parametrize("dtype", [0, 2, 3])
@pytest.mark.parametrize("tokens,sinks,left,heads,batch", [(32768, 32768, 127, 8, 2), (32768, 4, 127, 64, 64), (1 << 20, 1 << 19, 255, 1, 1), (1000, 2 ** 31 - 1, 0, 2, 3)])
def test_scratch_memory_of_first_tokens_is_bounded(ca, dtype, tokens, sinks, left, heads, batch):
    """The backward's parts of key tiles with first tokens: at most 1024 of them, 128 keys and 128 features of dk and dv in
    Float32 each; apart from those a few numbers for every row."""
    d = _seq(ca, dtype=dtype, dim=128, heads_q=heads, heads_kv=heads, tokens=tokens, batch=batch, sinks=sinks, left=left)
    rows = tokens * heads * batch
    assert 4 * rows <= ca.lib.ca_window_bwd_workspace(d) <= 4 * rows + rows // 4 + 4096 + 1024 * 2 * 128 * 128 * 4
    few = _seq(ca, dtype=dtype, dim=128, heads_q=2, heads_kv=2, tokens=16384, batch=1, sinks=4, left=1023)
    assert ca.lib.ca_window_bwd_workspace(few) > 4 * 2 * 16384 + 2 * 8 * 64 * 128 * 4       # these are dealt out
