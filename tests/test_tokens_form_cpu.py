"""CPU-side checks of attention with other scores and masks: its 64-bit formulas against automatic differentiation, and calls that
are refused before any device work."""
import math

import pytest
import torch

from tests import tokens_form_reference as ref
from tests.test_tokens_cpu import _seq, _views


@pytest.mark.parametrize("cap,slopes,left,sinks,documents,groups", [
    (2.0, [0.3, 0.1], None, 0, [0, 0, 0, 5, 5, -1, 5, 5, 5, 5], [1, 1, 0, 0, 2, 0, 0, 3, 3, 0]),
    (None, [0.5, 0.0], 3, 1, None, None),
    (0.7, None, None, 0, [1] * 10, None),
])
def test_reference_gradients(cap, slopes, left, sinks, documents, groups):
    g = torch.Generator().manual_seed(1)
    q, k, v, dy = (torch.randn(6, h, 10, 1, generator=g, dtype=torch.float64).float() for h in (2, 1, 1, 2))
    want = ref.window(q, k, v, left, 0, sinks, None, cap, slopes, documents and [documents], groups and [groups], dy)
    x = [t.double().requires_grad_(True) for t in (q, k, v)]
    y = torch.zeros(6, 2, 10, 1, dtype=torch.float64)
    for h in range(2):
        for i in range(10):
            seen = []
            for j in range(10):
                if documents is None:
                    on = j <= i
                else:
                    low, high = min(i, j), max(i, j)
                    same = all(documents[a] == documents[i] for a in range(low, high + 1)) and documents[i] >= 0
                    both = groups is not None and groups[i] > 0 and all(groups[a] == groups[i] for a in range(low, high + 1))
                    on = same and (j <= i or both)
                if on and (left is None or j >= i - left or j < sinks):
                    seen.append(j)
            if not seen:
                continue
            s = torch.stack([(x[0][:, h, i, 0] * x[1][:, 0, j, 0]).sum() / math.sqrt(6) for j in seen])
            s = cap * torch.tanh(s / cap) if cap else s
            s = s - (slopes[h] if slopes else 0.0) * torch.tensor([abs(i - j) for j in seen])
            y[:, h, i, 0] = (torch.softmax(s, 0)[None] * x[2][:, 0, seen, 0]).sum(1)
    grads = torch.autograd.grad(y, x, dy.double())
    for name, t in zip(("y", "dq", "dk", "dv"), (y, *grads)):
        assert torch.allclose(want[name][0], t.detach(), atol=1e-12), name


def _form(**kw):
    from circatt_b200._lib import ca_seq_form
    return ca_seq_form(**{**dict(cap=0.0, slopes=None, spans=None, prefix=None), **kw})


@pytest.mark.parametrize("form,desc,msg", [
    (dict(cap=-1.0), {}, "cap must be positive"),
    (dict(cap=math.inf), {}, "cap must be positive"),
    (dict(cap=math.nan), {}, "cap must be positive"),
    (dict(cap=1e-40), {}, "too small"),
    (dict(cap=3e38), {}, "too large"),
    (dict(spans=264), {}, "not aligned"),
    (dict(slopes=258), {}, "not aligned"),
    (dict(prefix=256), {}, "a dense call takes spans"),
    (dict(spans=256), dict(right=1), "spans say what a token sees"),
    (dict(spans=256), dict(sinks=2), "spans say what a token sees"),
])
def test_bad_forms(ca, form, desc, msg):
    lib, views = ca.lib, _views(ca, 9)
    d = _seq(ca, **desc)
    assert lib.ca_window_form_fwd(d, _form(**form), *views[:3], None, views[3], None, None, None) == -1
    assert msg in lib.ca_last_error().decode()
    assert lib.ca_window_form_bwd(d, _form(**form), *views[:6], None, 256, *views[6:], 256, None) == -1
    assert msg in lib.ca_last_error().decode()


def test_bad_calls(ca):
    from circatt_b200._lib import ca_page_view, ca_pages
    lib, err, views = ca.lib, lambda: ca.lib.ca_last_error().decode(), _views(ca, 4)
    pool = ca_page_view(data=256, token=64, head=1024, page=2048)
    pages = ca_pages(table=256, starts=256, lengths=256, width=4, page=16, pages=9, sequences=2)
    one = _seq(ca, batch=1)
    assert lib.ca_paged_window_form(one, _form(spans=256), views[0], pool, pool, pages, views[1], None) == -1 and "dense" in err()
    assert lib.ca_window_form_fwd(_seq(ca, tokens=0), _form(cap=2.0), *views[:3], None, views[3], None, None, None) == 0
    assert lib.ca_window_form_fwd(_seq(ca, dim=60), _form(cap=2.0), *views[:3], None, views[3], None, None, None) == -1 and "multiples of 8" in err()
    assert lib.ca_token_spans(256, None, -1, 1, 256, None) == -1 and "negative" in err()
    assert lib.ca_token_spans(256, None, 5, 70000, 256, None) == -5 and "grid limit" in err()
    assert lib.ca_token_spans(None, None, 5, 1, 256, None) == -3 and "NULL" in err()
    assert lib.ca_token_spans(256, None, 5, 1, None, None) == -3
    assert lib.ca_token_spans(256, None, 5, 1, 264, None) == -1 and "not aligned" in err()
    assert lib.ca_token_spans(None, None, 0, 1, None, None) == 0


def test_cpu_tensors_are_refused(ca):
    q = torch.zeros(1, 5, 2, 64).permute(3, 2, 1, 0)
    with pytest.raises(RuntimeError, match="only CUDA"):
        ca.window_attention(q, q, q, 3, cap=5.0)
    with pytest.raises(RuntimeError, match="only CUDA"):
        ca.token_spans(torch.zeros(5, dtype=torch.int32))
