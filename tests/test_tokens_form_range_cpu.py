"""Caps at the ends of Float32, refused before any device work."""
import pytest

from tests.test_tokens_cpu import _seq, _views
from tests.test_tokens_form_cpu import _form


@pytest.mark.parametrize("cap,scale,msg", [
    (1.3e30, 0.125, "too large"),               # scores below cap 2^-126 would be zeros
    (1e37, 0.125, "too large"),
    (1e38, 0.125, "too large"),
    (1e20, 1e-20, "too large for scale"),       # scale / cap is zero on the device
    (1e20, -1e-20, "too large for scale"),
    (1.25e30, 0.125, None),
    (1.25e30, 0.0, None),
    (1e20, 1e-17, None),
    (50.0, 1e-39, None),                        # a scale that is zero without a cap too
])
def test_large_caps(ca, cap, scale, msg):
    lib, views, d = ca.lib, _views(ca, 9), _seq(ca, tokens=0, scale=scale)
    code = 0 if msg is None else -1
    assert lib.ca_window_form_fwd(d, _form(cap=cap), *views[:3], None, views[3], None, None, None) == code
    assert msg is None or msg in lib.ca_last_error().decode()
    assert lib.ca_window_form_bwd(d, _form(cap=cap), *views[:6], None, 256, *views[6:], 256, None) == code
    assert msg is None or msg in lib.ca_last_error().decode()
