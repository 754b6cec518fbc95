"""Tables and counts beyond what the page kernels' indices hold, refused before any device work."""
import pytest

from tests.test_tokens_pages_cpu import _pool, _table


@pytest.mark.parametrize("kw", [dict(pages=2 ** 30 + 1), dict(pages=2 ** 31 - 1), dict(sequences=2 ** 30 + 1), dict(sequences=2 ** 31 - 1, width=0)])
def test_too_many(ca, kw):
    lib, t = ca.lib, _table(**kw)
    for code in (lib.ca_advance_pages(t, 256, -1, 0, 1024, 2048, 4096, 8192, None), lib.ca_fork_pages(t, 256, _pool(), 1, 1024, 2048, 3584, 4096, 8192, None),
                 lib.ca_compact_pages(t, _pool(), 1, 1024, 2048, 4096, 8192, None)):
        assert code == -5 and "2^30" in lib.ca_last_error().decode()
    assert lib.ca_pages_workspace(t) == 0


def test_largest(ca):
    assert ca.lib.ca_pages_workspace(_table(pages=2 ** 30, sequences=3)) >= 12 * 2 ** 30
