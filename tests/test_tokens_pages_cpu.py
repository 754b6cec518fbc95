"""Calls on the pages of a cache that are refused before any device work."""
import pytest
import torch


def _table(**kw):
    from circatt_b200._lib import ca_table
    return ca_table(**{**dict(table=256, refs=512, lengths=768, width=4, sequences=3, page=16, pages=20), **kw})


def _pool(**kw):
    from circatt_b200._lib import ca_pool
    return ca_pool(**{**dict(data=256, token=128, head=2048, page=4096, row=128, tokens=16, heads=2), **kw})


BAD_TABLES = [
    (dict(page=8), -1, "multiples of 16 tokens"),
    (dict(page=0), -1, "multiples of 16 tokens"),
    (dict(width=-1), -1, "must not be negative"),
    (dict(sequences=-1), -1, "must not be negative"),
    (dict(pages=-1), -1, "must not be negative"),
    (dict(width=2 ** 28), -5, "2^31 tokens"),
    (dict(table=None), -3, "must not be NULL"),
    (dict(refs=None), -3, "must not be NULL"),
]


@pytest.mark.parametrize("kw,code,msg", BAD_TABLES)
def test_bad_tables(ca, kw, code, msg):
    lib, err = ca.lib, lambda: ca.lib.ca_last_error().decode()
    t = _table(**kw)
    assert lib.ca_advance_pages(t, 256, -1, 0, 1024, 2048, 4096, 8192, None) == code and msg in err()
    assert lib.ca_fork_pages(t, 256, _pool(), 1, 1024, 2048, 3584, 4096, 8192, None) == code and msg in err()
    assert lib.ca_compact_pages(t, _pool(), 1, 1024, 2048, 4096, 8192, None) == code and msg in err()
    assert lib.ca_pages_workspace(t) == 0


def test_workspace(ca):
    assert ca.lib.ca_pages_workspace(_table(pages=1000, sequences=30)) >= 4 * 1000


@pytest.mark.parametrize("kw,code,msg", [
    (dict(data=None), -3, "no data"),
    (dict(data=264), -1, "multiples of 16 bytes"),
    (dict(token=136), -1, "multiples of 16 bytes"),
    (dict(head=-2048), -1, "not negative"),
    (dict(row=120), -1, "rows of 120 bytes"),
    (dict(row=0), -1, "rows of 0 bytes"),
    (dict(heads=0), -1, "0 heads"),
    (dict(tokens=32), -1, "pages of 32 tokens"),
])
def test_bad_pools(ca, kw, code, msg):
    lib, err = ca.lib, lambda: ca.lib.ca_last_error().decode()
    assert lib.ca_fork_pages(_table(), 256, _pool(**kw), 1, 1024, 2048, 3584, 4096, 8192, None) == code and msg in err()
    assert lib.ca_compact_pages(_table(), _pool(**kw), 1, 1024, 2048, 4096, 8192, None) == code and msg in err()


def test_bad_results(ca):
    lib, err, t, pool = ca.lib, lambda: ca.lib.ca_last_error().decode(), _table(), _pool()
    assert lib.ca_advance_pages(None, 256, -1, 0, 1024, 2048, 4096, 8192, None) == -3 and "table is NULL" in err()
    assert lib.ca_advance_pages(t, None, -1, 0, 1024, 2048, 4096, 8192, None) == -3 and "starts" in err()
    assert lib.ca_advance_pages(t, 256, -1, -1, 1024, 2048, 4096, 8192, None) == -1 and "sinks=-1" in err()
    assert lib.ca_advance_pages(_table(lengths=None), 256, -1, 0, 1024, 2048, 4096, 8192, None) == -3
    for x in ((None, 2048, 4096, 8192), (1024, None, 4096, 8192), (1024, 2048, None, 8192), (1024, 2048, 4096, None)):
        assert lib.ca_advance_pages(t, 256, -1, 0, *x, None) == -3 and "must not be NULL" in err()
        assert lib.ca_compact_pages(t, pool, 1, *x, None) == -3 and "must not be NULL" in err()
    assert lib.ca_advance_pages(t, 256, -1, 0, 256, 2048, 4096, 8192, None) == -1 and "old one's place" in err()
    assert lib.ca_advance_pages(t, 256, -1, 0, 1024, 512, 4096, 8192, None) == -1 and "old ones' place" in err()
    assert lib.ca_advance_pages(t, 256, -1, 0, 1024, 2048, 4096, 8200, None) == -1 and "16-byte aligned" in err()
    assert lib.ca_fork_pages(t, None, pool, 1, 1024, 2048, 3584, 4096, 8192, None) == -3 and "parents" in err()
    assert lib.ca_fork_pages(t, 256, None, 1, 1024, 2048, 3584, 4096, 8192, None) == -3 and "without pools" in err()
    assert lib.ca_fork_pages(t, 256, pool, 1, 1024, 2048, 768, 4096, 8192, None) == -1 and "lengths" in err()


def test_cpu_tensors_are_refused(ca):
    table, refs, n = torch.zeros(2, 1, dtype=torch.int32), torch.zeros(4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    pool = torch.zeros(4, 1, 16, 8).permute(3, 2, 1, 0)
    for call in (lambda: ca.advance_pages(table, refs, torch.zeros(2, dtype=torch.int32), n, 16), lambda: ca.fork_pages([pool], table, refs, n, n),
                 lambda: ca.compact_pages([pool], table, refs)):
        with pytest.raises(RuntimeError, match="only CUDA"):
            call()
