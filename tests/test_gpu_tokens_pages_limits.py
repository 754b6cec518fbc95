"""The pages of a cache where sequences outgrow their table, or are made shorter into pages that others hold."""
import pytest
import torch

from tests.test_gpu_tokens_pages import columns, ints

pytestmark = pytest.mark.gpu


def test_tokens_beyond_the_table(ca):
    """Places of the table get pages; tokens without a place change nothing, and what a caller stores there is not stored."""
    D, page, width = 64, 16, 3
    table, refs = columns([[0, -1, -1], [1, 2, -1]], width), ints([1, 1, 1, 0, 0, 0])
    starts, lengths = ints([0, 50, 90]), ints([60, 70])               # 4 and 5 pages of tokens
    table, refs, missing = ca.advance_pages(table, refs, starts, lengths, page)
    assert table.t().tolist() == [[0, 3, 4], [1, 2, 5]] and refs.tolist() == [1] * 6 and missing.item() == 0
    k = torch.ones(90, 1, D, device="cuda").permute(2, 1, 0)
    pools = [torch.zeros(6, 1, page, D, device="cuda").permute(3, 2, 1, 0) for _ in range(2)]
    ca.rotary_append_(k, k, k, *pools, table, starts, lengths, torch.zeros(1, 90, dtype=torch.int32, device="cuda"), ca.rotary_turns(D // 2))
    filled = (pools[1][0, :, 0] != 0).t().int()                       # (pages, places)
    assert filled[0].tolist() == [0] * 10 + [1] * 6 and filled[1].sum() == 0       # new tokens from 10 and from 30 on
    assert filled[3].all() and filled[4].all() and filled[5].all() and filled[2].tolist() == [0] * 14 + [1] * 2


def test_shorter_sequences_and_shared_pages(ca):
    """Two sequences hold the same full pages.  One is made shorter and forked: the copy ends in a page of its own, and what is
    appended to it leaves the others' tokens alone."""
    D, page = 64, 16
    pool = torch.arange(8, dtype=torch.float32, device="cuda")[:, None, None, None].expand(8, 1, page, D).contiguous().permute(3, 2, 1, 0)
    table, refs, lengths = columns([[0, 1, 2], [0, 1, 3], [-1] * 3], 3), ints([2, 2, 1, 1, 0, 0, 0, 0]), ints([40, 40, 0])
    lengths = lengths - ints([0, 18, 0])                              # the second ends at 22, within page 1
    table, refs, lengths, missing = ca.fork_pages([pool], table, refs, lengths, ints([0, 1, 1]))
    assert table.t().tolist() == [[0, 1, 2], [0, 1, 3], [0, 4, -1]] and missing.item() == 0
    assert refs.tolist() == [3, 2, 1, 1, 1, 0, 0, 0] and lengths.tolist() == [40, 22, 22]
    # the copy goes on, the shorter one ends
    starts, lengths = ints([0, 0, 0, 4]), ints([40, 0, 26])
    table, refs, missing = ca.advance_pages(table, refs, starts, lengths, page)
    assert table.t().tolist() == [[0, 1, 2], [-1] * 3, [0, 4, -1]] and refs.tolist() == [2, 1, 1, 0, 1, 0, 0, 0]
    x = torch.full((4, 1, D), 9.0, device="cuda").permute(2, 1, 0)
    ca.rotary_append_(x, x, x, pool, pool, table, starts, lengths, torch.zeros(1, 4, dtype=torch.int32, device="cuda"), ca.rotary_turns(D // 2))
    assert (pool[..., 1] == 1).all() and pool[0, :, 0, 4].tolist() == [1.0] * 6 + [9.0] * 4 + [1.0] * 6
