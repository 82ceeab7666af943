"""Page bookkeeping of sequences that have given pages up behind a window, and of rejected drafts."""
from __future__ import annotations

import pytest
import torch

import attn_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


def consistent(c):
    """refs count the table entries; entries behind a sequence's last page name none."""
    tables, lens, n = c.tables.tolist(), c.lens.tolist(), len(c.refs)
    held = [p for row in tables for p in row if p >= 0]
    assert [held.count(p) for p in range(n)] == c.refs.tolist()
    for row, m in zip(tables, lens):
        assert all(p < 0 for p in row[-(-m // c.page_size):])


@pytest.mark.parametrize("ps", [16, 32, 64, 128])
def test_a_fork_that_ends_inside_a_page_given_up_is_refused(ps):
    """The child would count that page as its own: the tokens that grow has room for would lie in
    no page.  What the fork grants, grow can go on with."""
    from paris_moe_b200 import PagedKVCache
    c = PagedKVCache(60, ps, 2, 1, 64, 8, 9 * ps)
    assert c.grow([0], [6 * ps + 4]).tolist() == [1]
    c.free([0], window=ps + 4)                     # pages 0 to 4
    assert (c.tables[0] >= 0).tolist() == [False] * 5 + [True] * 2 + [False] * 2
    before = c.refs.clone()
    keep = [2 * ps + 8, 2 * ps, 5 * ps + 3, 1, 6 * ps + 4, 5 * ps - 1]
    dst = [1, 2, 3, 4, 5, 6]
    ok = c.fork([0] * 6, dst, keep)
    assert ok.tolist() == [0, 1, 1, 0, 1, 0]
    assert c.lens.tolist() == [6 * ps + 4, 0, 2 * ps, 5 * ps + 3, 0, 6 * ps + 4, 0, 0]
    for d in (1, 2, 4, 6):
        assert (c.tables[d] < 0).all()
    # the two granted tails took a fresh page each, the full page 5 is shared once
    assert int(c.refs.sum() - before.sum()) == 3
    consistent(c)
    old = c.lens.tolist()
    assert c.grow(dst, [ps + 4] * 6).tolist() == [1] * 6
    for d in dst:
        for j in range(old[d], old[d] + ps + 4):
            assert int(c.tables[d, j // ps]) >= 0, (d, j)
    consistent(c)


def test_a_fork_whose_last_page_is_not_in_the_pool_is_refused():
    from paris_moe_b200 import PagedKVCache
    c = PagedKVCache(10, 16, 1, 1, 64, 4, 64)
    c.grow([0], [40])
    last = c.tables[0, 2].clone()
    for entry in (-1, 10, -2 ** 31, 2 ** 31 - 1):
        c.tables[0, 2] = entry
        assert c.fork([0, 0], [1, 2], [33, 32]).tolist() == [0, 1]
        assert c.lens.tolist() == [40, 0, 32, 0] and int(c.refs.sum()) == 5
        c.free([2])
    c.tables[0, 2] = last
    assert c.fork([0], [1]).tolist() == [1]


def test_rejected_drafts_are_given_back_by_forking_what_stays():
    """Lengths only grow; a sequence is shortened by forking the tokens that stay into an empty slot
    and freeing the old one.  No page is lost, and the keys that stay are the same."""
    from paris_moe_b200 import PagedKVCache
    g = torch.Generator().manual_seed(1)
    c = PagedKVCache(40, 16, 2, 1, 64, 4, 160)
    c.pages.copy_(torch.randn(c.pages.shape, generator=g))
    one = lambda s, n: c.k(1)[c.tables[s, :-(-n // 16)].long(), 0].reshape(-1, 64)[:n].clone()  # noqa: E731
    slot, spare, n = 0, 1, 30
    assert c.grow([slot], [n]).tolist() == [1]
    for accepted in (0, 1, 2, 5, 5, 3, 0, 4):
        assert c.grow([slot], [5]).tolist() == [1]            # five drafted tokens
        kept = one(slot, n + accepted)
        if accepted < 5:
            assert c.fork([slot], [spare], [n + accepted]).tolist() == [1]
            c.free([slot])
            slot, spare = spare, slot
        n += accepted
        assert int(c.lens[slot]) == n and torch.equal(one(slot, n), kept)
        assert int((c.refs > 0).sum()) == -(-n // 16)
        consistent(c)
