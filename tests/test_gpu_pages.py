"""Page bookkeeping on the GPU against the same steps on plain lists (attn_ref.Cache): whole
numbers, equal everywhere."""
from __future__ import annotations

import random

import pytest
import torch

import attn_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


class Pair:
    """A cache and its plain twin; pages hold whole numbers, so that copies show."""

    def __init__(self, n_pages, ps, S, width, layers=1, Hkv=1, D=64, seed=0):
        from paris_moe_b200 import PagedKVCache
        self.c = PagedKVCache(n_pages, ps, layers, Hkv, D, S, width * ps)
        g = torch.Generator().manual_seed(seed)
        self.c.pages.copy_(torch.randint(-128, 128, self.c.pages.shape, generator=g))
        self.m = R.Cache(n_pages, ps, S, width)
        self.data = self.c.pages.cpu()

    def grow(self, slots, add):
        assert self.c.grow(slots, add).tolist() == self.m.grow(slots, add)

    def fork(self, src, dst, keep):
        ok, copies = self.m.fork(src, dst, keep)
        got = self.c.fork(src, dst, keep)
        assert got.tolist() == ok
        for a, b, used in copies:
            self.data[b, ..., :used, :] = self.data[a, ..., :used, :]

    def free(self, slots, window=0, sinks=0):
        self.c.free(slots, window, sinks)
        self.m.free(slots, window, sinks)

    def compact(self):
        live, remap = self.c.compact()
        want, wmap = self.m.compact()
        assert int(live) == want and remap.tolist() == wmap
        for p, q in enumerate(wmap):
            if q >= 0 and q != p:
                self.data[q] = self.data[p]

    def check(self):
        assert self.c.refs.tolist() == self.m.refs
        assert self.c.tables.tolist() == self.m.tables
        assert self.c.lens.tolist() == self.m.lens
        assert torch.equal(self.c.pages.cpu(), self.data)


@pytest.mark.parametrize("ps", [16, 32, 64, 128])
def test_a_session(ps):
    p = Pair(40, ps, 8, 6, layers=2, Hkv=2, seed=ps)
    p.grow([0, 1, 2], [ps * 2 + 3, ps, 1])
    p.check()
    p.fork([0, 0, 1, 2], [3, 4, 5, 6], [ps * 2 + 3, ps + 1, ps, 0])
    p.check()
    p.grow([3, 6, 2], [ps, 5, ps - 1])
    p.free([0, 5, 0])                       # listed twice: freed once
    p.check()
    p.compact()
    p.check()
    p.free([3], window=ps + 2, sinks=1)
    p.check()
    p.grow([0], [6 * ps])
    p.check()
    p.compact()
    p.check()


def test_refused_requests_change_nothing():
    p = Pair(6, 16, 6, 4)
    p.grow([0, 9, -1, 0, 1, 2], [20, 5, 5, 5, -3, 65])   # out of range, twice, negative, too long
    p.check()
    p.grow([1, 2, 3], [40, 40, 0])          # 3 pages, 3 more than the 1 left, none needed but behind
    p.check()
    p.grow([2, 3], [17, 16])                # 2 > 1 left: refused, and so is what follows
    p.check()
    p.grow([3, 2], [16, 17])                # the other way round the first fits
    p.check()
    p.fork([0, 0, 5, 1], [1, 0, 4, 9], [5, 5, 5, 5])     # not empty, itself, too long, out of range
    p.check()
    p.fork([0, 0], [4, 4], [16, 16])        # same target: the first one alone
    p.check()
    p.fork([0, 4], [5, 2], [17, -1])        # no page left for the tail
    p.check()
    p.free([-1, 6, 100])
    p.check()


def test_a_source_that_is_also_a_target_is_refused():
    p = Pair(12, 16, 6, 4)
    p.grow([0], [30])
    p.fork([0, 1, 0], [1, 2, 3], [30, 0, 16])
    p.check()


def test_fork_of_everything_refuses_sources_out_of_range():
    from paris_moe_b200 import PagedKVCache
    c = PagedKVCache(8, 16, 1, 1, 64, 4, 64)
    c.grow([0], [20])
    assert c.fork([0, -3, 4, 2 ** 31 - 1], [1, 2, 3, 3]).tolist() == [1, 0, 0, 0]
    assert c.lens.tolist() == [20, 20, 0, 0] and int(c.refs.sum()) == 4


def test_full_pool_and_empty_lists():
    p = Pair(5, 16, 4, 8)
    p.grow([], [])
    p.fork([], [], [])
    p.free([])
    p.compact()
    p.check()
    p.grow([2], [80])
    p.check()
    p.grow([1], [1])
    p.compact()
    p.check()
    p.free([2])
    p.compact()
    p.check()


def test_many_sequences_and_pages():
    """Lists longer than a block, a pool of several scan rounds."""
    p = Pair(9001, 16, 3000, 5, D=64)
    order = list(range(3000))
    random.Random(5).shuffle(order)
    p.grow(order[:1500], [1 + (i * 7) % 40 for i in range(1500)])
    p.check()
    p.fork(order[:1300], order[1500:2800], [1 + (i * 5) % (1 + (i * 7) % 40) for i in range(1300)])
    p.check()
    p.free(order[100:1400])
    p.compact()
    p.check()
    p.grow(order[:2990], [30] * 2990)       # more than fits: a prefix is granted
    p.check()


def test_requests_that_add_up_to_more_than_32_bits():
    """Sums of many huge requests do not wrap round into grants."""
    from paris_moe_b200 import ops
    S, width = 600, 1 << 22
    refs, lens = torch.zeros(50, dtype=torch.int32, device=DEV), torch.zeros(S, dtype=torch.int32, device=DEV)
    tables = torch.full((S, width), -1, dtype=torch.int32, device=DEV)
    add = [width * 16] * S
    add[0] = 33
    ok = ops.pages_grow(refs, tables, lens, torch.arange(S, dtype=torch.int32, device=DEV), i32(add), 16)
    assert ok.tolist() == [1] + [0] * (S - 1) and refs.tolist() == [1] * 3 + [0] * 47
    assert lens.tolist() == [33] + [0] * (S - 1)


def test_random_sessions():
    for seed in range(6):
        rng = random.Random(seed)
        p = Pair(60, 16, 10, 7, seed=seed)
        for _ in range(40):
            n = rng.randrange(5)
            slots = [rng.randrange(-1, 11) for _ in range(n)]
            op = rng.randrange(6)
            if op < 2:
                p.grow(slots, [rng.randrange(-1, 50) for _ in slots])
            elif op == 2:
                p.fork(slots, [rng.randrange(-1, 11) for _ in slots],
                       [rng.randrange(0, 60) for _ in slots])
            elif op == 3:
                p.free(slots)
            elif op == 4:
                p.free(slots, rng.randrange(1, 60), rng.randrange(0, 40))
            else:
                p.compact()
        p.check()


def test_captured_bookkeeping_replays():
    """A beam step captured once: free the branches, fork, grow; replays see the new state."""
    from paris_moe_b200 import PagedKVCache
    c = PagedKVCache(64, 16, 2, 1, 64, 6, 100)
    c.grow([0, 1], [37, 20])
    src, dst, keep, add = i32([0, 1, 0]), i32([2, 3, 4]), i32([37, 20, 16]), i32([1, 1, 1])

    def step():
        c.free(dst)
        return c.fork(src, dst, keep), c.grow(dst, add)
    step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ok = step()
    g.replay()
    assert ok[0].tolist() == [1, 1, 1] and ok[1].tolist() == [1, 1, 1]
    keep.copy_(i32([5, 20, 99]))
    g.replay()
    assert ok[0].tolist() == [1, 1, 0] and ok[1].tolist() == [1, 1, 1]
    m = R.Cache(64, 16, 6, 7)
    m.grow([0, 1], [37, 20])
    m.fork([0, 1], [2, 3], [5, 20])
    m.grow([2, 3, 4], [1, 1, 1])
    assert c.lens.tolist() == m.lens and sorted(c.refs.tolist()) == sorted(m.refs)


def test_bad_arguments_raise():
    from paris_moe_b200 import PagedKVCache, ops
    c = PagedKVCache(8, 16, 1, 1, 64, 3, 64)
    s = i32([0])
    with pytest.raises(RuntimeError, match="add has"):
        ops.pages_grow(c.refs, c.tables, c.lens, s, i32([1, 2]), 16)
    with pytest.raises(RuntimeError, match="status -5"):
        ops.pages_grow(c.refs, c.tables, c.lens, s, s, 17)
    with pytest.raises(RuntimeError, match="slots"):
        ops.pages_free(c.refs, c.tables, c.lens, s.long(), 16)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ops.pages_grow(c.refs, c.tables, c.lens, s.cpu(), s, 16)
    with pytest.raises(RuntimeError, match="pages holds"):
        ops.pages_compact(c.pages[:5], c.refs, c.tables)
    with pytest.raises(RuntimeError, match="contiguous"):
        ops.pages_compact(c.pages.transpose(1, 2).transpose(4, 5), c.refs, c.tables)
    with pytest.raises(RuntimeError, match="status -1"):
        ops.pages_free(c.refs, c.tables, c.lens, s, 16, -1, 0)
