"""The attention half on the GPU against its plain 64-bit forms (attn_ref.py), with the bounds
derived there.  Every place of the cache that a call may not read holds NaN."""
from __future__ import annotations

import math

import pytest
import torch

import attn_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make_cache(lens, Hkv, D, ps, seed=0, layers=2, extra=3, fill=math.nan):
    """Random pages for sequences of the given lengths, at shuffled places of a pool that is
    `fill` everywhere else; returns (pages, table, lens)."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-max(n, 0) // ps) for n in lens]
    n_pages = sum(need) + extra
    pages = torch.full((n_pages, layers, 2, Hkv, ps, D), fill, dtype=R.BF16)
    order = torch.randperm(n_pages, generator=g).tolist()
    table = torch.full((len(lens), max(max(need), 1)), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        for j in range(need[b]):
            p = order.pop()
            table[b, j] = p
            rows = min(ps, n - j * ps)
            pages[p, :, :, :, :rows] = torch.randn(layers, 2, Hkv, rows, D, generator=g).to(R.BF16)
    return pages.to(DEV), table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)


def rand_q(T, Hq, D, seed=1, pad=0):
    """q rows; with pad, a view of a wider buffer (other token and head strides)."""
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(T, Hq, D + pad, generator=g).to(R.BF16).to(DEV)
    return q[..., :D]


def cu_of(new):
    return torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device=DEV)


def check_decode(lens, Hq, Hkv, D, ps, window=0, sinks=0, seed=0, pad=0, scale=None):
    from paris_moe_b200 import ops
    pages, table, n = make_cache(lens, Hkv, D, ps, seed)
    q = rand_q(len(lens), Hq, D, seed + 1, pad)
    scale = D ** -0.5 if scale is None else scale
    k, v = pages[:, 1, 0], pages[:, 1, 1]
    got = ops.attn_decode(q, k, v, table, n, scale, window, sinks)
    want, bound = R.attention(q, k, v, table, n, cu_of([1] * len(lens)), scale, window, sinks)
    R.within(got, want, bound, f"decode {lens} {Hq}/{Hkv} D{D} ps{ps} w{window} s{sinks}")


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("ps", [16, 32, 64, 128])
def test_decode_lengths(D, ps):
    check_decode([0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 500, 1000], 4, 2, D, ps)


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (2, 2), (3, 1), (16, 2), (10, 2), (16, 1), (17, 1),
                                    (40, 1), (128, 1), (8, 8)])
def test_decode_head_groups(Hq, Hkv):
    check_decode([70, 5, 333], Hq, Hkv, 128, 16, pad=8)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 3), (64, 4), (65, 64), (100, 130),
                                          (300, 0), (1000, 5), (128, 16)])
def test_decode_window_and_sinks(window, sinks):
    check_decode([1, 6, 64, 65, 200, 390, 777], 6, 2, 64, 16, window, sinks)
    check_decode([1, 129, 700], 4, 1, 256, 64, window, sinks)


def test_decode_reads_no_key_outside_the_window():
    """Keys that the window has passed may be anything, and their pages may be gone."""
    from paris_moe_b200 import ops
    lens, ps, window, sinks = [200, 333], 16, 50, 5
    pages, table, n = make_cache(lens, 2, 128, ps)
    for b, m in enumerate(lens):
        see = R.visible(m - 1, m, window, sinks)
        for j in torch.nonzero(~see)[:, 0].tolist():
            pages[table[b, j // ps].item(), :, :, :, j % ps] = math.nan
        for i in range(table.shape[1]):
            if not see[i * ps:(i + 1) * ps].any():
                table[b, i] = -1
    q = rand_q(2, 4, 128)
    args = (pages[:, 0, 0], pages[:, 0, 1], table, n)
    got = ops.attn_decode(q, *args, 0.1, window, sinks)
    want, bound = R.attention(q, *args, cu_of([1, 1]), 0.1, window, sinks)
    assert not torch.isnan(want).any()
    R.within(got, want, bound)


def test_decode_long_ragged():
    check_decode([9000, 1, 4097, 0, 2500], 8, 2, 128, 64)
    check_decode([20011], 16, 2, 256, 16)


def test_decode_many_sequences():
    check_decode([(i * 37) % 300 for i in range(200)], 4, 2, 64, 32)


def test_decode_extreme_scores():
    """Scores far apart: one key takes all; large scale, negative scale, zero scale."""
    for scale in (30.0, -2.0, 0.0):
        check_decode([100, 64, 1], 4, 2, 64, 16, scale=scale)


def test_decode_infinite_and_nan_keys_reach_only_their_own_sequence():
    from paris_moe_b200 import ops
    pages, table, n = make_cache([100, 90, 80], 1, 64, 16, layers=1)
    pages[table[1, 2].item(), 0, 0, 0, 3] = math.nan
    pages[table[2, 1].item(), 0, 1, 0, 5, 7] = math.inf
    q = rand_q(3, 2, 64)
    got = ops.attn_decode(q, pages[:, 0, 0], pages[:, 0, 1], table, n, 0.1)
    want, bound = R.attention(q, pages[:, 0, 0], pages[:, 0, 1], table, n, cu_of([1, 1, 1]), 0.1)
    assert torch.isnan(got[1]).all() and torch.isinf(got[2, :, 7]).all()
    got, want = got.cpu(), want.clone()
    assert torch.equal(torch.isinf(got), torch.isinf(want))
    want[2, :, 7], got[2, :, 7], bound[2, :, 7] = 0, 0, 1
    R.within(got, want, bound)


def test_missing_pages_give_nan_and_touch_nothing():
    from paris_moe_b200 import ops
    pages, table, n = make_cache([100, 100, 100, 100], 2, 64, 16)
    table[0, 3], table[1, 6], table[2, 0] = -1, pages.shape[0], -2 ** 31
    n[3] = table.shape[1] * 16 + 1       # longer than the table
    q = rand_q(4, 4, 64)
    k, v = pages[:, 0, 0], pages[:, 0, 1]
    got = ops.attn_decode(q, k, v, table, n, 0.1)
    assert torch.isnan(got).all()
    new = [3, 30, 2, 5]
    qp = rand_q(40, 4, 64)
    got = ops.attn_prefill(qp, k, v, table, n, cu_of(new), 0.1)
    want, bound = R.attention(qp, k, v, table, n, cu_of(new), 0.1)
    R.within(got, want, bound)
    assert torch.isnan(got[:3]).all() and not torch.isnan(got[3:20]).any()


def check_prefill(new, ctx, Hq, Hkv, D, ps, window=0, sinks=0, seed=0, pad=0, behind=0):
    from paris_moe_b200 import ops
    lens = [a + b for a, b in zip(new, ctx)]
    pages, table, n = make_cache(lens, Hkv, D, ps, seed)
    q = rand_q(sum(new) + behind, Hq, D, seed + 1, pad)
    k, v = pages[:, 0, 0], pages[:, 0, 1]
    cu = cu_of(new)
    got = ops.attn_prefill(q, k, v, table, n, cu, D ** -0.5, window, sinks)
    want, bound = R.attention(q, k, v, table, n, cu, D ** -0.5, window, sinks)
    R.within(got, want, bound, f"prefill {new} {ctx} {Hq}/{Hkv} D{D} ps{ps} w{window} s{sinks}")
    assert not got[sum(new):].any()


@pytest.mark.parametrize("scale", [30.0, -2.0, 0.0, 1e-42])
@pytest.mark.parametrize("D,Hq,new,ctx", [(64, 2, [100, 3], [0, 90]), (128, 4, [5], [2000]),
                                          (256, 16, [130, 200], [40, 0])])
def test_prefill_extreme_scales(D, Hq, new, ctx, scale):
    """One key takes all; all keys weigh the same; also where the keys are split and in pairs."""
    from paris_moe_b200 import ops
    pages, table, n = make_cache([a + b for a, b in zip(new, ctx)], 2, D, 16, 3)
    q, cu = rand_q(sum(new), Hq, D), cu_of(new)
    got = ops.attn_prefill(q, pages[:, 0, 0], pages[:, 0, 1], table, n, cu, scale, 70, 3)
    want, bound = R.attention(q, pages[:, 0, 0], pages[:, 0, 1], table, n, cu, scale, 70, 3)
    R.within(got, want, bound)
    got = ops.attn_prefill(q, pages[:, 0, 0], pages[:, 0, 1], table, n, cu, scale)
    want, bound = R.attention(q, pages[:, 0, 0], pages[:, 0, 1], table, n, cu, scale)
    R.within(got, want, bound)


def test_a_scale_that_is_not_a_number_gives_nan_where_keys_are_seen():
    from paris_moe_b200 import ops
    pages, table, n = make_cache([40, 0], 2, 64, 16)
    q = rand_q(2, 4, 64)
    cu = cu_of([1, 1])
    k, v = pages[:, 0, 0], pages[:, 0, 1]
    for got in (ops.attn_decode(q, k, v, table, n, math.nan),
                ops.attn_prefill(q, k, v, table, n, cu, math.nan)):
        assert torch.isnan(got[0]).all() and not got[1].any()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("ps", [16, 32, 64, 128])
def test_prefill_lengths(D, ps):
    check_prefill([1, 5, 0, 16, 17, 64, 65, 130], [0, 3, 40, 0, 64, 1, 0, 77], 4, 2, D, ps)


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (3, 1), (5, 1), (16, 2), (16, 1), (17, 1), (128, 1),
                                    (100, 1), (8, 8)])
def test_prefill_head_groups(Hq, Hkv):
    check_prefill([33, 1, 80], [0, 200, 9], Hq, Hkv, 64, 16, pad=16)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 3), (64, 4), (65, 64), (100, 130),
                                          (300, 0), (1000, 5), (128, 16)])
def test_prefill_window_and_sinks(window, sinks):
    check_prefill([70, 1, 150], [0, 300, 260], 4, 2, 64, 16, window, sinks)
    check_prefill([90, 3], [200, 333], 3, 1, 256, 64, window, sinks)


def test_prefill_one_long_prompt():
    check_prefill([1500], [0], 4, 1, 128, 64)
    check_prefill([700], [0], 16, 2, 256, 16)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_prefill_many_rows(D):
    """Enough tiles to fill the GPU: whole keys per CTA, in pairs of CTAs where D allows."""
    check_prefill([700, 1, 33, 250], [0, 3, 500, 130], 16, 1, D, 16)
    check_prefill([301, 222], [40, 0], 32, 1, D, 64, window=100, sinks=7, pad=8)
    check_prefill([9] * 20 + [40] * 3, [300] * 23, 100, 1, D, 32)


@pytest.mark.parametrize("Hq,Hkv,D,new,ctx", [(16, 1, 128, [500, 300], [900, 1300]), (16, 1, 256, [400], [1500]),
                                              (2, 1, 256, [130], [1700]), (4, 4, 64, [260, 40], [800, 2000])])
def test_prefill_maxima_that_keep_growing(Hq, Hkv, D, new, ctx):
    """Keys get larger along the sequence, so that every tile moves most rows' maxima."""
    from paris_moe_b200 import ops
    lens = [a + b for a, b in zip(new, ctx)]
    pages, table, n = make_cache(lens, Hkv, D, 32, 7, layers=1)
    for b, m in enumerate(lens):
        for i in range(-(-m // 32)):
            pages[table[b, i].item(), :, 0] *= 0.2 + 0.15 * i
    q, cu = rand_q(sum(new), Hq, D, 8), cu_of(new)
    args = (pages[:, 0, 0], pages[:, 0, 1], table, n, cu, D ** -0.5)
    got = ops.attn_prefill(q, *args)
    want, bound = R.attention(q, *args)
    R.within(got, want, bound)
    for _ in range(30):
        assert torch.equal(ops.attn_prefill(q, *args), got)


def test_prefill_many_short_sequences_and_rows_behind_the_last():
    check_prefill([i % 7 for i in range(70)], [(i * 11) % 50 for i in range(70)], 8, 2, 128, 16,
                  behind=13)


def test_prefill_rows_before_the_cache_get_zeros():
    """More new tokens than cached keys: the first rows lie at indexes below zero."""
    from paris_moe_b200 import ops
    pages, table, n = make_cache([10, 20], 1, 64, 16)
    n[0] = 4
    cu = cu_of([10, 20])
    q = rand_q(30, 2, 64)
    k, v = pages[:, 0, 0], pages[:, 0, 1]
    got = ops.attn_prefill(q, k, v, table, n, cu, 0.1)
    want, bound = R.attention(q, k, v, table, n, cu, 0.1)
    assert not got[:6].any() and got[6:].any()
    R.within(got, want, bound)


@pytest.mark.parametrize("D,Hq", [(64, 2), (256, 2), (64, 64), (128, 64), (256, 64)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_prefill_nonfinite_keys_and_values_stay_behind_the_mask(D, Hq, bad):
    """A non-finite key or value changes the rows that see it and no other row."""
    from paris_moe_b200 import ops
    new, ctx, window, sinks = [100, 40], [60, 0], 37, 3
    lens = [a + b for a, b in zip(new, ctx)]
    for where in ("k", "v", "both"):
        for win, snk in ((0, 0), (window, sinks)):
            pages, table, n = make_cache(lens, 1, D, 16, layers=1)
            clean = pages.clone()
            for b, j in ((0, 100), (0, 117), (0, 62), (1, 20), (1, 1)):
                p = table[b, j // 16].item()
                if where in ("k", "both"):
                    pages[p, 0, 0, 0, j % 16, 3] = bad
                if where in ("v", "both"):
                    pages[p, 0, 1, 0, j % 16, 5] = bad
            q, cu = rand_q(140, Hq, D), cu_of(new)
            args = (table, n, cu, 0.1, win, snk)
            got = ops.attn_prefill(q, pages[:, 0, 0], pages[:, 0, 1], *args).cpu()
            want, bound = R.attention(q, pages[:, 0, 0], pages[:, 0, 1], *args)
            good, gbound = R.attention(q, clean[:, 0, 0], clean[:, 0, 1], *args)
            fine = torch.isfinite(want)
            # where a key is infinite the weights are 0, 1 or NaN: only who is touched counts
            hit = ~torch.isclose(good, want, rtol=1e-9, atol=1e-9, equal_nan=False)
            assert torch.equal(torch.isnan(got)[~hit], torch.zeros_like(got[~hit], dtype=torch.bool))
            off = ((got.double() - good).abs() / gbound)[~hit]
            assert float(off.max()) <= 1.0
            both = hit & fine & ~torch.isnan(got)
            if where == "v" and both.any():
                assert float(((got.double() - want).abs() / bound)[both].max()) <= 1.0
            if where == "v":
                assert torch.equal(torch.isnan(got) | torch.isinf(got), ~fine)


@pytest.mark.parametrize("window,sinks", [(0, 0), (180, 70)])
@pytest.mark.parametrize("D,Hq", [(64, 1), (64, 16), (128, 1), (128, 16), (256, 1), (256, 16)])
def test_prefill_many_nonfinite_values_in_all_dims(D, Hq, window, sinks):
    """Values that are not finite in every tile, at every 64 dims: each row has them in exactly
    the dims and from the keys that it sees."""
    from paris_moe_b200 import ops
    new, ctx = [300, 290], [500, 0]
    lens = [a + b for a, b in zip(new, ctx)]
    pages, table, n = make_cache(lens, 1, D, 32, layers=1)
    g = torch.Generator().manual_seed(D + Hq + window)
    for b in (0, 1):
        for j in torch.randperm(lens[b], generator=g)[:40].tolist():
            d = int(torch.randint(0, D, (1,), generator=g))
            bad = (math.nan, math.inf, -math.inf)[j % 3]
            pages[table[b, j // 32].item(), 0, 1, 0, j % 32, d] = bad
    q, cu = rand_q(sum(new), Hq, D), cu_of(new)
    args = (table, n, cu, 0.02, window, sinks)
    got = ops.attn_prefill(q, pages[:, 0, 0], pages[:, 0, 1], *args).cpu()
    want, bound = R.attention(q, pages[:, 0, 0], pages[:, 0, 1], *args)
    fine = torch.isfinite(want)
    assert 0 < int(fine.sum()) < fine.numel()
    assert torch.equal(torch.isfinite(got), fine)
    assert float(((got.double() - want).abs() / bound)[fine].max()) <= 1.0


def test_prefill_of_single_tokens_agrees_with_decode():
    from paris_moe_b200 import ops
    lens = [1, 64, 100, 333]
    pages, table, n = make_cache(lens, 2, 128, 32)
    q = rand_q(4, 8, 128)
    k, v = pages[:, 0, 0], pages[:, 0, 1]
    a = ops.attn_decode(q, k, v, table, n, 0.09, 50, 4)
    b = ops.attn_prefill(q, k, v, table, n, cu_of([1] * 4), 0.09, 50, 4)
    _, bound = R.attention(q, k, v, table, n, cu_of([1] * 4), 0.09, 50, 4)
    assert bool(((a.cpu().double() - b.cpu().double()).abs() <= 2 * bound).all())


def test_calls_repeat_bit_for_bit_and_replay_from_graphs():
    """Same inputs, same bits: eager, on another stream, and two captured graphs replayed in
    turns with new contents in the same tensors."""
    from paris_moe_b200 import ops
    pages, table, n = make_cache([700, 3000, 1, 64], 2, 128, 16)
    q, qp = rand_q(4, 8, 128), rand_q(60, 8, 128, 5)
    k, v, cu = pages[:, 0, 0], pages[:, 0, 1], cu_of([40, 15, 1, 4])

    def both():
        return (ops.attn_decode(q, k, v, table, n, 0.1, 0, 0),
                ops.attn_prefill(qp, k, v, table, n, cu, 0.1, 100, 4))
    first = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = both()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = both()
        graphs.append((g, out))
    for g, out in graphs + graphs:
        g.replay()
        assert all(torch.equal(a, b) for a, b in zip(first, out))
    q.copy_(rand_q(4, 8, 128, 9))
    n.copy_(torch.tensor([650, 2000, 1, 33], dtype=torch.int32))
    cu.copy_(cu_of([7, 33, 1, 2]))
    third = both()
    for g, out in graphs:
        g.replay()
        assert all(torch.equal(a, b) for a, b in zip(third, out))
    want, bound = R.attention(q, k, v, table, n, cu_of([1] * 4), 0.1)
    R.within(third[0], want, bound)


def test_calls_follow_lengths_that_the_kernel_before_them_wrote():
    """Back to back: bookkeeping that moves the lengths, then the calls that read them."""
    from paris_moe_b200 import PagedKVCache, ops
    g = torch.Generator().manual_seed(2)
    c = PagedKVCache(200, 16, 1, 1, 64, 3, 900)
    c.pages.copy_(torch.randn(c.pages.shape, generator=g))
    one = torch.ones(3, dtype=torch.int32, device=DEV)
    slots = torch.arange(3, dtype=torch.int32, device=DEV)
    q = rand_q(3, 2, 64)
    c.grow(slots, [1, 300, 100])
    got, at = [], []
    for _ in range(120):
        c.grow(slots, one)
        got.append(ops.attn_decode(q, c.k(0), c.v(0), c.tables, c.lens, 0.2))
        got.append(ops.attn_prefill(q, c.k(0), c.v(0), c.tables, c.lens, cu_of([1, 1, 1]), 0.2))
        at.append(c.lens.clone())
    for i in (0, 1, 17, 60, 119):
        want, bound = R.attention(q, c.k(0), c.v(0), c.tables, at[i], cu_of([1, 1, 1]), 0.2)
        R.within(got[2 * i], want, bound)
        R.within(got[2 * i + 1], want, bound)
    # every step's row differs from the one before: a call on stale lengths would repeat it
    for i in range(1, 120):
        assert not torch.equal(got[2 * i], got[2 * i - 2])


def test_calls_on_two_streams_at_once():
    from paris_moe_b200 import ops
    pages, table, n = make_cache([700, 3000, 1, 64], 2, 128, 16)
    pages2, table2, n2 = make_cache([2500, 90], 2, 128, 64, 5)
    q, qp = rand_q(4, 8, 128), rand_q(300, 32, 128, 5)
    cu = cu_of([180, 120 - 30])
    qp = qp[:270]

    def left():
        return ops.attn_decode(q, pages[:, 0, 0], pages[:, 0, 1], table, n, 0.1)

    def right():
        return ops.attn_prefill(qp, pages2[:, 1, 0], pages2[:, 1, 1], table2, n2, cu, 0.1)
    a, b = left(), right()
    torch.cuda.synchronize()
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    out = []
    for _ in range(40):
        with torch.cuda.stream(s):
            out.append((left(), right()))
        with torch.cuda.stream(t):
            out.append((left(), right()))
    torch.cuda.synchronize()
    assert all(torch.equal(x, a) and torch.equal(y, b) for x, y in out)


def test_empty_calls():
    from paris_moe_b200 import ops
    pages, table, n = make_cache([5], 1, 64, 16)
    k, v = pages[:, 0, 0], pages[:, 0, 1]
    none = table[:0], n[:0]
    assert ops.attn_decode(rand_q(0, 2, 64), k, v, *none, 0.1).shape == (0, 2, 64)
    assert ops.attn_prefill(rand_q(0, 2, 64), k, v, table, n, cu_of([0]), 0.1).shape == (0, 2, 64)
    # no pages at all, and a table without entries
    out = ops.attn_decode(rand_q(1, 2, 64), k[:0], v[:0], table[:, :0], n * 0, 0.1)
    assert not out.any()


def test_bad_arguments_raise():
    from paris_moe_b200 import ops
    pages, table, n = make_cache([5, 9], 2, 64, 16)
    k, v, q = pages[:, 0, 0], pages[:, 0, 1], rand_q(2, 4, 64)
    for match, args in (("bf16", (q.float(), k, v, table, n)), ("q must be", (q[..., :32], k, v, table, n)),
                        ("page_table", (q, k, v, table.long(), n)),
                        ("CUDA", (q, k, v, table.cpu(), n)), ("differ", (q, k, v[:1], table, n)),
                        ("rows", (q, k, v, table, n[:1])), ("q must be", (q[:1], k, v, table, n)),
                        ("contiguous", (q, k.transpose(2, 3), v.transpose(2, 3), table, n)),
                        ("status -1", (q[:, :3], k, v, table, n))):
        with pytest.raises(RuntimeError, match=match):
            ops.attn_decode(*args, 0.1)
    with pytest.raises(RuntimeError, match="status -1"):
        ops.attn_decode(q, k, v, table, n, 0.1, -1)
    with pytest.raises(RuntimeError, match="cu_q"):
        ops.attn_prefill(q, k, v, table, n, cu_of([1]), 0.1)
    with pytest.raises(RuntimeError, match="16-byte"):
        ops.attn_decode(rand_q(2, 4, 68)[..., 4:], k, v, table, n, 0.1)
    grad = q.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no backward pass"):
        ops.attn_decode(grad, k, v, table, n, 0.1)
    with torch.no_grad():
        assert torch.equal(ops.attn_decode(grad, k, v, table, n, 0.1), ops.attn_decode(q, k, v, table, n, 0.1))


def test_caches_and_gains_that_require_grad_are_refused():
    """They would get no gradient, so the calls raise instead."""
    from paris_moe_b200 import ops
    pages, table, n = make_cache([5, 9], 2, 64, 16)
    k, v = pages[:, 0, 0], pages[:, 0, 1]
    q, kn = rand_q(2, 4, 64), rand_q(2, 2, 64)
    grad = pages.clone().requires_grad_()
    for kk, vv in ((grad[:, 0, 0], v), (k, grad[:, 0, 1])):
        with pytest.raises(RuntimeError, match="no backward pass"):
            ops.attn_decode(q, kk, vv, table, n, 0.1)
        with pytest.raises(RuntimeError, match="no backward pass"):
            ops.attn_prefill(q, kk, vv, table, n, cu_of([1, 1]), 0.1)
    at = torch.zeros(1, 2, dtype=torch.int64, device=DEV)
    freq = torch.ones(8, device=DEV)
    gain = torch.nn.Parameter(torch.zeros(64, dtype=torch.bfloat16, device=DEV))

    def turn(wq, wk):
        return ops.rope_append(q, kn, kn, at, freq, [8], False, k, v, table, n, w_qnorm=wq, w_knorm=wk)
    for wq, wk in ((gain, None), (None, gain), (gain, gain)):
        with pytest.raises(RuntimeError, match="no backward pass"):
            turn(wq, wk)
    with torch.no_grad():
        assert torch.equal(turn(gain, gain), turn(gain.detach(), gain.detach()))


# ---- rotary positions and the cache write -------------------------------------------------


def check_rope(T, new, ctx, Hq, Hkv, D, ps, rot, sections, interleaved, norm, seed=0, mscale=1.0,
               base=0, fused=True):
    from paris_moe_b200 import ops
    B = len(new)
    g = torch.Generator().manual_seed(seed)
    lens = [a + b for a, b in zip(new, ctx)]
    pages, table, n = make_cache(lens, Hkv, D, ps, seed)
    before = pages.clone()
    if fused:
        qkv = torch.randn(T, (Hq + 2 * Hkv) * D, generator=g).to(R.BF16).to(DEV)
        q, k, v = torch.split(qkv, [Hq * D, Hkv * D, Hkv * D], 1)
        q, k, v = q.view(T, Hq, D), k.view(T, Hkv, D), v.view(T, Hkv, D)
    else:   # a gated projection's layout: heads of 2D, of which q is the first half
        q = torch.randn(T, Hq, 2 * D, generator=g).to(R.BF16).to(DEV)[..., :D]
        k, v = (torch.randn(T, Hkv, D, generator=g).to(R.BF16).to(DEV) for _ in range(2))
    pos = torch.randint(0, 5000, (len(sections), T), generator=g).to(DEV) + base
    inv = (1e6 ** (-torch.arange(rot // 2).double() * 2 / max(rot, 1))).float().to(DEV)
    w = [(torch.randn(D, generator=g) * 0.2).to(R.BF16).to(DEV) for _ in range(2)]
    wq, wk = w if norm else (None, None)
    cu = None if new == [1] * B and T == B else cu_of(new)
    out = ops.rope_append(q, k, v, pos, inv, sections, interleaved, pages[:, 1, 0], pages[:, 1, 1],
                          table, n, cu_q=cu, w_qnorm=wq, w_knorm=wk, eps=1e-6, mscale=mscale)
    want, bound = R.rope(q, pos, inv, sections, interleaved, wq, 1e-6, mscale)
    R.within(out, want, bound, "q")
    wantk, boundk = R.rope(k, pos, inv, sections, interleaved, wk, 1e-6, mscale)
    pages, before, table = pages.cpu(), before.cpu(), table.cpu()
    t = 0
    for b in range(B):
        for i in range(new[b]):
            j = ctx[b] + i
            p = int(table[b, j // ps])
            R.within(pages[p, 1, 0, :, j % ps], wantk[t], boundk[t], "k")
            assert torch.equal(pages[p, 1, 1, :, j % ps], v[t].cpu())
            pages[p, 1, :, :, j % ps] = before[p, 1, :, :, j % ps]
            t += 1
    # nothing else of the pool has changed (compared as bits: much of it is NaN)
    assert torch.equal(pages.view(torch.int16), before.view(torch.int16))


@pytest.mark.parametrize("D,rot", [(64, 64), (64, 16), (128, 128), (128, 32), (256, 64), (256, 256),
                                   (256, 0)])
@pytest.mark.parametrize("norm", [False, True])
def test_rope_append(D, rot, norm):
    half = rot // 2
    for axes, inter in ((1, False), (3, True), (3, False), (4, True)):
        rest = [half // axes] * (axes - 1)
        check_rope(24, [5, 1, 0, 18], [0, 33, 7, 14], 6, 2, D, 16, rot, [half - sum(rest)] + rest,
                   inter, norm)


def test_rope_append_single_tokens_and_layouts():
    check_rope(5, [1] * 5, [0, 15, 16, 64, 99], 16, 2, 256, 64, 64, [11, 11, 10], True, True)
    check_rope(5, [1] * 5, [0, 15, 16, 64, 99], 16, 2, 256, 16, 64, [11, 11, 10], True, True, fused=False)
    check_rope(3, [1] * 3, [0, 1, 2], 5, 5, 64, 128, 32, [16], False, False, mscale=1.25)
    check_rope(40, [40], [0], 1, 1, 128, 32, 64, [8, 24], False, True)


def test_rope_far_positions():
    """Angles keep their precision at positions past 2^31."""
    check_rope(6, [6], [0], 2, 1, 64, 16, 64, [32], False, False, base=1 << 20)
    check_rope(6, [6], [0], 2, 1, 64, 16, 64, [32], False, False, base=3 << 30)


def test_rope_rows_behind_the_last_and_missing_pages_are_not_written():
    from paris_moe_b200 import ops
    pages, table, n = make_cache([20, 20], 1, 64, 16, layers=1)
    table[1, 1] = -1
    table[0, 1] = pages.shape[0] + 5
    before = pages.clone()
    q, k, v = rand_q(9, 2, 64), rand_q(9, 1, 64, 2), rand_q(9, 1, 64, 3)
    pos = torch.arange(9, device=DEV)[None].contiguous()
    inv = torch.ones(16, device=DEV)
    ops.rope_append(q, k, v, pos, inv, [16], False, pages[:, 0, 0], pages[:, 0, 1], table, n,
                    cu_q=cu_of([2, 5]))
    changed = (pages.view(torch.int16) != before.view(torch.int16)).any(-1).nonzero()
    # tokens 18, 19 of the first sequence and 16.. of the second have no page: token 15 alone
    assert {(int(r[0]), int(r[-1])) for r in changed} == {(int(table[1, 0]), 15)}


def test_together_prompt_fork_and_decode():
    """The calls in a row, as a server makes them: a prompt in two chunks, a fork into branches
    that each decode their own tokens, against attention over the whole recomputed history."""
    from paris_moe_b200 import PagedKVCache, ops
    Hq, Hkv, D, ps = 4, 2, 64, 16
    g = torch.Generator().manual_seed(3)
    cache = PagedKVCache(64, ps, 2, Hkv, D, 8, 200)
    hist = {}          # slot -> list of (k, v) rows, in 64 bits
    inv = (1e4 ** (-torch.arange(16).double() / 16)).float().to(DEV)

    def step(slots, new):
        T = sum(new)
        add = torch.tensor(new, dtype=torch.int32, device=DEV)
        assert cache.grow(slots, add).all()
        q, k, v = (torch.randn(T, h, D, generator=g).to(R.BF16).to(DEV) for h in (Hq, Hkv, Hkv))
        sl = torch.tensor(slots, device=DEV)
        table, lens = cache.tables[sl], cache.lens[sl]
        cu = cu_of(new)
        pos = torch.cat([torch.arange(int(n) - m, int(n)) for n, m in zip(lens, new)]).to(DEV)[None]
        qr = ops.rope_append(q, k, v, pos, inv, [16], False, cache.k(1), cache.v(1), table, lens,
                             cu_q=cu)
        kr, _ = R.rope(k, pos, inv, [16], False)
        t = 0
        for s, m in zip(slots, new):
            for _ in range(m):
                hist.setdefault(s, []).append((kr[t].to(R.BF16), v[t].cpu()))
                t += 1
        if new == [1] * len(slots):
            out = ops.attn_decode(qr, cache.k(1), cache.v(1), table, lens, 0.125)
        else:
            out = ops.attn_prefill(qr, cache.k(1), cache.v(1), table, lens, cu, 0.125)
        # the same from the recorded history, laid out in pages of its own
        width = max(-(-len(hist[s]) // ps) for s in slots)
        kp = torch.zeros(len(slots) * width, Hkv, ps, D, dtype=R.BF16)
        vp = torch.zeros_like(kp)
        for i, s in enumerate(slots):
            for j, (a, b) in enumerate(hist[s]):
                kp[i * width + j // ps, :, j % ps] = a
                vp[i * width + j // ps, :, j % ps] = b
        rows = torch.arange(len(slots) * width).view(len(slots), width)
        want, bound = R.attention(qr, kp, vp, rows, torch.tensor([len(hist[s]) for s in slots]), cu, 0.125)
        # keys in the cache may round the other way: one bf16 step of a key moves a score by
        # 2^-7 * scale * sum|q k|, about 0.125 * 2^-7 * 50, for the few keys on a border
        R.within(out, want, bound + 0.05 * U_OF(want), "together")

    def U_OF(x):
        return x.abs() + 0.5

    step([0, 3], [37, 5])
    step([0, 3], [16, 1])
    assert cache.fork([0, 0, 3], [1, 2, 5], [53, 20, 6]).tolist() == [1, 1, 1]
    hist[1], hist[2], hist[5] = list(hist[0]), list(hist[0][:20]), list(hist[3])
    for _ in range(14):
        step([0, 1, 2, 3, 5], [1] * 5)
    cache.free([0, 3])
    live, _ = cache.compact()
    assert int(live) == int((cache.refs > 0).sum()) and (cache.refs[:int(live)] > 0).all()
    for _ in range(3):
        step([1, 2, 5], [1] * 3)
