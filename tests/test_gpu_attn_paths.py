"""Sizes at which the attention half takes other kernels or other paths in them, against the plain
64-bit forms (attn_ref.py)."""
from __future__ import annotations

import pytest
import torch

import attn_ref as R
from test_gpu_attn import DEV, check_decode, check_rope, cu_of, make_cache, rand_q
from test_gpu_pages import Pair

pytestmark = pytest.mark.gpu


# one warp a token from 148 * 16 tokens on, two from 148 * 4
@pytest.mark.parametrize("T", [591, 592, 2367, 2368, 2411])
@pytest.mark.parametrize("D,rot,norm", [(64, 64, True), (128, 32, False), (256, 64, True)])
def test_rope_of_prompts(T, D, rot, norm):
    new = [T // 2 + 3, 0, 1, T - T // 2 - 4]
    sec = [rot // 2 - 2 * (rot // 6), rot // 6, rot // 6]
    check_rope(T, new, [0, 5, 77, 300], 6, 3, D, 32, rot, sec, D != 128, norm)


@pytest.mark.parametrize("T", [640, 2400])
def test_rope_of_prompts_one_head_and_gated_layout(T):
    check_rope(T, [T], [1], 1, 1, 256, 64, 256, [128], False, False)
    check_rope(T, [T - 1, 1], [0, 9], 16, 2, 256, 64, 64, [11, 11, 10], True, True, fused=False)
    check_rope(T, [T], [0], 3, 1, 64, 16, 0, [0], False, True)


@pytest.mark.parametrize("B,D", [(257, 64), (700, 64), (300, 128), (193, 256), (401, 256)])
def test_decode_of_more_sequences_than_a_block_has_threads(B, D):
    check_decode([(i * 29) % 67 if i % 5 else 0 for i in range(B)], 2, 1, D, 16)
    check_decode([0] * (B - 1) + [900], 2, 2, D, 32, window=100, sinks=3)


def test_bookkeeping_of_more_sequences_than_marks_in_shared_memory():
    S = 5000
    p = Pair(7001, 16, S, 3, D=64)
    slots = [(i * 1237) % S for i in range(S)]
    p.grow(slots[:2500] + [slots[0]], [1 + (i * 7) % 40 for i in range(2500)] + [3])
    p.check()
    p.fork(slots[:2000] + [slots[1]], slots[2500:4500] + [slots[2500]],
           [(i * 5) % (2 + (i * 7) % 40) for i in range(2000)] + [1])
    p.check()
    p.free(slots[1000:3000])
    p.compact()
    p.check()
    p.grow(slots[4400:] + [0, S, -1], [20] * 603)
    p.check()


@pytest.mark.parametrize("D,Hq,T", [(64, 4, 100), (128, 2, 3), (256, 16, 259), (256, 16, 300), (64, 16, 1)])
def test_prefill_of_the_first_rows_of_a_batch(D, Hq, T):
    """cu_q may count more rows than the call has: a row's index goes by its sequence's own tokens."""
    from paris_moe_b200 import ops
    new, ctx = [90, 0, 170, 41], [700, 3, 0, 12]
    pages, table, n = make_cache([a + b for a, b in zip(new, ctx)], 2 if Hq < 16 else 1, D, 16)
    q, cu = rand_q(sum(new), Hq, D), cu_of(new)
    k, v = pages[:, 0, 0], pages[:, 0, 1]
    for window, sinks in ((0, 0), (40, 3)):
        want, bound = R.attention(q, k, v, table, n, cu, 0.1, window, sinks)
        got = ops.attn_prefill(q[:T], k, v, table, n, cu, 0.1, window, sinks)
        R.within(got, want[:T], bound[:T], f"{T} of {sum(new)} rows")
