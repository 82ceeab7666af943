"""Captured stacks: a graph owns what it works in, whatever is called, freed or captured after it."""
from __future__ import annotations

import pytest
import torch

import attn_ref as R
from test_gpu_decoder_stack import DEV, H, make, step_of

pytestmark = pytest.mark.gpu


def rows(n, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(n, H, generator=g).to(R.BF16).to(DEV)


def occupy(stream=None):
    """Take up freed memory with a pattern; returns the tensors."""
    with torch.cuda.stream(stream):
        return [torch.full((n,), 0x5a, dtype=torch.uint8, device=DEV)
                for n in [1 << k for k in range(9, 25)] * 3]


def untouched(taken):
    return all(bool((t == 0x5a).all()) for t in taken)


def test_a_longer_call_after_a_capture_leaves_the_graph_its_scratch():
    """A decode step is captured first, then a prompt of more tokens runs and new tensors take what
    memory is free: replays give the eager results and write to none of those tensors."""
    x, prompt = rows(2, 1), rows(45, 2)
    want_st, _ = make()
    step_of(want_st, [0, 3], [1, 1])
    st, _ = make()
    first = step_of(st, [0, 3], [1, 1])
    hs = x.clone()
    graph = st.capture(hs, first)
    st.forward(prompt.clone(), step_of(st, [1], [45]))
    torch.cuda.synchronize()
    taken = occupy()
    want = want_st.forward(x.clone(), first)
    for _ in range(3):
        hs.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(hs, want)
    assert untouched(taken)


def test_a_graph_keeps_its_step_alive():
    """The tensors of a step that the caller has dropped are not given to others."""
    x = rows(2, 3)
    st, _ = make()
    hs = x.clone()
    graph = st.capture(hs, step_of(st, [0, 3], [1, 1]))
    hs.copy_(x)
    taken = occupy()
    small = [torch.full((n,), 0x5a, dtype=torch.uint8, device=DEV) for n in range(8, 512, 8)]
    graph.replay()
    got = hs.clone()
    other, _ = make()
    want = other.forward(x.clone(), step_of(other, [0, 3], [1, 1]))
    assert torch.equal(got, want)
    assert untouched(taken) and untouched(small)


@pytest.mark.parametrize("attention", [False, True])
def test_two_graphs_replay_at_once(attention):
    """Two captured steps, of one stack or (with caches of their own) of two, on two streams."""
    from paris_moe_b200 import stack
    xs = [rows(6, 5), rows(4, 6)]
    if attention:
        pair = [make()[0], make()[0]]
        args = [(step_of(pair[0], list(range(6)), [1] * 6),), (step_of(pair[1], [0, 1, 2, 5], [1] * 4),)]
    else:
        one = make()[0]
        pair, args = [stack.MoEStack(one.norms, one.blocks)] * 2, [(), ()]
    hs = [x.clone() for x in xs]
    graphs = [p.capture(h, *a) for p, h, a in zip(pair, hs, args)]
    want = [p.forward(x.clone(), *a) for p, x, a in zip(pair, xs, args)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(30):
        for h, x, g, s in zip(hs, xs, graphs, streams):
            with torch.cuda.stream(s):
                h.copy_(x)
                g.replay()
        torch.cuda.synchronize()
        assert torch.equal(hs[0], want[0]) and torch.equal(hs[1], want[1])


def test_eager_calls_of_a_stack_on_two_streams_at_once():
    from paris_moe_b200 import stack
    st, _ = make()
    st = stack.MoEStack(st.norms, st.blocks)
    xs = [rows(40, 7), rows(23, 8)]
    want = [st.forward(x.clone()) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(30):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(st.forward(xs[i].clone()))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(y, want[i]) for y in got[i])


def test_a_graph_outlives_the_one_captured_before_it():
    """The second graph's matrix products do not work in the first one's memory."""
    x = rows(6, 9)
    st, _ = make()
    step = step_of(st, list(range(6)), [1] * 6)
    hs = x.clone()
    first = st.capture(x.clone(), step)
    second = st.capture(hs, step)
    del first
    st._graph = None
    torch.cuda.empty_cache()
    taken = occupy()
    hs.copy_(x)
    second.replay()
    want = st.forward(x.clone(), step)
    assert torch.equal(hs, want) and untouched(taken)
