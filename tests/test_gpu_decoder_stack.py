"""The decoder stack with its attention half: prompts, chunks, forks and single tokens through
the public calls, each layer's attention half checked against its 64-bit form from the GPU's
own input, and the captured decode step equal to the eager one."""
from __future__ import annotations

import pytest
import torch

import attn_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
H, HQ, HKV, D, PS, ROT = 256, 4, 2, 64, 16, 32
SECTIONS = [6, 5, 5]


def make(layers=3, gated=True, window=0, sinks=0):
    from paris_moe_b200 import PagedKVCache, stack, workload as W
    shape = W.MoEShape(H=H, E=16, K=4, I=64, Is=64)
    norms, blocks = stack.make_stack_weights(layers, shape, seed=2, device=DEV)
    att = stack.make_attention_weights(layers, H, HQ, HKV, D, gated, seed=3, device=DEV)
    att[1] = None                                   # a layer whose token mixing is elsewhere
    for w in att:
        if w is not None:
            w.w_qkv.mul_(8)                         # scores worth a softmax
    cache = PagedKVCache(64, PS, layers - 1, HKV, D, 6, 160)
    inv = (1e4 ** (-torch.arange(ROT // 2).double() * 2 / ROT)).float().to(DEV)
    return stack.DecoderStack(norms, blocks, att, cache, inv, SECTIONS, True, window, sinks), att


def step_of(st, slots, new):
    from paris_moe_b200 import Step
    assert bool(st.cache.grow(slots, new).all())
    sl = torch.tensor(slots, device=DEV)
    lens = st.cache.lens[sl]
    pos = torch.cat([torch.arange(int(n) - m, int(n)) for n, m in zip(lens, new)]).to(DEV)
    cu = None
    if new != [1] * len(new):
        cu = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device=DEV)
    return Step(st.cache.tables[sl], lens, torch.stack([pos, pos + 3, pos * 2]), cu)


def attend_ref(st, h, w, layer, step):
    """h + Attention(RMSNorm(h)) in 64 bits after the kernels' own bf16 projection, and a bound.
    The attention's bound covers its kernels; the gate (one rounding each of the sigmoid and the
    product) adds 2 U |o|; the output projection is a library product in 32 bits, one rounding."""
    from paris_moe_b200 import ops
    T = h.shape[0]
    qkv = (ops.rmsnorm(h, w.w_norm, st.eps) @ w.w_qkv.t()).cpu()
    wide = HQ * D * (2 if w.gated else 1)
    q = qkv[:, :wide].view(T, HQ, -1)
    qr, _ = R.rope(q[..., :D], step.positions, st.inv_freq, SECTIONS, True, w.q_norm, st.eps)
    # (the kernel's own rounded q and its cache of rounded k: rope_append is tested by itself)
    args = (q[..., :D].to(DEV), qkv[:, wide:wide + HKV * D].view(T, HKV, D).to(DEV),
            qkv[:, wide + HKV * D:].view(T, HKV, D).to(DEV))
    got_q = ops.rope_append(*args, step.positions, st.inv_freq, SECTIONS, True, st.cache.k(layer),
                            st.cache.v(layer), step.page_table, step.kv_lens, cu_q=step.cu_q,
                            w_qnorm=w.q_norm, w_knorm=w.k_norm, eps=st.eps)
    assert float((got_q.cpu().double() - qr).abs().max()) <= 2 * R.U * float(qr.abs().max())
    cu = step.cu_q if step.cu_q is not None else torch.arange(T + 1)
    o, bound = R.attention(got_q, st.cache.k(layer), st.cache.v(layer), step.page_table, step.kv_lens,
                           cu, D ** -0.5, st.window, st.sinks)
    if w.gated:
        g = torch.sigmoid(q[..., D:].double())
        o, bound = o * g, bound * g + 2 * R.U * (o * g).abs()
    wo = w.w_o.cpu().double()
    y = h.cpu().double() + o.reshape(T, -1) @ wo.T
    yb = bound.reshape(T, -1) @ wo.abs().T + (R.U + HQ * D * 2.0 ** -24) * y.abs() + 1e-6
    return y, yb


@pytest.mark.parametrize("gated,window,sinks", [(True, 0, 0), (False, 20, 3)])
def test_layers_match_their_plain_form(gated, window, sinks):
    st, att = make(gated=gated, window=window, sinks=sinks)
    g = torch.Generator().manual_seed(1)
    for slots, new in (([0, 2], [37, 5]), ([0, 2], [1, 1]), ([2, 0, 4], [20, 3, 1]), ([0, 2, 4], [1] * 3)):
        step = step_of(st, slots, new)
        h = torch.randn(sum(new), H, generator=g).to(R.BF16).to(DEV)
        for layer, l in ((0, 0), (1, 2)):
            want, bound = attend_ref(st, h, att[l], layer, step)
            got = h.clone()
            st._attend(got, att[l], layer, step)
            R.within(got, want, bound, f"{slots} {new} layer {l}")
        # and the whole stack is its layers in order
        a, b = st.forward(h.clone(), step), h.clone()
        layer = 0
        for l in range(3):
            if att[l] is not None:
                st._attend(b, att[l], layer, step)
                layer += 1
            st.group.layer_forward(b, st.norms[l], st.eps, st.blocks[l].tensors(), out=b,
                                   workspace=st._workspace(b.shape[0], b.device))
        assert torch.equal(a, b)


def test_prompt_fork_and_captured_decode():
    """A prompt, a fork into two branches, then decode steps from one captured graph against
    eager steps of a second stack with the same weights."""
    from paris_moe_b200 import Step
    g = torch.Generator().manual_seed(4)
    prompt = torch.randn(45, H, generator=g).to(R.BF16).to(DEV)
    tokens = [torch.randn(2, H, generator=g).to(R.BF16).to(DEV) for _ in range(5)]
    runs = []
    for captured in (False, True):
        st, _ = make()
        st.forward(prompt.clone(), step_of(st, [0], [45]))
        assert bool(st.cache.fork([0], [3]).all())
        out = []
        if captured:
            # static tensors of a step at the tables' full width
            static = Step(st.cache.tables[torch.tensor([0, 3], device=DEV)].clone(),
                          st.cache.lens[torch.tensor([0, 3], device=DEV)].clone(),
                          torch.zeros((3, 2), dtype=torch.int64, device=DEV))
            hs = tokens[0].clone()
            graph = None
        for x in tokens:
            step = step_of(st, [0, 3], [1, 1])
            if not captured:
                out.append(st.forward(x.clone(), step).clone())
                continue
            static.page_table.copy_(step.page_table)
            static.kv_lens.copy_(step.kv_lens)
            static.positions.copy_(step.positions)
            if graph is None:
                graph = st.capture(hs, static)
            hs.copy_(x)
            graph.replay()
            out.append(hs.clone())
        runs.append(out)
    for a, b in zip(*runs):
        assert torch.equal(a, b)
    # the branches share the prompt and see the same tokens' difference only
    assert not torch.equal(runs[0][0][0], runs[0][0][1])


def test_refusals():
    from paris_moe_b200 import AttentionWeights, stack
    st, att = make()
    h = torch.zeros(2, H, dtype=R.BF16, device=DEV)
    with pytest.raises(RuntimeError, match="need a Step"):
        st.forward(h)
    with pytest.raises(RuntimeError, match="bf16"):
        st.forward(h.float(), step_of(st, [0], [2]))
    with pytest.raises(ValueError, match="per layer"):
        stack.DecoderStack(st.norms, st.blocks, att[:2], st.cache, st.inv_freq, SECTIONS)
    with pytest.raises(ValueError, match="attention layers"):
        stack.DecoderStack(st.norms, st.blocks, [att[0]] * 3, st.cache, st.inv_freq, SECTIONS)
    with pytest.raises(ValueError, match="w_qkv"):
        AttentionWeights(att[0].w_norm, att[0].w_qkv, att[0].w_o, HQ, HKV, D, gated=False)
