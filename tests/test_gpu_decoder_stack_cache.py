"""The decoder stack's use of its cache, against a history that the test keeps itself: which layer
writes where, and that attention reads what was written there."""
from __future__ import annotations

import pytest
import torch

import attn_ref as R
from test_gpu_decoder_stack import D, DEV, H, HKV, HQ, PS, SECTIONS, make, step_of

pytestmark = pytest.mark.gpu


class Layer:
    """One attention half: the rows its tokens' keys and values should have, by sequence slot."""

    def __init__(self, st, w):
        self.st, self.w = st, w
        self.rows = {}             # slot -> [(key, how far off it may be, value)]
        self.scratch = torch.zeros_like(st.cache.k(0)).contiguous()

    def project(self, h, step, slots, new):
        """The tokens' turned queries; their keys and values go to the history."""
        from paris_moe_b200 import ops
        st, w, T = self.st, self.w, h.shape[0]
        qkv = ops.rmsnorm(h, w.w_norm, st.eps) @ w.w_qkv.t()
        wide = qkv.shape[1] - 2 * HKV * D
        q = qkv[:, :wide].view(T, HQ, -1)
        k, v = (qkv[:, a:a + HKV * D].view(T, HKV, D) for a in (wide, wide + HKV * D))
        kr, kb = R.rope(k, step.positions, st.inv_freq, SECTIONS, True, w.k_norm, st.eps)
        t = 0
        for s, m in zip(slots, new):
            for _ in range(m):
                self.rows.setdefault(s, []).append((kr[t], kb[t], v[t].cpu()))
                t += 1
        # (queries alone: the call writes to a cache of its own)
        turned = ops.rope_append(q[..., :D], k, v, step.positions, st.inv_freq, SECTIONS, True,
                                 self.scratch, self.scratch.clone(), step.page_table, step.kv_lens,
                                 cu_q=step.cu_q, w_qnorm=w.q_norm, w_knorm=w.k_norm, eps=st.eps)
        qr, qb = R.rope(q[..., :D], step.positions, st.inv_freq, SECTIONS, True, w.q_norm, st.eps)
        R.within(turned, qr, qb, "queries")
        return turned, q[..., D:].cpu().double()

    def expected_pages(self, layer):
        """The layer's keys and values as the history has them: each row checked in the cache and
        taken from there (a key may round either way); NaN everywhere else."""
        c = self.st.cache
        pages, tables = c.pages[:, layer].cpu(), c.tables.cpu()
        want = torch.full_like(pages, float("nan"))
        for s, rows in self.rows.items():
            for j, (kr, kb, v) in enumerate(rows):
                p, r = int(tables[s, j // PS]), j % PS
                R.within(pages[p, 0, :, r], kr, kb, f"key {j} of slot {s}")
                assert torch.equal(pages[p, 1, :, r], v), f"value {j} of slot {s}"
                want[p, :, :, r] = pages[p, :, :, r]
        return want


def attended(st, w, h, q, gate, pages, step):
    """h + the layer's attention half in 64 bits, and how far the kernels may be off: the
    attention's own bound, two roundings of the gate (2 U), and the projection's sum in 32 bits with one
    rounding."""
    cu = step.cu_q if step.cu_q is not None else torch.arange(h.shape[0] + 1)
    o, bound = R.attention(q, pages[:, 0], pages[:, 1], step.page_table, step.kv_lens, cu, D ** -0.5,
                           st.window, st.sinks)
    if w.gated:
        g = torch.sigmoid(gate)
        o, bound = o * g, bound * g + 2 * R.U * (o * g).abs()
    wo = w.w_o.cpu().double()
    y = h.cpu().double() + o.reshape(h.shape[0], -1) @ wo.T
    return y, bound.reshape(h.shape[0], -1) @ wo.abs().T + (R.U + HQ * D * 2.0 ** -24) * y.abs() + 1e-6


@pytest.mark.parametrize("gated,window,sinks", [(True, 0, 0), (False, 20, 3)])
def test_each_layer_writes_and_reads_its_own_part_of_the_cache(gated, window, sinks):
    st, att = make(gated=gated, window=window, sinks=sinks)
    twin, _ = make(gated=gated, window=window, sinks=sinks)
    for s in (st, twin):
        s.cache.pages.fill_(float("nan"))
    layers = [Layer(st, w) for w in att if w is not None]
    g = torch.Generator().manual_seed(6)
    for slots, new in (([0, 2], [37, 5]), ([2, 0], [1, 1]), ([2, 0, 4], [20, 3, 1]), ([0, 2, 4], [1] * 3)):
        step, step2 = step_of(st, slots, new), step_of(twin, slots, new)
        h = torch.randn(sum(new), H, generator=g).to(R.BF16).to(DEV)
        whole = twin.forward(h.clone(), step2)
        at = 0
        for l, w in enumerate(att):
            if w is not None:
                q, gate = layers[at].project(h, step, slots, new)
                before = h.clone()
                st._attend(h, w, at, step)
                pages = layers[at].expected_pages(at)
                want, bound = attended(st, w, before, q, gate, pages, step)
                R.within(h, want, bound, f"{slots} {new} layer {l}")
                at += 1
            h = st.group.layer_forward(h, st.norms[l], st.eps, st.blocks[l].tensors())
        assert torch.equal(h, whole)
        # both caches hold the histories and nothing else, bit for bit
        for at, layer in enumerate(layers):
            want = layer.expected_pages(at).view(torch.int16)
            for s in (st, twin):
                assert torch.equal(s.cache.pages[:, at].cpu().view(torch.int16), want)


@pytest.mark.parametrize("single", [False, True])
def test_a_step_without_tokens(single):
    from paris_moe_b200 import Step
    st, _ = make()
    step_of(st, [0], [5])
    i32 = dict(dtype=torch.int32, device=DEV)
    rows = torch.tensor([], dtype=torch.int64, device=DEV) if single else torch.tensor([0], device=DEV)
    step = Step(st.cache.tables[rows], st.cache.lens[rows], torch.zeros((3, 0), dtype=torch.int64, device=DEV),
                None if single else torch.zeros(2, **i32))
    before = st.cache.pages.clone()
    h = torch.empty((0, H), dtype=R.BF16, device=DEV)
    out = st.forward(h, step)
    assert out.shape == (0, H) and torch.equal(st.cache.pages, before)


def test_a_step_too_long_for_the_exchange_is_refused_before_it_changes_anything():
    """Across ranks a layer takes as many tokens as the exchange holds: more are refused ahead of the
    first layer's attention half, not behind it."""
    from paris_moe_b200 import stack
    from paris_moe_b200.ep import EPGroup
    one, att = make()
    group = EPGroup.emulated(16, H, 4, rank=0, world=2)          # no exchange buffers at all
    st = stack.DecoderStack(one.norms, one.blocks, att, one.cache, one.inv_freq, SECTIONS, group=group)
    step = step_of(st, [0, 2], [30, 40])
    h = torch.randn(70, H, generator=torch.Generator().manual_seed(1)).to(R.BF16).to(DEV)
    before, pages = h.clone(), st.cache.pages.clone()
    with pytest.raises(ValueError, match="fused exchange"):
        st.forward(h, step)
    assert torch.equal(h, before) and torch.equal(st.cache.pages, pages)
    group.close()
