"""Decoder stacks: MoE halves alone, or with the attention half over a paged cache.

MoE-only decoder stack: per layer
``h = h + MoEBlock(RMSNorm(h))`` -- Qwen3_5MoeDecoderLayer with the attention
half omitted (post_attention_layernorm, mlp, residual add:
modeling_qwen3_5_moe.py:795-812, 862-868).

Each layer is one ``pmoe_layer_forward`` call (RMSNorm kernel, router,
expert kernels, combine with the residual folded in), updating the residual
stream in place; with an :class:`~.ep.EPGroup` of several ranks the expert
rows cross NVLink inside the down-projection epilogue and every rank ends
each layer with the full hidden state.  The whole stack can be captured in
one CUDA graph (the exchange uses device-side epochs).

:class:`DecoderStack` puts ``h = h + Attention(RMSNorm(h))`` ahead of the MoE half of the layers
that have attention weights (Qwen3_5MoeDecoderLayer's input_layernorm, self_attn and first
residual add): RMSNorm, the q/k/v projection, ``rope_append`` (per-head norms, rotary positions,
the write into the cache's pages), ``attn_decode`` or ``attn_prefill``, the output projection
onto the residual stream.  The projections are plain library matrix products.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lib, ops
from . import workload as W
from .ep import EPGroup

_BF16 = torch.bfloat16


def make_stack_weights(n_layers: int, shape: W.MoEShape = W.MoEShape(), seed: int = 0,
                       device="cuda"):
    """Seeded random-init weights for ``n_layers`` layers: layer l uses the block
    generator with seed ``seed + l`` and the RMSNorm weights of
    ``workload.make_rmsnorm_weights``.  Returns (norm [L,H] bf16, [MoEWeights])."""
    norms = W.make_rmsnorm_weights(n_layers, shape.H, seed=seed, device=device)
    blocks = [W.make_weights(shape, seed=seed + l, device=device) for l in range(n_layers)]
    return norms, blocks


class MoEStack:
    """``n_layers`` MoE-only decoder layers over a [T, H] bf16 residual stream.

    ``group`` (optional) is an :class:`EPGroup`; without one the stack runs on
    the current GPU.  ``forward(h)`` updates ``h`` in place and returns it."""

    def __init__(self, norms: torch.Tensor, blocks, eps: float = 1e-6,
                 group: EPGroup | None = None):
        if len(blocks) != norms.shape[0]:
            raise ValueError("one RMSNorm weight row per layer")
        self.norms = norms
        self.blocks = blocks
        self.eps = float(eps)
        shape = blocks[0].shape
        self.group = group or EPGroup(shape.E, shape.H, shape.K, mode="fused")
        self._graph = None

    def _workspace(self, T: int, device) -> torch.Tensor:
        """Scratch of one forward.  Each has its own, from the caching allocator's pool of the
        stream that it runs on, so calls on two streams do not meet; one that is captured
        gets it from its graph's pool, which lives as long as the graph."""
        s = self.blocks[0].shape
        nbytes = _lib.workspace_size(T, s.H, s.E, s.K, s.I, s.Is)
        return torch.empty(nbytes, dtype=torch.uint8, device=device)

    def _held(self):
        """What a captured forward reads and writes besides its arguments."""
        return [self.group, self.norms, *(t for b in self.blocks for t in b.tensors())]

    def forward(self, h: torch.Tensor) -> torch.Tensor:
        if h.dtype != _BF16 or not h.is_cuda or not h.is_contiguous():
            raise RuntimeError("MoEStack: h must be a contiguous bf16 CUDA tensor")
        ws = self._workspace(h.shape[0], h.device)
        for l, b in enumerate(self.blocks):
            self.group.layer_forward(h, self.norms[l], self.eps, b.tensors(), out=h,
                                     workspace=ws)
        return h

    # -- CUDA graph of the whole stack at a fixed T ---------------------------
    def capture(self, h_static: torch.Tensor) -> torch.cuda.CUDAGraph:
        """Capture ``forward(h_static)`` (in place) into a CUDA graph; replay with
        ``graph.replay()`` after writing the step's input into ``h_static``.  The graph keeps
        what it reads and writes alive and shares no scratch with other calls."""
        return self._capture([], h_static)

    def _capture(self, held, h_static: torch.Tensor, *args) -> torch.cuda.CUDAGraph:
        s = torch.cuda.Stream(device=h_static.device)
        s.wait_stream(torch.cuda.current_stream(h_static.device))
        with torch.cuda.stream(s):   # warm-up outside the graph (lazy init, tensor maps)
            self.forward(h_static.clone(), *args)
        torch.cuda.current_stream(h_static.device).wait_stream(s)
        g = torch.cuda.CUDAGraph()
        # (torch keeps the matrix products' scratch by stream, and all captures use one stream:
        # cleared before, it comes from this graph's pool; cleared after, the next has its own)
        torch._C._cuda_clearCublasWorkspaces()
        with torch.cuda.graph(g):
            self.forward(h_static, *args)
        torch._C._cuda_clearCublasWorkspaces()
        g.held = [h_static, *held, *self._held()]
        self._graph = g
        return g


@dataclass
class AttentionWeights:
    """bf16 weights of one layer's attention half."""
    w_norm: torch.Tensor               # [H]  input_layernorm, scales by (1 + w)
    w_qkv: torch.Tensor                # [(Hq + 2 Hkv) D, H]; gated: q rows are heads of 2D, q then gate
    w_o: torch.Tensor                  # [H, Hq D]
    heads: int                         # Hq
    kv_heads: int                      # Hkv
    head_dim: int                      # D
    q_norm: torch.Tensor | None = None  # [D]
    k_norm: torch.Tensor | None = None  # [D]
    gated: bool = False                # the attention's output times sigmoid(gate)

    def __post_init__(self):
        q = self.heads * self.head_dim
        rows = q * (2 if self.gated else 1) + 2 * self.kv_heads * self.head_dim
        H = self.w_norm.shape[0]
        if self.w_qkv.shape != (rows, H) or self.w_o.shape != (H, q):
            raise ValueError(f"attention weights: w_qkv {tuple(self.w_qkv.shape)}, w_o "
                             f"{tuple(self.w_o.shape)}, expected {(rows, H)} and {(H, q)}")


@dataclass
class Step:
    """The tokens that one forward call works on: rows of the batch's sequences in order, their
    keys' places already in the cache (``PagedKVCache.grow``)."""
    page_table: torch.Tensor           # [B, max_pages] int32
    kv_lens: torch.Tensor              # [B] int32, the step's tokens included
    positions: torch.Tensor            # [axes, T] int64
    cu_q: torch.Tensor | None = None   # [B + 1] int32; None: one token per sequence


class DecoderStack(MoEStack):
    """Decoder layers over a paged cache.  ``attention[l]`` is the layer's attention half, or None
    for a layer whose token mixing happens elsewhere; the k-th layer that has one uses layer k of
    ``cache``.  ``forward(h, step)`` updates the [T, H] residual stream ``h`` in place.
    Across ranks T is at most the group's ``t_max`` (its decode exchange)."""

    def __init__(self, norms: torch.Tensor, blocks, attention, cache, inv_freq: torch.Tensor,
                 sections, interleaved: bool = True, window: int = 0, sinks: int = 0,
                 eps: float = 1e-6, group: EPGroup | None = None):
        super().__init__(norms, blocks, eps, group)
        if len(attention) != len(blocks):
            raise ValueError("one attention half (or None) per layer")
        mine = [w for w in attention if w is not None]
        if len(mine) > cache.pages.shape[1]:
            raise ValueError(f"{len(mine)} attention layers, the cache has {cache.pages.shape[1]}")
        if any((w.kv_heads, w.head_dim) != (cache.pages.shape[3], cache.pages.shape[5]) for w in mine):
            raise ValueError("the cache's kv_heads and head_dim differ from the layers'")
        self.attention = list(attention)
        self.cache = cache
        self.inv_freq = inv_freq
        self.sections = list(sections)
        self.interleaved = bool(interleaved)
        self.window, self.sinks = int(window), int(sinks)

    def _attend(self, h: torch.Tensor, w: AttentionWeights, layer: int, step: Step) -> None:
        T, Hq, Hkv, D = h.shape[0], w.heads, w.kv_heads, w.head_dim
        qkv = ops.rmsnorm(h, w.w_norm, self.eps) @ w.w_qkv.t()
        q, k, v = qkv.split([qkv.shape[1] - 2 * Hkv * D, Hkv * D, Hkv * D], 1)
        q = q.view(T, Hq, (2 if w.gated else 1) * D)
        cache = (self.cache.k(layer), self.cache.v(layer), step.page_table, step.kv_lens)
        r = ops.rope_append(q[..., :D], k.view(T, Hkv, D), v.view(T, Hkv, D), step.positions,
                            self.inv_freq, self.sections, self.interleaved, *cache,
                            cu_q=step.cu_q, w_qnorm=w.q_norm, w_knorm=w.k_norm, eps=self.eps)
        if step.cu_q is None:
            o = ops.attn_decode(r, *cache, D ** -0.5, self.window, self.sinks)
        else:
            o = ops.attn_prefill(r, *cache, step.cu_q, D ** -0.5, self.window, self.sinks)
        if w.gated:
            o.mul_(torch.sigmoid(q[..., D:]))
        h.addmm_(o.view(T, Hq * D), w.w_o.t())

    @torch.no_grad()
    def forward(self, h: torch.Tensor, step: Step | None = None) -> torch.Tensor:
        if h.dtype != _BF16 or not h.is_cuda or not h.is_contiguous():
            raise RuntimeError("DecoderStack: h must be a contiguous bf16 CUDA tensor")
        if step is None and any(w is not None for w in self.attention):
            raise RuntimeError("DecoderStack: attention layers need a Step")
        if self.group.world > 1 and not self.group.uses_exchange(h.shape[0]):
            # (what layer_forward would say behind the first attention half)
            raise ValueError("DecoderStack across ranks needs the fused exchange (T <= t_max)")
        ws = self._workspace(h.shape[0], h.device)
        layer = 0
        for l, b in enumerate(self.blocks):
            if self.attention[l] is not None:
                self._attend(h, self.attention[l], layer, step)
                layer += 1
            self.group.layer_forward(h, self.norms[l], self.eps, b.tensors(), out=h,
                                     workspace=ws)
        return h

    def capture(self, h_static: torch.Tensor, step: Step | None = None) -> torch.cuda.CUDAGraph:
        """Capture ``forward(h_static, step)`` into a CUDA graph.  A replay works on what
        ``h_static`` and the step's tensors hold then, so the lengths and tables may have moved
        on (captured at the largest table width).  The warm-up runs outside the graph and writes
        the step's keys and values once.  The graph keeps what it reads and writes alive (the
        step's tensors and the cache's pages among it) and shares no scratch with other calls."""
        return self._capture([] if step is None else list(vars(step).values()), h_static, step)

    def _held(self):
        return [*super()._held(), self.cache.pages, self.inv_freq,
                *(t for w in self.attention if w is not None for t in vars(w).values())]


def make_attention_weights(n_layers: int, H: int = W.HIDDEN, heads: int = 16, kv_heads: int = 2,
                           head_dim: int = 256, gated: bool = True, seed: int = 0, device="cuda"):
    """Seeded random-init attention halves: projections N(0, 0.02), norms N(0, 0.02)."""
    out = []
    for l in range(n_layers):
        g = torch.Generator(device=device).manual_seed(seed + 15485863 + l)
        rows = heads * head_dim * (2 if gated else 1) + 2 * kv_heads * head_dim
        draw = lambda *shape: (torch.randn(shape, generator=g, device=device) * 0.02).to(_BF16)  # noqa: E731
        out.append(AttentionWeights(draw(H), draw(rows, H), draw(H, heads * head_dim), heads,
                                    kv_heads, head_dim, draw(head_dim), draw(head_dim), gated))
    return out
