"""The PyTorch operators ``torch.ops.paris_moe.*``, registered in C++
(csrc/torch_ops.cpp, built into libparis_moe_torch.so) over the C ABI.

    moe_block(x, w_router, w_gate_up, w_down, w_sh_gate, w_sh_up, w_sh_down, w_sh_gvec,
              top_k=8, expert_lo=0, expert_hi=-1, flags=3, *, ep_rank=0, ep_size=1,
              comm_handle=0) -> y
    moe_route(x, w_router, w_sh_gvec, k) -> (topk_idx, topk_w, offsets, sorted_tok,
                                            sorted_slot, shared_gate)
    moe_layer(x, w_norm, eps, <7 weights>, top_k=8, flags=3) -> y
    rmsnorm(x, w_norm, eps) -> y
    rope_append(q, k, v, positions, inv_freq, sections, interleaved, k_pages, v_pages,
                page_table, kv_lens, *, cu_q=None, w_qnorm=None, w_knorm=None, eps=1e-6,
                mscale=1.0) -> q       (k and v are written to the cache)
    attn_decode(q, k_pages, v_pages, page_table, kv_lens, scale, window=0, sinks=0) -> out
    attn_prefill(q, k_pages, v_pages, page_table, kv_lens, cu_q, scale, window=0, sinks=0) -> out
    pages_grow(refs, tables, lens, slots, add, page_size) -> ok
    pages_fork(pages, refs, tables, lens, src, dst, keep) -> ok
    pages_free(refs, tables, lens, slots, page_size, window=0, sinks=0)
    pages_compact(pages, refs, tables) -> (live, remap)

The ops run on the current CUDA stream, allocate their outputs and workspace
through PyTorch's caching allocator, never synchronise the host, and have
Meta kernels, so they can be captured in CUDA graphs at fixed T.  The CPU
kernels only raise (no fallback), a missing library raises at
import, and a kernel status other than 0 raises RuntimeError naming it.
``comm_handle`` is an ``EPGroup.comm_handle`` (pmoe_comm_create).
"""
from __future__ import annotations

import os

import torch

from . import _lib

OPS_LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "libparis_moe_torch.so")


if not os.path.exists(OPS_LIB_PATH):
    raise RuntimeError(
        f"{OPS_LIB_PATH} is missing: build it with `python "
        f"{os.path.dirname(OPS_LIB_PATH)}/build.py` (no CPU or Python fallback)")
_lib.load()  # the C ABI first, so the operator library's dependency resolves to it
torch.ops.load_library(OPS_LIB_PATH)

moe_block = torch.ops.paris_moe.moe_block
moe_route = torch.ops.paris_moe.moe_route
moe_layer = torch.ops.paris_moe.moe_layer
rmsnorm = torch.ops.paris_moe.rmsnorm
rope_append = torch.ops.paris_moe.rope_append
attn_decode = torch.ops.paris_moe.attn_decode
attn_prefill = torch.ops.paris_moe.attn_prefill
pages_grow = torch.ops.paris_moe.pages_grow
pages_fork = torch.ops.paris_moe.pages_fork
pages_free = torch.ops.paris_moe.pages_free
pages_compact = torch.ops.paris_moe.pages_compact
