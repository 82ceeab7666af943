"""Host logic of the stacks that needs no GPU."""
from __future__ import annotations

import pytest
import torch


@pytest.fixture(scope="module")
def mk():
    from paris_moe_b200 import build, stack, workload as W
    build.build()
    shape = W.MoEShape(H=256, E=16, K=4, I=64, Is=64)
    norms, blocks = stack.make_stack_weights(2, shape, seed=2, device="cpu")
    return lambda: stack.MoEStack(norms, blocks)


def test_every_forward_has_a_workspace_of_its_own(mk):
    """A captured call goes on writing to the one it was captured with: no later call may
    replace it, and no call on another stream may use it."""
    st = mk()
    few, same, many = (st._workspace(T, torch.device("cpu")) for T in (2, 2, 45))
    spans = sorted((t.data_ptr(), t.data_ptr() + t.numel()) for t in (few, same, many))
    assert all(a[1] <= b[0] for a, b in zip(spans, spans[1:]))
    from paris_moe_b200 import _lib
    assert many.numel() >= _lib.workspace_size(45, 256, 16, 4, 64, 64)
    assert not any(isinstance(x, torch.Tensor) and x.dtype == torch.uint8 for x in vars(st).values())
