"""The rows a Transition's backward pass leaves out are those its b200 forward pass leaves out, whatever the
key mask's dtype."""

from __future__ import annotations

import pytest
import torch

from foldforge_b200 import kernels
from foldforge_b200.engine import modules, training
from foldforge_b200.engine.modules import Transition


@pytest.mark.parametrize("shape", [(1, 6), (1, 6, 6)])
@pytest.mark.parametrize("key_mask", [torch.tensor([[True, False, True, True, False, True]]),
                                      torch.tensor([[1.0, 0.0, 0.5, 0.99, 2.0, -0.5]]),
                                      torch.tensor([[1, 0, 256, 257, 3, 512]])])
def test_both_passes_read_a_mask_alike(monkeypatch, shape, key_mask):
    seen = []
    monkeypatch.setattr(modules, "_device_reason", lambda *ts: None)
    monkeypatch.setattr(modules, "_library_reason", lambda: None)
    monkeypatch.setattr(training, "transition", lambda x, mask, *args: seen.append(mask))
    module = Transition(16, 2)
    module.set_backend("b200")
    module.set_checkpoint("exact")
    module(torch.randn(*shape, 16, dtype=torch.bfloat16).requires_grad_(), key_mask)
    kept = kernels._mask_u8(key_mask) != 0  # what the kernels read
    assert torch.equal(seen[0], kept if len(shape) == 2 else kept[:, :, None] & kept[:, None, :])
