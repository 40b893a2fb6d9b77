"""A Transition too wide for its weight gradients is refused before its forward pass, not in its backward pass."""

from __future__ import annotations

import pytest
import torch

from foldforge_b200.engine import modules
from foldforge_b200.engine.modules import Transition


@pytest.mark.parametrize("d,n,taken", [(8, 1 << 16, True), (8, (1 << 16) + 2, False), (8192, 64, True), (8192, 65, False)])
def test_hidden_channels(monkeypatch, d, n, taken):
    monkeypatch.setattr(modules, "_device_reason", lambda *ts: None)
    monkeypatch.setattr(modules, "_library_reason", lambda: None)
    with torch.device("meta"):
        module = Transition(d, n)
    module.set_backend("b200")
    module.set_checkpoint("exact")
    reason = module.unsupported(torch.zeros(1, 2, d, dtype=torch.bfloat16, requires_grad=True))
    assert reason is None if taken else "hidden channels" in reason
