"""Where an update's dropout takes its seed and its kernels from, without a GPU."""

from __future__ import annotations

import pytest
import torch

import attention_reference as ref
from foldforge_b200.engine import training


@pytest.mark.parametrize("device", ["cpu", "meta"])
def test_the_seed_comes_from_the_cpu_generator_whatever_the_default_device(device):
    """``torch.manual_seed`` repeats a mask, and another default device neither changes nor breaks it."""
    residual, update = torch.zeros(2, 5, 5, 8), torch.ones(2, 5, 5, 8)
    torch.manual_seed(13)
    seed = int(torch.empty((), dtype=torch.int64, device="cpu").random_())
    state = torch.random.get_rng_state()
    torch.manual_seed(13)
    with torch.device(device):
        out = training.dropout_add(residual, update, 0.25, -3)
    assert torch.equal(out != 0, ref.kept(update.shape, 0.25, seed, 0, (1,), device="cpu"))
    assert torch.equal(torch.random.get_rng_state(), state)  # one draw
