"""Where an update's dropout takes its seed and its kernels from (B200 only)."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

from foldforge_b200.engine import training  # noqa: E402


def test_the_seed_comes_from_the_cpu_generator_whatever_the_default_device():
    residual, update = torch.randn(1, 6, 6, 32), torch.randn(1, 6, 6, 32)
    torch.manual_seed(13)
    want = training.dropout_add(residual, update, 0.25, -3)
    torch.manual_seed(13)
    state = torch.cuda.get_rng_state()
    with torch.device("cuda"):
        got = training.dropout_add(residual.cuda(), update.cuda(), 0.25, -3)
    assert torch.equal(got.cpu(), want) and torch.equal(torch.cuda.get_rng_state(), state)
