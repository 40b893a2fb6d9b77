"""Where an update's dropout takes its seed and its kernels from (B200 only)."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

from foldforge_b200 import _lib, kernels  # noqa: E402
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


def test_without_the_kernels_the_integer_form_serves(monkeypatch):
    """An op on the pytorch backend needs no library for its dropout, forward or backward."""
    g = torch.Generator(device="cuda").manual_seed(2)
    residual, update = (torch.randn(1, 9, 9, 32, device="cuda", generator=g).requires_grad_() for _ in range(2))
    dout = torch.randn(1, 9, 9, 32, device="cuda", generator=g)

    def step():
        torch.manual_seed(3)
        out = training.dropout_add(residual, update, 0.25, -2)
        return out, *torch.autograd.grad(out, (residual, update), dout)

    want = step()

    def not_built():
        raise _lib.LibraryMissing("not built")

    monkeypatch.setattr(_lib, "binding", not_built)
    with pytest.raises(_lib.LibraryMissing):
        kernels.dropout_train(update.detach(), 0.25, 1)
    assert all(torch.equal(a, b) for a, b in zip(step(), want, strict=True))
