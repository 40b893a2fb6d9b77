"""Where an update's dropout takes its seed and its kernels from, without a GPU."""

from __future__ import annotations

import pytest
import torch

import attention_reference as ref
from foldforge_b200 import _lib
from foldforge_b200.engine import modules, training


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


class OnB200:
    """What the choice of a kernel looks at, of a tensor on a B200."""

    is_cuda, dtype, device = True, torch.bfloat16, torch.device("cuda", 0)


@pytest.mark.parametrize("missing", ["load", "binding"])
def test_without_the_kernels_the_integer_form_serves(monkeypatch, missing):
    monkeypatch.setattr(torch.cuda, "get_device_capability", lambda device=None: (10, 0))
    there = object()
    monkeypatch.setattr(_lib, "load", lambda: there)
    monkeypatch.setattr(_lib, "binding", lambda: there)
    assert training._on_b200(OnB200(), OnB200())

    def not_built():
        raise _lib.LibraryMissing("not built")

    monkeypatch.setattr(_lib, "binding", not_built)
    if missing == "load":
        monkeypatch.setattr(_lib, "load", not_built)
    assert not training._on_b200(OnB200())


def test_qk_norm_refuses_b200_without_the_torch_facing_calls(monkeypatch):
    """The library alone does not serve it: its calls go through the binding."""
    monkeypatch.setattr(modules, "_cuda_reason", lambda *ts: None)
    monkeypatch.setattr(_lib, "load", lambda: object())
    norm = modules.QKNorm(8, elementwise_affine=False)
    norm.set_backend("b200")
    q = torch.randn(3, 2, 8)
    monkeypatch.setattr(_lib, "binding", lambda: object())
    assert norm.unsupported(q, q) is None

    def not_built():
        raise _lib.LibraryMissing("the calls are not built")

    monkeypatch.setattr(_lib, "binding", not_built)
    assert norm.unsupported(q, q) == "the calls are not built"
