"""Backward passes form the gradients that are asked for and no others (the kernels have stand-ins in 64 bits)."""

from __future__ import annotations

import itertools

import pytest
import torch

from foldforge_b200 import kernels
from foldforge_b200.engine import training
from foldforge_b200.engine.modules import LayerNorm, Transition
from test_engine_training import on_device, plain_kernels, reference_transition  # noqa: F401 - fixtures

DOUBLE = torch.float64
GROUPS = {"x": (), "norm": ("ln_in.weight", "ln_in.bias"), "expand": ("expand_a.weight", "expand_b.weight"),
          "squeeze": ("squeeze.weight",)}


@pytest.fixture
def calls(plain_kernels, monkeypatch):  # noqa: F811
    """The kernels called, with what was asked of them."""
    seen = []
    norm_backward, gate_backward, weight_grad = kernels.layer_norm_backward, kernels.swiglu_backward, kernels.weight_grad

    def norm(dy, saved, weight, *, weight_gradient=True, bias=True, residual=None):
        seen.append(("norm", weight is not None and weight_gradient, bias))
        dx, dweight, dbias = norm_backward(dy, saved, weight, bias=bias, residual=residual)
        return dx, dweight if weight_gradient else None, dbias

    def gate(dh, ab, *, output=False):
        seen.append(("gate", output))
        return gate_backward(dh, ab, output=output)

    def wgrad(dy, x):
        seen.append(("weight_grad", dy.shape[-1]))
        return weight_grad(dy, x)

    monkeypatch.setattr(kernels, "layer_norm_backward", norm)
    monkeypatch.setattr(kernels, "swiglu_backward", gate)
    monkeypatch.setattr(kernels, "weight_grad", wgrad)
    return seen


@pytest.mark.parametrize("wanted", [w for n in range(1, 5) for w in itertools.combinations(GROUPS, n)])
@pytest.mark.parametrize("rows", [5, 0])
def test_transition(calls, monkeypatch, wanted, rows):
    monkeypatch.setattr(training, "CHUNK_ROWS", 3)
    g = torch.Generator().manual_seed(1)
    module = Transition(16, 2)
    for p in module.parameters():
        p.data = torch.randn(p.shape, generator=g, dtype=DOUBLE) * 0.5
    named = dict(module.named_parameters())
    asked = [named[name] for group in wanted for name in GROUPS[group]]
    for p in named.values():
        p.requires_grad_(any(p is a for a in asked))
    module.set_backend("b200")
    module.set_checkpoint("exact")
    x = torch.randn(1, rows, 16, generator=g, dtype=DOUBLE, requires_grad="x" in wanted)
    dy = torch.randn(x.shape, generator=g, dtype=DOUBLE)
    leaves = [*([x] if "x" in wanted else []), *asked]
    got = torch.autograd.grad(module(x), leaves, dy)
    for a, b in zip(got, torch.autograd.grad(reference_transition(module, x, None), leaves, dy)):
        torch.testing.assert_close(a, b.to(a.dtype))
    names = [c[0] for c in calls]
    if rows == 0:
        assert not calls
        return
    assert ("norm" in names) == ("x" in wanted or "norm" in wanted)
    assert all(c[1:] == ("norm" in wanted,) * 2 for c in calls if c[0] == "norm")
    assert all(c[1] == ("squeeze" in wanted) for c in calls if c[0] == "gate")
    assert (("weight_grad", 64) in calls) == ("expand" in wanted)
    assert (("weight_grad", 16) in calls) == ("squeeze" in wanted)


@pytest.mark.parametrize("wanted", [("x",), ("weight",), ("bias",), ("x", "weight"), ("x", "bias"), ("x", "weight", "bias")])
def test_layer_norm(calls, wanted):
    g = torch.Generator().manual_seed(2)
    norm = LayerNorm(40)
    for p in norm.parameters():
        p.data = torch.randn(p.shape, generator=g, dtype=DOUBLE)
    norm.weight.requires_grad_("weight" in wanted)
    norm.bias.requires_grad_("bias" in wanted)
    x = torch.randn(3, 40, generator=g, dtype=DOUBLE, requires_grad="x" in wanted)
    dy = torch.randn(3, 40, generator=g, dtype=DOUBLE)
    leaves = [{"x": x, "weight": norm.weight, "bias": norm.bias}[name] for name in wanted]
    got = torch.autograd.grad(training.layer_norm(x, norm.weight, norm.bias, norm.eps, "exact"), leaves, dy)
    want = torch.autograd.grad(torch.nn.functional.layer_norm(x, (40,), norm.weight, norm.bias, norm.eps), leaves, dy)
    for a, b in zip(got, want):
        torch.testing.assert_close(a, b)
    assert calls == [("norm", "weight" in wanted, "bias" in wanted)]
