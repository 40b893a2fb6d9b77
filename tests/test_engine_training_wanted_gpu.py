"""A gradient is the same whichever others are formed beside it (B200 only)."""

from __future__ import annotations

import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu

from foldforge_b200 import _lib, kernels  # noqa: E402
from foldforge_b200.engine import factories  # noqa: E402
from foldforge_b200.engine.modules import Transition  # noqa: E402

BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    torch.cuda.synchronize()
    assert _lib.device_error() == 0


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("rows,c", [(0, 16), (3, 7), (3, 128), (3000, 128), (700, 129), (50, 1200)])
def test_layer_norm_backward(rows, c, mx):
    g = torch.Generator(device="cuda").manual_seed(rows + c)
    x, dy = (torch.randn(rows, c, device="cuda", generator=g).to(BF16) for _ in range(2))
    w, b = torch.randn(c, device="cuda", generator=g), torch.randn(c, device="cuda", generator=g)
    _, saved = kernels.layer_norm_train(x, w, b, checkpoint=mx)
    dx, dw, db = kernels.layer_norm_backward(dy, saved, w)
    for weight_gradient, bias in itertools.product((False, True), repeat=2):
        one, two, three = kernels.layer_norm_backward(dy, saved, w, weight_gradient=weight_gradient, bias=bias)
        assert torch.equal(one, dx)
        assert torch.equal(two, dw) if weight_gradient else two is None
        assert torch.equal(three, db) if bias else three is None


@pytest.mark.parametrize("kind", ["exact", "mxfp8"])
@pytest.mark.parametrize("make,shape", [(lambda: Transition(128, 4), (1, 20, 20, 128)), (lambda: Transition(64, 4), (3, 50, 64)),
                                        (lambda: factories.layer_norm(128), (700, 128))])
def test_modules(make, shape, kind):
    torch.manual_seed(1)
    module = make().cuda()
    module.set_backend("b200")
    module.set_checkpoint(kind)
    x, dy = torch.randn(shape, device="cuda").to(BF16), torch.randn(shape, device="cuda").to(BF16)
    params = list(module.parameters())

    def grads(wanted):
        for i, p in enumerate(params):
            p.requires_grad_(i in wanted)
        leaf = x.clone().requires_grad_(-1 in wanted)
        leaves = [leaf if i < 0 else params[i] for i in wanted]
        return dict(zip(wanted, torch.autograd.grad(module(leaf), leaves, dy)))

    every = range(-1, len(params))
    want = grads(every)
    for wanted in [(-1,), *((i,) for i in range(len(params))), tuple(range(len(params))), (-1, len(params) - 1)]:
        for i, got in grads(wanted).items():
            assert torch.equal(got, want[i]), (wanted, i)
