"""LayerNorm's training forward pass: rows that do not vary, and beside the pass without gradients (B200 only)."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

import training_reference as ref  # noqa: E402
from foldforge_b200 import _lib, kernels  # noqa: E402

BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    torch.cuda.synchronize()
    assert _lib.device_error() == 0


def gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("c", [1, 7, 8, 15, 24, 40, 100, 127, 128, 129, 358, 384, 520, 1000, 1024, 1200, 2047, 2056, 4096,
                               5003, 8191, 8192])
def test_rows_that_do_not_vary(c, dtype):
    """Their mean is their value to the last bit, so y is the bias and no gradient of the weight has a share,
    whatever the width and the value (c equal values whose sum rounds among them)."""
    values = torch.tensor([1000.0, 0.1, -1234.567, 1e-30, 7.0, 1e34, -1e30, 1.0 / 3.0, 0.0, 65537.0], device="cuda")
    x = values[:, None].expand(10, c).to(dtype).contiguous()
    w, b = torch.full((c,), 3.0, device="cuda"), torch.randn(c, device="cuda", generator=gen(c))
    for mx in (False, True):
        y, saved = kernels.layer_norm_train(x, w, b, checkpoint=mx)
        assert torch.equal(saved.stats[0], x[:, 0].float())
        assert torch.equal(y, b.to(dtype).expand(10, c))
    dy = torch.randn(10, c, device="cuda", generator=gen(c + 1)).to(dtype)
    _, dw, _ = kernels.layer_norm_backward(dy, kernels.layer_norm_train(x, w, b)[1], w)
    assert torch.equal(dw, torch.zeros_like(dw))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("c", [7, 40, 96, 128, 129, 384, 1024, 1200, 4096, 8191])
def test_beside_the_pass_without_gradients(c, dtype):
    """Another kernel with another order of sums: both are within the arithmetic's bound of the definition,
    also where the mean is large beside the deviations and where the first channel stands out."""
    g = gen(c)
    w, b = 1 + 0.3 * torch.randn(c, device="cuda", generator=g), torch.randn(c, device="cuda", generator=g)
    x = torch.randn(60, c, device="cuda", generator=g)
    x[20:40] += 300.0
    x[40:, 0] = 1000.0
    x = x.to(dtype)
    (want, *_), (bound, *_) = ref.layer_norm(x, torch.zeros_like(x), w, b, 1e-5, False)
    for y in (kernels.layer_norm_train(x, w, b)[0], kernels.layer_norm(x, w, b)):
        assert ref.worst(y, want, bound, dtype) <= 1
