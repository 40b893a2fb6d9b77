"""The weight gradient's sums against the definition in 64 bits, by norms (B200 only)."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

import training_reference as ref  # noqa: E402
import weight_grad_precision as precision  # noqa: E402
from foldforge_b200 import _lib, kernels  # noqa: E402

BF16 = torch.bfloat16


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("rows,n,k", [(1, 8, 16), (63, 7, 9), (129, 1536, 384), (512, 1536, 384), (1000, 512, 128), (3001, 64, 64),
                                      (20000, 40, 72), (20000, 2048, 2048), (40000, 64, 64), (40000, 256, 250), (90000, 129, 68),
                                      (512 * 512, 512, 128)])
def test_sums(rows, n, k, mx):
    g = torch.Generator(device="cuda").manual_seed(rows + 7 * n + k)
    spread = torch.exp(torch.randn(k, device="cuda", generator=g))
    x = (torch.randn(rows, k, device="cuda", generator=g) * spread + 0.5).to(BF16)
    dy = (torch.randn(rows, n, device="cuda", generator=g) * 1e-2).to(BF16)
    got = kernels.weight_grad(dy, kernels.checkpoint_pack(x) if mx else x)
    want, size = precision.definition(dy, ref.rounded_to_8_bits(x) if mx else x)
    assert precision.worst(got, want, size, rows) <= 1
    torch.cuda.synchronize()
    assert _lib.device_error() == 0
