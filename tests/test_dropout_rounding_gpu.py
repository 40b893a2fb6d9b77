"""Dropout's arithmetic: an update over 1 - p is rounded to fp32 before the residual is added, so that a sum which
lies half way between two values rounds as its definition does, and as the engine's integer form does (B200 only)."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

import attention_reference as ref  # noqa: E402
from foldforge_b200 import kernels  # noqa: E402
from foldforge_b200.engine import training  # noqa: E402

BF16, F32 = torch.bfloat16, torch.float32

# every kernel: an element for itself with and without a rest, a mask shared by rows of whole vectors and of single
# elements, masks closer than 32 elements, tensors off 16 bytes
PLACES = [((4, 512), None, 0), ((37, 111), None, 0), ((3, 9, 64), 1, 0), ((3, 9, 33), 1, 0), ((3, 9, 8), 1, 0), ((3, 9, 4), 1, 0),
          ((4, 512), None, 1), ((3, 9, 64), 1, 1)]


def placed(t, off):
    """``t`` in memory that starts ``off`` elements behind an allocation's beginning"""
    return torch.empty(t.numel() + off, device="cuda", dtype=t.dtype)[off:].view(t.shape).copy_(t)


@pytest.mark.parametrize("shape,shared,off", PLACES)
@pytest.mark.parametrize("dtype,out_dtype", [(BF16, BF16), (F32, BF16), (BF16, F32), (F32, F32)])
def test_a_sum_half_way_between_two_values(shape, shared, off, dtype, out_dtype):
    """255 over 3 / 4 is 340, and 340 - 127.5 = 212.5: in bf16 the even one of 212 and 213. The fp32 number next to 4 / 3 is
    too large by 2^-25 of itself: the product unrounded, the sum would be 212.500015 and round to 213."""
    x = placed(torch.full(shape, 255.0, dtype=dtype), off)
    residual = placed(torch.full(shape, -127.5, dtype=out_dtype), off)
    out, _ = kernels.dropout_train(x, 0.25, 3, residual=residual, shared=shared)
    keep = ref.kept(shape, 0.25, 3, 0, () if shared is None else (shared,))
    want = torch.where(keep, 212.0 if out_dtype == BF16 else 212.5, -127.5).to(out_dtype)
    assert torch.equal(out, want)


@pytest.mark.parametrize("p", [0.05, 0.1, 0.15, 0.25, 0.5])
@pytest.mark.parametrize("shape,shared,off", PLACES)
@pytest.mark.parametrize("dtype,out_dtype", [(BF16, BF16), (F32, BF16), (F32, F32)])
def test_each_operation_rounds(shape, shared, off, dtype, out_dtype, p):
    """Bit for bit a product in fp32, a sum in fp32 and one rounding to the output's type."""
    g = torch.Generator(device="cuda").manual_seed(5)
    x = placed((3 * torch.randn(shape, device="cuda", generator=g)).to(dtype), off)
    residual = placed((3 * torch.randn(shape, device="cuda", generator=g)).to(out_dtype), off)
    keep = ref.kept(shape, p, 8, 0, () if shared is None else (shared,))
    update = torch.where(keep, x.float() * (1.0 / (1.0 - p)), 0.0)
    out, saved = kernels.dropout_train(x, p, 8, residual=residual, shared=shared)
    assert torch.equal(out, (residual.float() + update).to(out_dtype))
    alone, _ = kernels.dropout_train(x, p, 8, shared=shared)
    assert torch.equal(alone, update.to(dtype))
    dout = residual
    assert torch.equal(kernels.dropout_backward(dout, saved), torch.where(keep, dout.float() * (1.0 / (1.0 - p)), 0.0).to(dtype))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_the_same_numbers_on_both_machines(dtype):
    g = torch.Generator().manual_seed(6)
    residual, update = torch.randn(2, 30, 30, 128, generator=g).to(dtype), torch.randn(2, 30, 30, 128, generator=g)
    torch.manual_seed(4)
    host = training.dropout_add(residual, update, 0.25, -3)
    torch.manual_seed(4)
    assert torch.equal(training.dropout_add(residual.cuda(), update.cuda(), 0.25, -3).cpu(), host)
