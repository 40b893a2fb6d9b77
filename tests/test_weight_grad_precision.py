"""What the weight gradient's precision check lets through and what it does not, without a GPU."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import weight_grad_precision as precision


def data(rows, n, k, seed=0):
    g = torch.Generator().manual_seed(seed)
    spread = torch.exp(torch.randn(k, generator=g))
    x = (torch.randn(rows, k, generator=g) * spread + 0.5).bfloat16()
    return (torch.randn(rows, n, generator=g) * 1e-2).bfloat16(), x


def cut(v: np.ndarray) -> np.ndarray:
    """64-bit values cut off to 24 bits."""
    r = v.astype(np.float32)
    return np.where(np.abs(r.astype(np.float64)) > np.abs(v), np.nextafter(r, np.float32(0)), r).astype(np.float64)


def summed(dy, x, chain, splits):
    """The kernel's scheme: chains of additions of 16 rows' products that are cut off, added in fp32."""
    a, b = dy.double().numpy(), x.double().numpy()
    per = -(-a.shape[0] // splits)
    total = np.zeros((a.shape[1], b.shape[1]), dtype=np.float32)
    for first in range(0, a.shape[0], per):
        last, part = min(first + per, a.shape[0]), np.zeros_like(total)
        for start in range(first, last, 16 * chain):
            acc = np.zeros(total.shape)
            for r in range(start, min(start + 16 * chain, last), 16):
                stop = min(r + 16, last)
                acc = cut(acc + a[r:stop].T @ b[r:stop])
            part += acc.astype(np.float32)
        total += part
    return torch.from_numpy(total)


@pytest.mark.parametrize("rows,splits", [(1, 1), (100, 1), (5000, 1), (5000, 80), (20000, 1), (20000, 148)])
def test_the_scheme_passes(rows, splits):
    dy, x = data(rows, 24, 20)
    want, size = precision.definition(dy, x)
    assert precision.worst(summed(dy, x, 32, splits), want, size, rows) <= 1


def test_one_long_chain_does_not():
    dy, x = data(20000, 24, 20)
    want, size = precision.definition(dy, x)
    assert precision.worst(summed(dy, x, 1250, 1), want, size, 20000) > 2


@pytest.mark.parametrize("rows,n,k", [(40000, 64, 64), (40000, 256, 250), (3001, 64, 64)])
def test_a_missing_row_or_a_scaled_result_does_not(rows, n, k):
    dy, x = data(rows, n, k)
    want, size = precision.definition(dy, x)
    assert precision.worst(want.float(), want, size, rows) <= 1
    for row in (0, rows // 2, rows - 1):
        without = want - dy[row].double()[:, None] * x[row].double()
        assert precision.worst(without.float(), want, size, rows) > 100
    assert precision.worst((want * (1 - 1e-5)).float(), want, size, rows) > 2
    one = want.float()
    one[n // 2, k // 3] *= 1 - 1e-3  # a single entry
    assert precision.worst(one, want, size, rows) > 1
