"""How near a weight gradient's sums have to come to the definition, by norms of its rows and columns.

The tensor cores cut the accumulator off after each addition of 16 rows' products: at most a step 2^-23 of it,
half of that on average. 32 additions make a chain (512 rows); a chain's accumulator is a random walk, of 2/3
of its last size on average, so a chain's sum is off by 32 * 2/3 * 2^-24 of its size. The chains' sums are then
added in fp32, at most ``rows / 512 + 148`` of them one after the other, each rounded to nearest: independent errors
of at most 2^-24, which grow as a random walk does. Errors of a row or column of dW are compared by their norm with
the norm of its entries and of the random walk of their terms together.
"""

from __future__ import annotations

import torch

Tensor = torch.Tensor


def tolerance(rows: int) -> float:
    chain = min(32, -(-rows // 16))
    return (chain * 2 / 3 + (-(-rows // 512) + 148) ** 0.5) * 2.0**-24


def definition(dy: Tensor, x: Tensor) -> tuple[Tensor, Tensor]:
    """``dy^T x`` in 64 bits and the size of its entries."""
    dy, x = dy.double(), x.double()
    want = dy.t() @ x
    return want, (want.square() + dy.square().t() @ x.square()).sqrt()


def worst(got: Tensor, want: Tensor, size: Tensor, rows: int) -> float:
    """The largest error of a row's or column's norm in units of the tolerance (at most 1 where the sums are right)."""
    error = got.double() - want
    return max((error.norm(dim=d) / size.norm(dim=d).clamp_min(1e-300)).max().item() for d in (0, 1)) / tolerance(rows)
