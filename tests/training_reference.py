"""Plain 64-bit forms of the training operators, and bounds on what the kernels' arithmetic may lose.

A bound counts roundings: ``eps / 2`` relative for the one to the output's type, and for the fp32
arithmetic before it a number of steps of 2^-24 relative to the magnitudes that enter the sums.
"""

from __future__ import annotations

import torch

Tensor = torch.Tensor
STEP = 2.0**-24  # half a step of fp32
BLOCK = 32


def half_step(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def rounded_to_8_bits(x: Tensor) -> Tensor:
    """The values (fp64) that an 8-bit checkpoint of ``x [rows, c]`` stands for: blocks of 32 channels,
    the smallest power of two that brings the largest finite magnitude to at most 448, then the nearest
    of e4m3's values (ties to the even one), looked up in a table of all of them."""
    codes = torch.arange(256, dtype=torch.uint8, device=x.device).view(torch.float8_e4m3fn).double()
    positive = codes[:127]  # ascending from 0 to 448; odd code = odd last bit
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for first in range(0, x.shape[1], BLOCK):
        v = x[:, first:first + BLOCK].double()
        finite = torch.isfinite(v)
        top = torch.where(finite, v.abs(), 0.0).amax(1, keepdim=True)
        e = torch.full_like(top, -127.0)
        for _ in range(512):
            small = top > 448.0 * torch.exp2(e)
            if not small.any():
                break
            e = torch.where(small, e + 1, e)
        m = torch.where(finite, v.abs(), 0.0) / torch.exp2(e)
        hi = torch.searchsorted(positive, m.contiguous()).clamp_max(126)
        lo = (hi - 1).clamp_min(0)
        up, down = positive[hi] - m, m - positive[lo]
        pick = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
        value = torch.copysign(positive[pick], v) * torch.exp2(e)
        out[:, first:first + BLOCK] = torch.where(finite, value, float("nan"))
    return out


def layer_norm(x: Tensor, dy: Tensor, weight: Tensor | None, bias: Tensor | None, eps: float, mx: bool,
               residual: Tensor | None = None):
    """``(y, dx, dweight, dbias)`` in 64 bits and the bounds of their fp32 arithmetic."""
    v, g = x.double(), dy.double()
    c = x.shape[1]
    w = torch.ones(c, dtype=torch.float64, device=x.device) if weight is None else weight.double()
    b = torch.zeros(c, dtype=torch.float64, device=x.device) if bias is None else bias.double()
    mean = v.mean(1, keepdim=True)
    rstd = ((v - mean).square().mean(1, keepdim=True) + eps).rsqrt()
    y = (v - mean) * rstd * w + b
    xh = ((rounded_to_8_bits(x) if mx else v) - mean) * rstd
    gw = g * w
    c1, c2 = gw.mean(1, keepdim=True), (gw * xh).mean(1, keepdim=True)
    dx = rstd * (gw - c1 - xh * c2)
    if residual is not None:
        dx = dx + residual.double()
    # a row's fp32 sums take at most 32 + 8 + 8 additions; with the subtraction, the square, the square
    # root and the scaling fewer than 128 roundings reach xh, each relative to the row's largest |x| rstd
    # (and to |xh|, which |x - mean| <= 2 max|x| bounds by twice that)
    size = v.abs().amax(1, keepdim=True) * rstd
    exh = 128 * STEP * (size + xh.abs())
    ey = exh * w.abs() + 4 * STEP * (y.abs() + b.abs())
    ec2 = (gw.abs() * exh).mean(1, keepdim=True) + 64 * STEP * (gw * xh).abs().mean(1, keepdim=True)
    edx = rstd * (64 * STEP * (gw.abs() + gw.abs().mean(1, keepdim=True)) + exh * c2.abs() + xh.abs() * ec2) \
        + 128 * STEP * (dx.abs() + (rstd * gw).abs() + (rstd * xh * c2).abs())
    if residual is not None:
        edx = edx + STEP * residual.double().abs()
    # rows of a column: fewer than 512 additions one after the other for the rows tested here
    dweight, dbias = (g * xh).sum(0), g.sum(0)
    edw = (g.abs() * exh).sum(0) + 512 * STEP * (g * xh).abs().sum(0)
    edb = 512 * STEP * g.abs().sum(0)
    return (y, dx, dweight, dbias), (ey, edx, edw, edb)


def swiglu(ab: Tensor, dh: Tensor, mx: bool):
    """``(h, dab, h from what was kept)`` in 64 bits and the bounds of their fp32 arithmetic: the
    exponential is off by at most 2 units in the last place and enters the sigmoid's relative error, fewer
    than 16 roundings follow, each relative to the product's magnitude before the sum 1 + a (1 - s)."""
    half = ab.shape[1] // 2

    def unit(t: Tensor):
        a, b = t[:, :half], t[:, half:]
        return a, b, torch.sigmoid(a)

    a, b, s = unit(ab.double())
    h = a * s * b
    ka, kb, ks = unit(rounded_to_8_bits(ab) if mx else ab.double())
    d = dh.double()
    # 1 - sigmoid(a) = sigmoid(-a), without the cancellation
    da, db = d * kb * ks * (1 + ka * torch.sigmoid(-ka)), d * ka * ks
    kept = ka * ks * kb
    eda = 16 * STEP * (d * kb * ks).abs() * (1 + ka.abs())
    bounds = (16 * STEP * h.abs(), torch.cat([eda, 16 * STEP * db.abs()], 1), 16 * STEP * kept.abs())
    return (h, torch.cat([da, db], 1), kept), bounds


def weight_grad(dy: Tensor, x: Tensor, mx: bool):
    """``dy^T x`` in 64 bits and its bound: products of bf16 values are exact in fp32, the tensor cores add
    them 16 rows at a time (one rounding or truncation, at most a whole step 2^-23, for each of the 16 and
    for each addition to the accumulator), then at most 148 partial sums are added."""
    v = rounded_to_8_bits(x) if mx else x.double()
    adds = 16 + -(-dy.shape[0] // 16) + 148
    return dy.double().t() @ v, 2 * adds * STEP * (dy.double().abs().t() @ v.abs())


def worst(got: Tensor, want: Tensor, bound: Tensor, dtype: torch.dtype) -> float:
    """The largest error in units of its bound (at most 1 where the kernel is right). A result below the
    type's normal range may be off by half its smallest step."""
    info = torch.finfo(dtype)
    allowed = bound + half_step(dtype) * (want.abs() + bound) + info.smallest_normal * info.eps
    return ((got.double() - want).abs() / allowed).max().item() if got.numel() else 0.0
