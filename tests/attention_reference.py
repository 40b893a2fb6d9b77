"""Plain 64-bit forms of the operators around an attention, and bounds on what the kernels' arithmetic may
lose (counted as in ``training_reference``: a rounding to fp32 is off by at most ``STEP`` of its value)."""

from __future__ import annotations

import torch

from training_reference import STEP

Tensor = torch.Tensor
MASK = (1 << 32) - 1


# --------------------------------------------------------------------------- heads
def angles(positions: Tensor, frequencies: list[float], axes: list[int]) -> Tensor:
    """``[.., tokens, 1, pairs]``"""
    f = torch.tensor(frequencies, dtype=torch.float64, device=positions.device)
    return (positions.double()[..., axes] * f)[..., None, :]


def rotate(x: Tensor, angle: Tensor, interleaved: bool) -> Tensor:
    n = angle.shape[-1]
    first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    y = x.clone()
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()
    return y


def partners(x: Tensor, n: int, interleaved: bool) -> Tensor:
    """For each channel the sum of the magnitudes of its pair (its own behind the pairs)."""
    m = x.abs()
    y = m.clone()
    first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    y[..., first] = y[..., second] = m[..., first] + m[..., second]
    return y


def heads(x: Tensor, angle: Tensor, interleaved: bool, weight: Tensor | None = None, eps: float | None = None,
          dy: Tensor | None = None):
    """Forward (and with ``dy`` backward) of one tensor ``[.., tokens, heads, channels]``; ``eps`` None: the rotation alone.
    ``(outputs, bounds)``: y, and dx, dweight."""
    v, n, c = x.double(), angle.shape[-1], x.shape[-1]
    w = torch.ones(c, dtype=torch.float64, device=x.device) if weight is None else weight.double()
    # cosine and sine: the angle's fp32 rounding (at most pi / 4 of a step), the functions (less than 2 steps), and
    # angles found in 64 bits: at most 4 steps of 1; products and the sum: 3 more
    turn = 8 * STEP
    if eps is None:
        y = rotate(v, angle, interleaved)
        outputs, bounds = [y], [turn * partners(v, n, interleaved)]
        if dy is not None:
            g = dy.double()
            outputs.append(rotate(g, -angle, interleaved))
            bounds.append(turn * partners(g, n, interleaved))
        return outputs, bounds
    rstd = (v.square().mean(-1, keepdim=True) + eps).rsqrt()
    normal = v * rstd
    y = rotate(normal * w, angle, interleaved)
    # a head's sum of positive squares: at most 16 additions in a lane and 5 across; the mean, eps, the square root
    # (2 units in the last place) and two products: below 32 steps
    scale = 32 * STEP
    outputs, bounds = [y], [(turn + scale) * partners(normal * w, n, interleaved)]
    if dy is None:
        return outputs, bounds
    g = rotate(dy.double(), -angle, interleaved)
    eg = turn * partners(dy.double(), n, interleaved)
    gw = g * w
    mean = (gw * normal).mean(-1, keepdim=True)
    emean = (w.abs() * eg * normal.abs()).mean(-1, keepdim=True) + 2 * scale * (gw * normal).abs().mean(-1, keepdim=True)
    dx = rstd * (gw - normal * mean)
    edx = rstd * (w.abs() * eg + normal.abs() * emean + 2 * scale * (gw.abs() + (normal * mean).abs()))
    sums = tuple(range(x.dim() - 1))
    rows = x.numel() // c
    # a lane adds its heads of every 4000th token or so one after the other, then 8 warps, blocks and 32 parts
    adds = 256 + rows // 1024
    dw = (g * normal).sum(sums)
    edw = (eg * normal.abs()).sum(sums) + (scale + adds * STEP) * (g * normal).abs().sum(sums)
    return outputs + [dx, dw], bounds + [edx, edw]


# --------------------------------------------------------------------------- dropout
def philox(counter: tuple[int, int, int, int], key: tuple[int, int]) -> tuple[int, int, int, int]:
    """Philox4x32-10 in Python's own integers (Salmon et al., 2011)."""
    c, k = list(counter), list(key)
    for _ in range(10):
        p, q = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(q >> 32) ^ c[1] ^ k[0], q & MASK, (p >> 32) ^ c[3] ^ k[1], p & MASK]
        k = [(k[0] + 0x9E3779B9) & MASK, (k[1] + 0xBB67AE85) & MASK]
    return tuple(c)


def words(index: Tensor, seed: int, offset: int) -> Tensor:
    """The 32-bit words (int64) of mask elements ``index`` (int64, one dimension)."""
    seed, offset = seed % 2**64, offset % 2**64
    group = index // 4
    zero = torch.zeros_like(group)
    c = [group & MASK, group >> 32, zero + (offset & MASK), zero + (offset >> 32)]
    k = [seed & MASK, seed >> 32]
    for _ in range(10):
        p, q = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57  # 64-bit products wrap and keep their bits
        c = [(q >> 32 & MASK) ^ c[1] ^ k[0], q & MASK, (p >> 32 & MASK) ^ c[3] ^ k[1], p & MASK]
        k = [(k[0] + 0x9E3779B9) & MASK, (k[1] + 0xBB67AE85) & MASK]
    return torch.stack(c).gather(0, (index % 4)[None])[0]


def kept(shape, p: float, seed: int, offset: int, shared: tuple[int, ...] = (), device="cuda") -> Tensor:
    """The mask of a tensor of ``shape`` (True: stays)."""
    small = [1 if i in shared else n for i, n in enumerate(shape)]
    index = torch.arange(torch.Size(small).numel(), device=device)
    return (words(index, seed, offset) >= round(p * 2**32)).view(small).expand(shape)


def dropout(x: Tensor, keep: Tensor, p: float, residual: Tensor | None = None):
    """``(out, bound)``: the scale's rounding and the product's, and the sum's."""
    scaled = torch.where(keep, x.double() / (1.0 - p) if p < 1 else 0.0, 0.0)
    out = scaled if residual is None else scaled + residual.double()
    return out, 2 * STEP * scaled.abs() + (0 if residual is None else STEP * (out.abs() + scaled.abs()))
