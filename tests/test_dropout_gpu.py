"""Dropout from a counter-based generator against its definition (B200 only)."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

import attention_reference as ref  # noqa: E402
from foldforge_b200 import _lib, kernels  # noqa: E402
from training_reference import worst  # noqa: E402

BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    torch.cuda.synchronize()
    assert _lib.device_error() == 0


def gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def values(g, *shape, dtype=BF16):
    return (1.5 * torch.randn(shape, device="cuda", generator=g) + 0.2).to(dtype)


def run(x, p, seed, offset=0, residual=None, shared=None):
    out, saved = kernels.dropout_train(x, p, seed, offset=offset, residual=residual, shared=shared)
    axes = () if shared is None else tuple(i % x.dim() for i in ((shared,) if isinstance(shared, int) else shared))
    keep = ref.kept(x.shape, p, seed, offset, axes)
    want, bound = ref.dropout(x, keep, p, residual)
    out_dtype = x.dtype if residual is None else residual.dtype
    assert out.dtype == out_dtype and out.shape == x.shape
    assert worst(out, want, bound, out_dtype) <= 1
    dropped = torch.zeros_like(out) if residual is None else residual
    assert torch.equal(out[~keep], dropped[~keep])
    dout = values(gen(99), *x.shape, dtype=out_dtype)
    dx = kernels.dropout_backward(dout, saved)
    want, bound = ref.dropout(dout, keep, p)
    assert dx.dtype == x.dtype and worst(dx, want, bound, x.dtype) <= 1
    assert not dx[~keep].any()
    return out


@pytest.mark.parametrize("residual", [None, BF16, F32])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shape", [(1,), (3,), (8,), (1, 384), (2, 31), (7, 33), (77, 390), (5, 1, 9), (1000, 128), (333, 129),
                                   (64, 4096), (20000, 37)])
def test_every_element_for_itself(shape, dtype, residual):
    g = gen(sum(shape))
    x = values(g, *shape, dtype=dtype)
    run(x, 0.2, 7 + sum(shape), 3, None if residual is None else values(g, *shape, dtype=residual))


@pytest.mark.parametrize("dtype,residual", [(BF16, BF16), (F32, BF16), (F32, None)])
@pytest.mark.parametrize("shape,shared", [
    ((1, 40, 40, 128), 1), ((1, 40, 40, 128), 2), ((2, 31, 31, 33), 1), ((2, 31, 31, 33), 2), ((2, 31, 31, 33), -1),
    ((3, 17, 64), 0), ((3, 17, 64), -1), ((3, 17, 64), (0, 1)), ((3, 17, 64), (1, 2)), ((3, 17, 64), (0, 1, 2)), ((5, 7, 6, 11), (1, 2)),
    ((4, 9, 8), (1,)), ((1000, 3), 0), ((2, 5000, 4), 1), ((1, 1, 16), 1), ((300, 1), 0), ((2, 3, 12), 1), ((2, 3, 20), 0),
])
def test_shared_masks(shape, shared, dtype, residual):
    g = gen(len(shape) * 100 + shape[-1])
    x = values(g, *shape, dtype=dtype)
    run(x, 0.25, 123456789012345, 5, None if residual is None else values(g, *shape, dtype=residual), shared)


@pytest.mark.parametrize("p", [0.0, 1e-9, 0.5, 0.999, 1.0])
@pytest.mark.parametrize("seed,offset", [(0, 0), (1, 0), (-1, -1), (2**63 - 1, 2**40 + 3), (2**64 - 1, 2**32)])
def test_rates_and_seeds(p, seed, offset):
    x = values(gen(1), 300, 40)
    out = run(x, p, seed, offset)
    if p == 0:
        assert torch.equal(out, x)
    if p == 1:
        assert not out.any()


def test_how_many_stay():
    """The share of kept elements lies within five standard deviations, and masks of other seeds, offsets or
    places agree as often as chance has them agree."""
    n, p = 1 << 22, 0.25
    x = torch.ones(n, device="cuda", dtype=BF16)
    masks = [kernels.dropout_train(x, p, s, offset=o)[0] != 0 for s, o in ((1, 0), (2, 0), (1, 1), (1, 2**32))]
    deviation = (p * (1 - p) / n) ** 0.5
    for m in masks:
        assert abs(m.float().mean().item() - (1 - p)) < 5 * deviation
    same = p * p + (1 - p) * (1 - p)
    for a, b in ((0, 1), (0, 2), (0, 3), (1, 2)):
        agree = (masks[a] == masks[b]).float().mean().item()
        assert abs(agree - same) < 5 * (same * (1 - same) / n) ** 0.5
    shifted = (masks[0][1:] == masks[0][:-1]).float().mean().item()
    assert abs(shifted - same) < 6 * (same * (1 - same) / n) ** 0.5


def test_dropped_values_count_as_zero_whatever_they_hold():
    x = values(gen(2), 64, 100)
    keep = ref.kept(x.shape, 0.3, 11, 0)
    bad = torch.where(keep, x, torch.tensor(float("nan"), device="cuda", dtype=BF16))
    bad[0, :50] = torch.where(keep[0, :50], x[0, :50], torch.tensor(float("inf"), device="cuda", dtype=BF16))
    residual = values(gen(3), 64, 100)
    want = kernels.dropout_train(x, 0.3, 11, residual=residual)[0]
    got, saved = kernels.dropout_train(bad, 0.3, 11, residual=residual)
    assert torch.equal(got, want)
    assert bool(torch.isfinite(kernels.dropout_backward(bad, saved)).all())
    x[keep] = float("inf")
    out, _ = kernels.dropout_train(x, 0.3, 11, residual=residual)
    assert bool(torch.isinf(out[keep]).all()) and torch.equal(out[~keep], residual[~keep])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_any_layout(dtype):
    """A mask belongs to places, not to memory: views give what their dense copies give."""
    g = gen(4)
    wide = values(g, 40, 96, dtype=dtype)
    for x in (wide[:, 8:72], wide.t(), wide.view(-1)[1:1 + 33 * 37].view(33, 37), wide.view(4, 10, 96).transpose(0, 1), wide[::2],
              wide[:1].expand(9, 96)):
        for shared in (None, 0):
            residual = values(g, *x.shape, dtype=BF16)
            got = kernels.dropout_train(x, 0.4, 5, residual=residual, shared=shared)[0]
            off = torch.empty(residual.numel() + 1, device="cuda", dtype=BF16)[1:].view(residual.shape).copy_(residual)
            dense = x.contiguous().clone()
            assert torch.equal(got, kernels.dropout_train(dense, 0.4, 5, residual=off, shared=shared)[0])
            assert torch.equal(got, kernels.dropout_train(dense, 0.4, 5, residual=residual.t().contiguous().t() if x.dim() == 2
                                                          else residual, shared=shared)[0])


@pytest.mark.parametrize("shape", [(0,), (4, 0), (0, 8)])
def test_nothing_to_do(shape):
    x = torch.empty(shape, device="cuda", dtype=BF16)
    out, saved = kernels.dropout_train(x, 0.1, 3, residual=x)
    assert out.shape == x.shape and kernels.dropout_backward(out, saved).shape == x.shape


def test_seed_on_the_device():
    x = values(gen(6), 50, 70)
    seed = torch.tensor([77, 4], device="cuda")
    want = kernels.dropout_train(x, 0.3, 77, offset=9)[0]
    got, saved = kernels.dropout_train(x, 0.3, seed, offset=5)
    assert torch.equal(got, want)
    assert torch.equal(kernels.dropout_backward(x, saved), kernels.dropout_backward(x, saved._replace(seed=77, offset=9)))
    negative = torch.tensor([-3, -1], device="cuda")
    assert torch.equal(kernels.dropout_train(x, 0.3, negative)[0], kernels.dropout_train(x, 0.3, -3, offset=2**64 - 1)[0])


def test_captured_steps_draw_new_masks():
    """A captured forward and backward pass reads its seed when it replays."""
    x, residual = values(gen(7), 100, 64), values(gen(8), 100, 64)
    seed = torch.tensor([5, 0], device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, saved = kernels.dropout_train(x, 0.5, seed, residual=residual)
        dx = kernels.dropout_backward(x, saved)
        seed[1] += 1
    seen = []
    for step in range(3):
        graph.replay()
        want, eager = kernels.dropout_train(x, 0.5, 5, offset=step, residual=residual)
        assert torch.equal(out, want) and torch.equal(dx, kernels.dropout_backward(x, eager))
        seen.append(out.clone())
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])


def test_other_stream():
    x = values(gen(9), 3000, 128)
    want = kernels.dropout_train(x, 0.1, 2)[0]
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        got = kernels.dropout_train(x, 0.1, 2)[0]
    torch.cuda.current_stream().wait_stream(other)
    assert torch.equal(got, want)


@pytest.mark.parametrize("shared,inner", [(None, 1), (1, 2**20 + 1)])
def test_elements_past_32_bits(shared, inner):
    """2^31 and more elements: the last ones' masks."""
    shape = (2**31 + 4099,) if shared is None else (3, 700, inner)
    x = torch.ones(shape, device="cuda", dtype=BF16)
    out, saved = kernels.dropout_train(x, 0.5, 21, shared=shared)
    dx = kernels.dropout_backward(x, saved)
    if shared is None:
        index = torch.arange(2**31 - 2000, 2**31 + 4099, device="cuda")
        keep = ref.words(index, 21, 0) >= 2**31
        assert torch.equal(out[index[0]:] != 0, keep)
    else:
        keep = ref.kept(shape, 0.5, 21, 0, (1,))
        for row in (0, 1, 698, 699):
            assert torch.equal(out[2, row] != 0, keep[2, 0])
    assert torch.equal(out, dx)


def test_narrow_shared_rows_and_views_past_32_bits():
    """2^31 and more elements where masks lie closer than rows of 32, and a tensor that starts off 16 bytes."""
    shape = (180_000_000, 3, 4)
    x = torch.ones(shape, device="cuda", dtype=BF16)
    out = kernels.dropout_train(x, 0.5, 8, shared=1)[0]
    index = torch.arange((shape[0] - 1000) * 4, shape[0] * 4, device="cuda")
    keep = (ref.words(index, 8, 0) >= 2**31).view(1000, 1, 4).expand(1000, 3, 4)
    assert torch.equal(out[-1000:] != 0, keep)
    del out
    flat = x.view(-1)[1:]
    out = kernels.dropout_train(flat, 0.5, 9)[0]
    index = torch.arange(flat.numel() - 5000, flat.numel(), device="cuda")
    assert torch.equal(out[-5000:] != 0, ref.words(index, 9, 0) >= 2**31)
    del x, flat, out
    torch.cuda.empty_cache()


def test_counters_past_32_bits():
    """More than 2^34 elements, whose groups of four take the counter's second word."""
    n = 2**34 + 1000
    x = torch.empty(n, device="cuda", dtype=BF16)
    x[2**34 - 1000:] = 1
    out, _ = kernels.dropout_train(x, 0.5, 33)
    index = torch.arange(2**34 - 1000, n, device="cuda")
    assert torch.equal(out[2**34 - 1000:] != 0, ref.words(index, 33, 0) >= 2**31)
    del x, out
    torch.cuda.empty_cache()
