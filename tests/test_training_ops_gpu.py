"""The training operators against their definitions in 64 bits (B200 only)."""

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


def activation(g, rows, c, dtype):
    spread = torch.exp(torch.randn(c, device="cuda", generator=g))
    return (torch.randn(rows, c, device="cuda", generator=g) * spread + 0.5).to(dtype)


def gradient(g, rows, c, dtype):
    return (torch.randn(rows, c, device="cuda", generator=g) * 1e-2).to(dtype)


# --------------------------------------------------------------------------- 8-bit checkpoints
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,c", [(1, 1), (1, 32), (3, 31), (5, 33), (7, 8), (64, 64), (129, 100), (2, 2050),
                                    (1000, 128), (257, 384), (0, 16)])
def test_checkpoint_values(rows, c, dtype):
    x = activation(gen(rows * 10007 + c), rows, c, dtype)
    kept = kernels.checkpoint_pack(x)
    assert kept.codes.shape == x.shape and kept.scales.shape == (rows, -(-c // 32)) and kept.dtype == dtype
    assert torch.equal(kernels.checkpoint_unpack(kept).double(), ref.rounded_to_8_bits(x).to(dtype).double())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_checkpoint_borders(dtype):
    """Every code's value and the midpoints between neighbours, blocks whose largest value is just at and
    just above 448 times a power of two, zeros of both signs, the smallest and largest values of the type."""
    codes = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    values = torch.cat([codes, (codes[1:] + codes[:-1]) / 2])
    values = torch.cat([values, -values, torch.zeros(1), -torch.zeros(1)])
    rows = []
    info = torch.finfo(dtype)
    for scale in (1.0, 2.0**-20, 2.0**60, 2.0**-100):
        for first in range(0, values.numel(), 31):
            piece = values[first:first + 31] * scale
            rows.append(torch.cat([torch.tensor([448.0 * scale]), piece, torch.zeros(31 - piece.numel())]))
    for top in (info.max, info.smallest_normal, info.smallest_normal * info.eps, 448.0, 450.0, 446.0, 255.0, 0.0):
        rows.append(torch.cat([torch.tensor([-top]), torch.linspace(-1, 1, 31) * min(top, 1e30)]))
    x = torch.stack(rows).to(dtype).cuda()
    got = kernels.checkpoint_unpack(kernels.checkpoint_pack(x))
    want = ref.rounded_to_8_bits(x).to(dtype)
    assert torch.equal(got, want)
    assert torch.equal(torch.signbit(got), torch.signbit(x))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("c", [32, 40, 77])
def test_checkpoint_of_values_that_are_not_finite(c, dtype):
    x = activation(gen(3), 6, c, dtype)
    x[0, 3], x[1, 4], x[2, 5] = float("inf"), float("-inf"), float("nan")
    x[3] = float("nan")
    got = kernels.checkpoint_unpack(kernels.checkpoint_pack(x))
    assert torch.equal(torch.isnan(got), ~torch.isfinite(x))
    finite = torch.isfinite(x)
    assert torch.equal(got[finite].double(), ref.rounded_to_8_bits(x)[finite].to(dtype).double())


def test_checkpoint_takes_any_layout():
    g = gen(4)
    wide = activation(g, 40, 96, BF16)
    for x in (wide[:, 8:72], wide.t(), wide.view(-1)[1:1 + 33 * 37].view(33, 37), wide.view(4, 10, 96).transpose(0, 1)):
        got = kernels.checkpoint_unpack(kernels.checkpoint_pack(x))
        flat = x.reshape(-1, x.shape[-1])
        assert got.shape == x.shape
        assert torch.equal(got.reshape(flat.shape).double(), ref.rounded_to_8_bits(flat))


# --------------------------------------------------------------------------- LayerNorm
def run_layer_norm(rows, c, dtype, mx, *, affine=True, with_bias=True, residual=False, seed=0):
    g = gen(seed + rows * 31 + c)
    x, dy = activation(g, rows, c, dtype), gradient(g, rows, c, dtype)
    w = 1 + 0.3 * torch.randn(c, device="cuda", generator=g) if affine else None
    b = 0.2 * torch.randn(c, device="cuda", generator=g) if affine and with_bias else None
    res = gradient(g, rows, c, dtype) if residual else None
    y, saved = kernels.layer_norm_train(x, w, b, 1e-5, checkpoint=mx)
    assert isinstance(saved.x, kernels.Checkpoint8) == mx
    dx, dw, db = kernels.layer_norm_backward(dy, saved, w, bias=with_bias, residual=res)
    (ry, rdx, rdw, rdb), (ey, edx, edw, edb) = ref.layer_norm(x, dy, w, b, 1e-5, mx, res)
    assert y.dtype == dx.dtype == dtype
    assert ref.worst(y, ry, ey, dtype) <= 1
    assert ref.worst(dx, rdx, edx, dtype) <= 1
    assert (dw is None) == (w is None) and (db is None) == (not with_bias)
    if dw is not None:
        assert dw.dtype == F32 and ref.worst(dw, rdw, edw, F32) <= 1
    if db is not None:
        assert db.dtype == F32 and ref.worst(db, rdb, edb, F32) <= 1


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,c", [(1, 1), (1, 384), (2, 7), (3, 8), (17, 31), (16, 33), (40, 64), (130, 96),
                                    (5000, 128), (333, 129), (100, 197), (64, 256), (513, 384), (65, 385), (31, 768),
                                    (19, 1000), (21, 1024), (9, 1032), (5, 2048), (700, 2052), (33, 4096), (3, 5000),
                                    (2, 8192), (3, 8191)])
def test_layer_norm(rows, c, dtype, mx):
    run_layer_norm(rows, c, dtype, mx)


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("c", [37, 128, 1200])
def test_layer_norm_options(c, mx):
    run_layer_norm(70, c, BF16, mx, affine=False, with_bias=False)
    run_layer_norm(70, c, BF16, mx, with_bias=False)
    run_layer_norm(70, c, F32, mx, residual=True)
    run_layer_norm(70, c, BF16, mx, residual=True)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_layer_norm_widest_rows_with_residual(dtype):
    run_layer_norm(5, 8192, dtype, False, residual=True)
    run_layer_norm(300, 6160, dtype, True, residual=True)


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("c", [64, 129])
def test_layer_norm_takes_any_layout(c, mx):
    """Rows in another order of memory, a start off 16 bytes, weights of another dtype, an expanded gradient."""
    g = gen(12)
    w, b = 1 + 0.3 * torch.randn(c, device="cuda", generator=g), torch.randn(c, device="cuda", generator=g)
    x = activation(g, 30, c, BF16).view(5, 6, c).transpose(0, 1)
    dy = gradient(g, 1, 30 * c + 1, BF16).view(-1)[1:].view(6, 5, c)
    w16 = w.to(BF16)
    y, saved = kernels.layer_norm_train(x, w16, torch.cat([b, b])[c:][:c], checkpoint=mx)
    dx, dw, db = kernels.layer_norm_backward(dy, saved, w16)
    (ry, rdx, rdw, rdb), (ey, edx, edw, edb) = ref.layer_norm(x.reshape(30, c), dy.reshape(30, c), w16, b, 1e-5, mx)
    assert y.shape == x.shape and dx.shape == dy.shape
    assert ref.worst(y.reshape(30, c), ry, ey, BF16) <= 1 and ref.worst(dx.reshape(30, c), rdx, edx, BF16) <= 1
    assert ref.worst(dw, rdw, edw, F32) <= 1 and ref.worst(db, rdb, edb, F32) <= 1
    one = dy[:1, :1].expand(6, 5, c)
    dx, _, _ = kernels.layer_norm_backward(one, saved, w16)
    (_, rdx, *_), (_, edx, *_) = ref.layer_norm(x.reshape(30, c), one.reshape(30, c), w16, b, 1e-5, mx)
    assert ref.worst(dx.reshape(30, c), rdx, edx, BF16) <= 1


def test_layer_norm_row_that_does_not_vary():
    """The normalised row is 0 to the last bit, whatever its value: y is the bias, dx has no x in it."""
    w, b = torch.full((96,), 3.0, device="cuda"), torch.randn(96, device="cuda", generator=gen(13))
    x = torch.tensor([[5.0], [-1e30], [0.0], [1e-30]], device="cuda").expand(4, 96).contiguous()
    y, saved = kernels.layer_norm_train(x, w, b)
    assert torch.equal(y, b.expand(4, 96))
    dy = gradient(gen(14), 4, 96, F32)
    _, dw, _ = kernels.layer_norm_backward(dy, saved, w)
    assert torch.equal(dw, torch.zeros_like(dw))


def test_layer_norm_of_no_rows():
    w = torch.ones(16, device="cuda")
    x = torch.empty(0, 16, device="cuda")
    for mx in (False, True):
        y, saved = kernels.layer_norm_train(x, w, w, checkpoint=mx)
        dx, dw, db = kernels.layer_norm_backward(torch.empty_like(x), saved, w)
        assert y.shape == dx.shape == (0, 16)
        assert torch.equal(dw, torch.zeros_like(w)) and torch.equal(db, torch.zeros_like(w))


def test_layer_norm_gradient_against_differences():
    """dx, dweight and dbias against central differences of the operator's own forward pass in fp32. A
    difference over 2 h is off by h^2 / 6 of the third derivative and by the outputs' rounding over h; with
    h = 2^-6, |y| < 8 and 24 channels both stay below 2e-3 of the gradients' size (order 1)."""
    g = gen(9)
    c = 24
    x = torch.randn(2, c, device="cuda", generator=g)
    w, b = 1 + 0.3 * torch.randn(c, device="cuda", generator=g), torch.randn(c, device="cuda", generator=g)
    dy = torch.randn(2, c, device="cuda", generator=g)
    dx, dw, db = kernels.layer_norm_backward(dy, kernels.layer_norm_train(x, w, b)[1], w)

    def loss(*args):
        return (kernels.layer_norm_train(*args)[0].double() * dy.double()).sum().item()

    h = 2.0**-6
    for which, grad in ((0, dx), (1, dw), (2, db)):
        base = [x, w, b]
        for i in range(grad.numel()):
            t = base[which]
            step = torch.zeros(t.numel(), device="cuda")
            step[i] = h
            step = step.view_as(t)
            up, down = list(base), list(base)
            up[which], down[which] = t + step, t - step
            assert abs((loss(*up) - loss(*down)) / (2 * h) - grad.view(-1)[i].item()) < 2e-3


@pytest.mark.parametrize("mx", [False, True])
def test_layer_norm_row_that_is_not_finite_stays_in_its_row(mx):
    g = gen(11)
    x, dy = activation(g, 9, 128, BF16), gradient(g, 9, 128, BF16)
    w = torch.ones(128, device="cuda")
    clean_y, saved = kernels.layer_norm_train(x, w, w, checkpoint=mx)
    clean_dx, _, db = kernels.layer_norm_backward(dy, saved, w)
    x[4, 7] = float("inf")
    y, saved = kernels.layer_norm_train(x, w, w, checkpoint=mx)
    dx, dw, db2 = kernels.layer_norm_backward(dy, saved, w)
    others = torch.arange(9, device="cuda") != 4
    assert torch.equal(y[others], clean_y[others]) and torch.equal(dx[others], clean_dx[others])
    assert torch.isnan(y[4]).all() and torch.isnan(dx[4]).all() and torch.isnan(dw).all()
    assert torch.equal(db, db2)


# --------------------------------------------------------------------------- weight gradient
@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("rows,n,k", [(1, 1, 1), (1, 8, 16), (63, 7, 9), (64, 128, 128), (65, 129, 68), (200, 130, 200),
                                      (1000, 512, 128), (513, 136, 264), (3001, 64, 64), (128, 257, 520), (77, 300, 33),
                                      (20000, 40, 72), (129, 1536, 384), (40000, 256, 250)])
def test_weight_grad(rows, n, k, mx):
    g = gen(rows + 7 * n + k)
    dy, x = gradient(g, rows, n, BF16), activation(g, rows, k, BF16)
    dw = kernels.weight_grad(dy, kernels.checkpoint_pack(x) if mx else x)
    want, bound = ref.weight_grad(dy, x, mx)
    assert dw.shape == (n, k) and dw.dtype == F32
    assert ref.worst(dw, want, bound, F32) <= 1


def test_weight_grad_layouts_and_no_rows():
    g = gen(21)
    dy, x = gradient(g, 6 * 50, 48, BF16).view(6, 50, 48), activation(g, 300, 72, BF16).view(6, 50, 72)
    want, bound = ref.weight_grad(dy.reshape(300, 48), x.reshape(300, 72), False)
    assert ref.worst(kernels.weight_grad(dy, x), want, bound, F32) <= 1
    # rows in another order of memory, an expanded gradient, a start that is not 16-byte aligned
    dyt, xt = dy.transpose(0, 1), x.transpose(0, 1)
    assert ref.worst(kernels.weight_grad(dyt, xt), want, bound, F32) <= 1
    one = dy[:1, :1].expand(6, 50, 48)
    want1, bound1 = ref.weight_grad(one.reshape(300, 48), x.reshape(300, 72), False)
    assert ref.worst(kernels.weight_grad(one, x), want1, bound1, F32) <= 1
    flat = activation(g, 1, 300 * 72 + 1, BF16).view(-1)[1:].view(300, 72)
    want2, bound2 = ref.weight_grad(dy.reshape(300, 48), flat, False)
    assert ref.worst(kernels.weight_grad(dy.reshape(300, 48), flat), want2, bound2, F32) <= 1
    empty = kernels.weight_grad(torch.empty(0, 48, device="cuda", dtype=BF16), torch.empty(0, 8, device="cuda", dtype=BF16))
    assert torch.equal(empty, torch.zeros(48, 8, device="cuda"))


def test_weight_grad_value_that_is_not_finite_stays_in_its_column():
    g = gen(22)
    dy, x = gradient(g, 200, 130, BF16), activation(g, 200, 70, BF16)
    clean = kernels.weight_grad(dy, x)
    x[37, 5] = float("nan")
    for kept in (x, kernels.checkpoint_pack(x)):
        dw = kernels.weight_grad(dy, kept)
        assert torch.isnan(dw[:, 5]).all()
        assert not torch.isnan(dw[:, torch.arange(70, device="cuda") != 5]).any()
    others = torch.arange(70, device="cuda") != 5
    assert torch.equal(kernels.weight_grad(dy, x)[:, others], clean[:, others])


# --------------------------------------------------------------------------- gated unit
@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,h", [(1, 1), (1, 32), (3, 7), (5, 8), (16, 31), (33, 40), (64, 256), (129, 100),
                                    (1000, 512), (7, 1536), (0, 8)])
def test_swiglu(rows, h, dtype, mx):
    g = gen(rows * 13 + h)
    ab, dh = activation(g, rows, 2 * h, dtype), gradient(g, rows, h, dtype)
    out, saved = kernels.swiglu_train(ab, checkpoint=mx)
    dab, again = kernels.swiglu_backward(dh, saved, output=True)
    (rh, rdab, rkept), (eh, edab, ekept) = ref.swiglu(ab, dh, mx)
    assert out.dtype == dab.dtype == dtype and out.shape == (rows, h) and dab.shape == (rows, 2 * h)
    assert ref.worst(out, rh, eh, dtype) <= 1
    assert ref.worst(dab, rdab, edab, dtype) <= 1
    assert ref.worst(again, rkept, ekept, dtype) <= 1
    assert torch.equal(kernels.swiglu_backward(dh, saved), dab)
    if mx:
        assert torch.equal(kernels.checkpoint_unpack(saved).double(), ref.rounded_to_8_bits(ab).to(dtype).double())


@pytest.mark.parametrize("h", [32, 40])
@pytest.mark.parametrize("mx", [False, True])
def test_swiglu_takes_any_layout(h, mx):
    g = gen(15)
    ab = activation(g, 1, 21 * 2 * h + 1, BF16).view(-1)[1:].view(7, 3, 2 * h)
    dh = gradient(g, 21, h, BF16).view(3, 7, h).transpose(0, 1)
    out, saved = kernels.swiglu_train(ab, checkpoint=mx)
    dab = kernels.swiglu_backward(dh, saved)
    (rh, rdab, _), (eh, edab, _) = ref.swiglu(ab.reshape(21, 2 * h), dh.reshape(21, h), mx)
    assert ref.worst(out.reshape(21, h), rh, eh, BF16) <= 1
    assert ref.worst(dab.reshape(21, 2 * h), rdab, edab, BF16) <= 1


def test_swiglu_far_from_zero():
    """Gates whose exponential overflows: silu(a) is a or -0, its derivative 1 or 0."""
    a = torch.tensor([1e4, -1e4, 3e38, -3e38, 90.0, -90.0, 0.0, -0.0], device="cuda")
    b = torch.full_like(a, 2.0)
    ab = torch.cat([a, b])[None]
    dh = torch.full((1, 8), 0.5, device="cuda")
    h, saved = kernels.swiglu_train(ab)
    dab = kernels.swiglu_backward(dh, saved)
    (rh, rdab, _), (eh, edab, _) = ref.swiglu(ab, dh, False)
    rh[rh.abs() > 3.4028235e38] = float("inf")  # 3e38 * 2 is past fp32
    assert torch.equal(torch.isinf(h), torch.isinf(rh))
    keep = ~torch.isinf(rh)
    assert ref.worst(h[keep], rh[keep], eh[keep], F32) <= 1
    assert torch.isfinite(dab).all()
    assert ref.worst(dab[:, :8], rdab[:, :8], edab[:, :8], F32) <= 1
    assert ref.worst(dab[:, 8:], rdab[:, 8:], edab[:, 8:], F32) <= 1


# --------------------------------------------------------------------------- offsets past 32 bits
def test_offsets_past_32_bits():
    """More than 2^32 elements: the last rows come out as they do in a call of their own. (Each of these
    tensors is about 9 GB; whole-tensor copies are let go before the next ones are made.)"""
    c, tail = 264, 40
    rows = (1 << 32) // c + 1000
    x = torch.zeros(rows, c, dtype=BF16, device="cuda")
    x[-tail:] = activation(gen(41), tail, c, BF16)
    w, b = torch.rand(c, device="cuda", generator=gen(42)), torch.rand(c, device="cuda", generator=gen(43))
    small_y, small = kernels.layer_norm_train(x[-tail:], w, b, checkpoint=True)
    y, saved = kernels.layer_norm_train(x, w, b, checkpoint=True)
    assert torch.equal(y[-tail:], small_y)
    assert torch.equal(saved.x.codes[-tail:].view(torch.uint8), small.x.codes.view(torch.uint8))
    assert torch.equal(saved.x.scales[-tail:], small.x.scales) and torch.equal(saved.stats[:, -tail:], small.stats)
    small_dx, small_dw, small_db = kernels.layer_norm_backward(x[-tail:], small, w)
    del y
    dx, dw, db = kernels.layer_norm_backward(x, saved, w)  # the gradient is 0 but for the last rows
    assert torch.equal(dx[-tail:], small_dx) and not dx[: rows - tail].any()
    bound = 512 * ref.STEP * (x[-tail:].double().abs().sum(0) * 40)
    assert ((dw - small_dw).abs() <= bound).all() and ((db - small_db).abs() <= bound).all()
    del dx
    whole = kernels.checkpoint_unpack(saved.x)
    assert torch.equal(whole[-tail:], kernels.checkpoint_unpack(small.x))
    del whole
    for kept, few in ((saved.x, small.x), (x, x[-tail:])):
        got = kernels.weight_grad(x, kept)
        want, allowed = ref.weight_grad(x[-tail:], x[-tail:], few is small.x)
        assert ref.worst(got, want, allowed, F32) <= 1
    del saved
    out, kept = kernels.swiglu_train(x, checkpoint=True)
    few_out, few_kept = kernels.swiglu_train(x[-tail:], checkpoint=True)
    assert torch.equal(out[-tail:], few_out)
    dab = kernels.swiglu_backward(out, kept)
    assert torch.equal(dab[-tail:], kernels.swiglu_backward(few_out, few_kept)) and not dab[: rows - tail].any()


# --------------------------------------------------------------------------- use
def test_results_do_not_depend_on_timing():
    g = gen(31)
    x, dy = activation(g, 20000, 128, BF16), gradient(g, 20000, 128, BF16)
    w = torch.ones(128, device="cuda")
    _, saved = kernels.layer_norm_train(x, w, w, checkpoint=True)
    first = (*kernels.layer_norm_backward(dy, saved, w), kernels.weight_grad(dy, saved.x))
    for _ in range(5):
        again = (*kernels.layer_norm_backward(dy, saved, w), kernels.weight_grad(dy, saved.x))
        for a, b in zip(first, again):
            assert torch.equal(a, b)


def test_captured_and_replayed_with_new_inputs():
    g = gen(32)
    x, dy = activation(g, 3000, 128, BF16), gradient(g, 3000, 128, BF16)
    ab, dh = activation(g, 500, 128, BF16), gradient(g, 500, 64, BF16)
    w, b = torch.ones(128, device="cuda"), torch.zeros(128, device="cuda")

    def step():
        y, saved = kernels.layer_norm_train(x, w, b, checkpoint=True)
        h, kept = kernels.swiglu_train(ab, checkpoint=True)
        return [y, *kernels.layer_norm_backward(dy, saved, w), kernels.weight_grad(dy, saved.x), h,
                kernels.swiglu_backward(dh, kept), kernels.checkpoint_unpack(kept)]

    step()
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    outs = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(step())
    for seed in (33, 34):
        g = gen(seed)
        for t in (x, ab):
            t.copy_(activation(g, *t.shape, BF16))
        for t in (dy, dh):
            t.copy_(gradient(g, *t.shape, BF16))
        want = step()
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        for out in outs:
            for a, c in zip(out, want):
                assert torch.equal(a, c)


def test_two_streams_at_once():
    g = gen(35)
    data = [(activation(g, 4000, 128, BF16), gradient(g, 4000, 128, BF16)) for _ in range(2)]
    w = torch.ones(128, device="cuda")

    def step(x, dy):
        y, saved = kernels.layer_norm_train(x, w, w, checkpoint=True)
        return [y, *kernels.layer_norm_backward(dy, saved, w), kernels.weight_grad(dy, saved.x)]

    want = [step(*d) for d in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None, None]
    for _ in range(4):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i] = step(*data[i])
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        for u, v in zip(a, b):
            assert torch.equal(u, v)
