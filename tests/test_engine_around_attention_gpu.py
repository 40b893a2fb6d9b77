"""Dropout of the engine ops' updates and the norm of queries and keys on the b200 backend, with their gradients, and
a run of the operators around an attention together (B200 only)."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

import attention_reference as ref  # noqa: E402
from foldforge_b200 import _lib, kernels  # noqa: E402
from foldforge_b200.engine import backends, policy, training  # noqa: E402
from foldforge_b200.engine.modules import BackendUnsupported, PairformerBlock, PairformerConfig, QKNorm, TriangleAttention  # noqa: E402
from training_reference import half_step, worst  # noqa: E402

BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    torch.cuda.synchronize()
    assert _lib.device_error() == 0


def gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def qk_norm(d, pairs, kind, interleaved=False):
    module = QKNorm(d, frequencies=[10.0 ** (-i / pairs) for i in range(pairs)], axes=[i % 2 for i in range(pairs)],
                    interleaved=interleaved).cuda()
    module.q_weight.data = 1 + 0.2 * torch.randn(d, device="cuda", generator=gen(1))
    module.k_weight.data = 1 + 0.2 * torch.randn(d, device="cuda", generator=gen(2))
    module.set_backend("b200")
    module.set_checkpoint(kind)
    return module


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("d,pairs", [(48, 24), (64, 20), (33, 7)])
def test_qk_norm_gradients(d, pairs, dtype):
    module = qk_norm(d, pairs, "exact")
    g = gen(3)
    rows = torch.randn(2, 40, 7, d, device="cuda", generator=g).to(dtype).requires_grad_()
    positions = torch.randint(0, 5000, (40, 2), device="cuda", generator=g)
    q, k = module(rows[:, :, :4], rows[:, :, 4:6], positions)
    dq, dk = (torch.randn(t.shape, device="cuda", generator=g).to(dtype) for t in (q, k))
    torch.autograd.backward([q, k], [dq, dk])
    angle = ref.angles(positions, module.frequencies, module.axes)
    for i, (part, out, dy, w) in enumerate(((slice(0, 4), q, dq, module.q_weight), (slice(4, 6), k, dk, module.k_weight))):
        (y, dx, dw), (ey, edx, edw) = ref.heads(rows.detach()[:, :, part], angle, False, w.detach(), 1e-6, dy)
        assert worst(out.detach(), y, ey, dtype) <= 1, i
        assert worst(rows.grad[:, :, part], dx, edx, dtype) <= 1, i
        assert worst(w.grad, dw, edw, F32) <= 1, i
    assert not rows.grad[:, :, 6:].any()
    with torch.no_grad():
        again = module(rows[:, :, :4], rows[:, :, 4:6], positions)
    assert torch.equal(again[0], q) and torch.equal(again[1], k)


def test_qk_norm_kept_in_8_bits():
    """The same numbers as the gradient at what the checkpoint stands for."""
    from training_reference import rounded_to_8_bits

    module = qk_norm(64, 32, "mxfp8")
    g = gen(4)
    q = torch.randn(1, 50, 4, 64, device="cuda", generator=g).bfloat16().requires_grad_()
    k = torch.randn(1, 50, 2, 64, device="cuda", generator=g).bfloat16()
    positions = torch.randint(0, 99, (1, 50, 2), device="cuda", generator=g)
    y, _ = module(q, k, positions)
    dy = torch.randn(y.shape, device="cuda", generator=g).bfloat16()
    y.backward(dy)
    kept = rounded_to_8_bits(q.detach().reshape(-1, 64)).reshape(q.shape).to(BF16)
    angle = ref.angles(positions, module.frequencies, module.axes)
    (_, dx, dw), (_, edx, edw) = ref.heads(kept, angle, False, module.q_weight.detach(), 1e-6, dy)
    assert worst(q.grad, dx, edx, BF16) <= 1 and worst(module.q_weight.grad, dw, edw, F32) <= 1
    assert not module.k_weight.grad.any()


def test_qk_norm_gradients_that_are_asked_for_and_refusals():
    module = qk_norm(32, 16, "exact")
    q = torch.randn(5, 2, 32, device="cuda")
    positions = torch.zeros(5, 2, dtype=torch.int64, device="cuda")
    module.q_weight.requires_grad_(False)
    module.k_weight.requires_grad_(False)
    x = q.clone().requires_grad_()
    y, z = module(x, q, positions)
    (y.sum() + z.sum()).backward()
    assert x.grad is not None and module.q_weight.grad is None
    module.set_checkpoint(None)
    with pytest.raises(BackendUnsupported, match="autograd"):
        module(x, q, positions)
    assert module(q, q, positions)[0].shape == q.shape
    for bad in ((q.half(), q.half(), positions), (q, q.bfloat16(), positions), (q[None, None], q[None, None], positions),
                (q, q, positions.double())):
        assert module.unsupported(*bad) is not None
    policy.guard(module)
    module(q.half(), q.half(), positions)  # the pytorch backend serves it


def test_a_step_with_dropout_draws_one_mask_on_both_machines():
    op = TriangleAttention(16, 2, d_hidden=8, starting=False, p_drop=0.25)
    g = torch.Generator().manual_seed(6)
    for p in op.parameters():
        p.data = torch.randn(p.shape, generator=g) * 0.3
    op.set_dropout()
    x = torch.randn(1, 9, 9, 16, generator=g)
    torch.manual_seed(5)
    host = op(x) != x
    on_gpu = op.cuda()
    torch.manual_seed(5)
    assert torch.equal((on_gpu(x.cuda()) != x.cuda()).cpu(), host)
    assert torch.equal(host.any(2), host.all(2))  # columns share it


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_dropout_add(dtype):
    g = gen(7)
    residual = torch.randn(2, 11, 11, 24, device="cuda", generator=g).to(dtype).requires_grad_()
    update = torch.randn(2, 11, 11, 24, device="cuda", generator=g).requires_grad_()
    torch.manual_seed(9)
    out = training.dropout_add(residual, update, 0.25, -2)
    torch.manual_seed(9)
    keep = ref.kept(update.shape, 0.25, int(torch.empty((), dtype=torch.int64).random_()), 0, (2,))
    want, bound = ref.dropout(update.detach(), keep, 0.25, residual.detach())
    assert out.dtype == dtype and worst(out.detach(), want, bound, dtype) <= 1
    dout = torch.randn(out.shape, device="cuda", generator=g).to(dtype)
    out.backward(dout)
    assert torch.equal(residual.grad, dout) and update.grad.dtype == F32
    want, bound = ref.dropout(dout, keep, 0.25)
    assert worst(update.grad, want, bound, F32) <= 1 and not update.grad[~keep].any()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="host"), torch.cuda.graph(graph):
        dout.add(1)
        training.dropout_add(residual.detach(), update.detach(), 0.25, -2)


def test_a_block_trains_with_dropout():
    """Under the fallback policy the dropping ops run the pytorch backend, the norms and transitions b200."""
    block = PairformerBlock(PairformerConfig(d_pair=128, d_single=0, p_drop=0.25)).cuda()
    g = torch.Generator().manual_seed(8)
    for p in block.parameters():
        p.data = (torch.randn(p.shape, generator=g) * 0.1).cuda()
    policy.apply_plan(torch.nn.ModuleList([block]), backends.BackendPlan.make("b200").resolve(torch.device("cuda")), torch.device("cuda"))
    training.set_checkpoint(block, "exact")
    training.set_dropout(block)
    x = torch.randn(1, 20, 20, 128, generator=g).bfloat16().cuda().requires_grad_()
    torch.manual_seed(1)
    out = block(x)
    out.float().square().mean().backward()
    first = [x.grad.clone()] + [p.grad.clone() for p in block.parameters()]
    assert all(bool(torch.isfinite(t).all()) and bool(t.any()) for t in first)
    x.grad = None
    block.zero_grad()
    torch.manual_seed(1)
    assert torch.equal(block(x), out)
    torch.manual_seed(2)
    assert not torch.equal(block(x), out)
    block.eval()
    with torch.no_grad():
        assert torch.equal(block(x), block(x))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_around_an_attention_together(dtype):
    """A training step as it would run: rows [q | k | v], norm and rotation of q and k, attention, dropout of its
    output into the residual; forward and backward against the same step in 64 bits. One captured step replays to
    the same numbers."""
    g = gen(10)
    b, t, h, hk, d = 2, 33, 4, 2, 32
    x = torch.randn(b, t, h * d, device="cuda", generator=g).to(dtype)
    rows = torch.randn(b, t, h + 2 * hk, d, device="cuda", generator=g).to(dtype)
    qw, kw = (1 + 0.2 * torch.randn(d, device="cuda", generator=g) for _ in range(2))
    positions = torch.stack([torch.arange(t, device="cuda"), torch.randint(0, 5, (t,), device="cuda", generator=g)], -1)
    frequencies, axes = kernels.rotary_frequencies(16) + kernels.rotary_frequencies(16), [0] * 8 + [1] * 8
    table = kernels.rotary_table(frequencies, axes)
    seed = torch.tensor([1234, 5], device="cuda")
    dout = torch.randn(x.shape, device="cuda", generator=g).to(dtype)

    def attend(q, k, v):  # [b, t, heads, d]
        k, v = (s.repeat_interleave(h // hk, 2) for s in (k, v))
        w = (torch.einsum("bqhd,bkhd->bhqk", q, k) * d**-0.5).softmax(-1)
        return torch.einsum("bhqk,bkhd->bqhd", w, v).reshape(b, t, h * d)

    def step():
        q, k, v = rows[:, :, :h], rows[:, :, h:h + hk], rows[:, :, h + hk:]
        qn, kn = kernels.qk_norm_rotary(q, k, positions, table, qw, kw)
        leaves = [s.float().requires_grad_() for s in (qn, kn, v)]
        with torch.enable_grad():
            o = attend(*leaves)
        out, saved = kernels.dropout_train(o.detach().to(dtype), 0.25, seed, residual=x)
        do = kernels.dropout_backward(dout, saved)
        dqn, dkn, dv = torch.autograd.grad(o, leaves, do.float())
        drows = torch.empty_like(rows)
        gradients = kernels.qk_norm_rotary_backward(dqn.to(dtype), dkn.to(dtype), q, k, positions, table, qw, kw,
                                                    out=(drows[:, :, :h], drows[:, :, h:h + hk]))
        drows[:, :, h + hk:] = dv.to(dtype)
        return out, drows, gradients[2], gradients[3]

    got = step()
    r64, qw64, kw64 = rows.double().requires_grad_(), qw.double().requires_grad_(), kw.double().requires_grad_()
    angle = ref.angles(positions, frequencies, axes)

    def normal(s, w):
        return ref.rotate(s * (s.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w, angle, False)

    o64 = attend(normal(r64[:, :, :h], qw64), normal(r64[:, :, h:h + hk], kw64), r64[:, :, h + hk:])
    keep = ref.kept(x.shape, 0.25, 1234, 5)
    out64 = x.double() + torch.where(keep, o64 / 0.75, 0.0)
    out64.backward(dout.double())
    # roundings to the type between the steps: q, k, the attention's output, the sum, and on the way back dropout's
    # gradient, those of q and k, and the result; each enters a later value by at most the logits' slope (logits of
    # normed heads are at most d^0.5 1.7^2 = 16 in size): fewer than 64 half steps of the largest value's norm
    tol = 64 * half_step(dtype) + 1e-4 * (dtype == F32)
    for a, w in zip(got, (out64, r64.grad, qw64.grad, kw64.grad), strict=True):
        assert float((a.double() - w.detach()).norm() / w.detach().norm()) < tol
    # captured without autograd's part: the kernels around the attention alone
    graph = torch.cuda.CUDAGraph()
    q, k = rows[:, :, :h], rows[:, :, h:h + hk]
    with torch.cuda.graph(graph):
        qn, kn = kernels.qk_norm_rotary(q, k, positions, table, qw, kw)
        out, saved = kernels.dropout_train(qn.reshape(b, t, h * d), 0.25, seed, residual=x)
        back = kernels.qk_norm_rotary_backward(kernels.dropout_backward(dout, saved).view(b, t, h, d), kn, q, k, positions, table, qw, kw)
    for _ in range(2):
        graph.replay()
    eager_q, eager_k = kernels.qk_norm_rotary(q, k, positions, table, qw, kw)
    eager, saved = kernels.dropout_train(eager_q.reshape(b, t, h * d), 0.25, seed, residual=x)
    want = kernels.qk_norm_rotary_backward(kernels.dropout_backward(dout, saved).view(b, t, h, d), eager_k, q, k, positions, table, qw, kw)
    assert torch.equal(out, eager) and all(torch.equal(a, c) for a, c in zip(back, want, strict=True))
