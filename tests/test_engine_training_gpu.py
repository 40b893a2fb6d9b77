"""Gradients of the engine ops on the b200 backend against automatic differentiation in 64 bits (B200 only)."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

import training_reference as ref  # noqa: E402
from foldforge_b200 import _lib, kernels  # noqa: E402
from foldforge_b200.engine import backends, factories, policy, training  # noqa: E402
from foldforge_b200.engine.modules import BackendUnsupported, Transition  # noqa: E402
from foldforge_b200.engine.pairformer import pairformer_block  # noqa: E402
from foldforge_b200.engine.serving import report_observations  # noqa: E402

BF16 = torch.bfloat16
#: A hidden activation is rounded to bf16 as v, as a and b (from rounded weights) and as the gated product,
#: its gradient as dh and [da | db], and both meet rounded weights once more: fewer than 8 roundings of at
#: most 2^-8 on the way to any gradient, relative to the gradient's norm.
TOL = 8 * 2.0**-8


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    torch.cuda.synchronize()
    assert _lib.device_error() == 0


def rel(a, b):
    return ((a.double() - b.double()).norm() / b.double().norm().clamp_min(1e-30)).item()


def randomised(module, seed):
    g = torch.Generator().manual_seed(seed)
    for name, p in module.named_parameters():
        scale = p.shape[-1] ** -0.5 if p.dim() == 2 else 0.3
        p.data = torch.randn(p.shape, generator=g) * scale + (1.0 if name.endswith("weight") and p.dim() == 1 else 0.0)
    return module.cuda()


def exact_transition(x, weights, eps, mask):
    """The transition in 64 bits on leaves made from ``x`` and the weights: (output, leaves)."""
    leaves = [x.detach().double().requires_grad_()] + [w.detach().double().requires_grad_() for w in weights]
    z, lw, lb, wa, wb, ws = leaves
    v = torch.nn.functional.layer_norm(z, (z.shape[-1],), lw, lb, eps)
    delta = (torch.nn.functional.silu(v @ wa.t()) * (v @ wb.t())) @ ws.t()
    return z + (delta if mask is None else torch.where(mask[..., None], delta, 0.0)), leaves


@pytest.mark.parametrize("kind", ["exact", "mxfp8"])
@pytest.mark.parametrize("d,n,shape,masked", [(128, 4, (2, 24, 24), True), (128, 4, (1, 1, 1), False),
                                              (128, 4, (1, 70, 70), True), (384, 4, (2, 77), True),
                                              (384, 4, (1, 1), False), (64, 4, (3, 50, 20), False),
                                              (128, 4, (5, 33), False), (40, 2, (7, 19), False)])
def test_transition(d, n, shape, masked, kind):
    module = randomised(Transition(d, n), 1)
    module.set_backend("b200")
    module.set_checkpoint(kind)
    g = torch.Generator().manual_seed(2)
    x = torch.randn(*shape, d, generator=g).to(BF16).cuda()
    dy = (torch.randn(*shape, d, generator=g) * 0.01).to(BF16).cuda()
    key_mask = full = None
    if masked:
        key_mask = torch.rand(shape[:2], generator=g) > 0.3
        key_mask[0, -1] = False
        key_mask = key_mask.cuda()
        full = key_mask[:, :, None] & key_mask[:, None, :] if len(shape) == 3 else key_mask
    xa = x.clone().requires_grad_()
    out = module(xa, key_mask)
    with torch.no_grad():
        assert torch.equal(out, module(x, key_mask))  # the forward pass is the inference one
    out.backward(dy)
    base = ref.rounded_to_8_bits(x.view(-1, d)).view(x.shape) if kind == "mxfp8" else x
    weights = [module.ln_in.weight, module.ln_in.bias, module.expand_a.weight, module.expand_b.weight, module.squeeze.weight]
    want_out, leaves = exact_transition(base, weights, module.ln_in.eps, full)
    want = torch.autograd.grad(want_out, leaves, dy.double())
    assert rel(xa.grad.double() - dy, want[0] - dy.double()) < TOL + 2.0**-8 * (dy.norm() / (want[0] - dy.double()).norm()).item()
    for p, w in zip(weights, want[1:]):
        assert p.grad.dtype == torch.float32 and rel(p.grad, w) < TOL
    if full is not None:
        assert torch.equal(xa.grad[~full], dy[~full])


@pytest.mark.parametrize("kind", ["exact", "mxfp8"])
@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_layer_norm(dtype, kind):
    norm = randomised(factories.layer_norm(128), 3)
    norm.set_backend("b200")
    norm.set_checkpoint(kind)
    g = torch.Generator().manual_seed(4)
    x = torch.randn(3, 20, 20, 128, generator=g).to(dtype).cuda()
    dy = torch.randn(3, 20, 20, 128, generator=g).to(dtype).cuda()
    xa = x.clone().requires_grad_()
    y = norm(xa)
    y.backward(dy)
    (ry, rdx, rdw, rdb), (ey, edx, edw, edb) = ref.layer_norm(x.view(-1, 128), dy.view(-1, 128), norm.weight.detach(),
                                                             norm.bias.detach(), norm.eps, kind == "mxfp8")
    assert ref.worst(y.detach().view(-1, 128), ry, ey, dtype) <= 1
    assert ref.worst(xa.grad.view(-1, 128), rdx, edx, dtype) <= 1
    assert ref.worst(norm.weight.grad, rdw, edw, torch.float32) <= 1
    assert ref.worst(norm.bias.grad, rdb, edb, torch.float32) <= 1
    # an expanded gradient, as a sum's is
    xa.grad = None
    norm(xa).sum().backward()
    (_, rdx, *_), (_, edx, *_) = ref.layer_norm(x.view(-1, 128), torch.ones(1200, 128, device="cuda"), norm.weight.detach(),
                                                norm.bias.detach(), norm.eps, kind == "mxfp8")
    assert ref.worst(xa.grad.view(-1, 128), rdx, edx, dtype) <= 1


def test_a_block_trains_where_it_can():
    """A Pairformer block under the fallback policy: ops without a gradient run pytorch, the transitions
    b200, and the gradients agree with the all-pytorch block's."""
    def run(backend, kind):
        block = randomised(pairformer_block(d_pair=128, triangle_model="af3", d_single=384), 5)
        plan = backends.BackendPlan.make(backend, unsupported="fallback").resolve(torch.device("cuda:0"))
        holder = torch.nn.ModuleList([block])
        policy.apply_plan(holder, plan, torch.device("cuda:0"))
        training.set_checkpoint(block, kind)
        g = torch.Generator().manual_seed(6)
        z = torch.randn(1, 20, 20, 128, generator=g).to(BF16).cuda().requires_grad_()
        s = torch.randn(1, 20, 384, generator=g).to(BF16).cuda().requires_grad_()
        mask = torch.ones(1, 20, dtype=torch.bool, device="cuda")
        mask[:, 17:] = False
        pair, single = block(z, mask, s)
        dp = torch.randn(pair.shape, generator=g).cuda().to(BF16)
        ds = torch.randn(single.shape, generator=g).cuda().to(BF16)
        torch.autograd.backward([pair, single], [dp, ds])
        grads = {n: p.grad for n, p in block.named_parameters() if p.grad is not None}
        return grads, z.grad, s.grad, report_observations(holder)["modules"]

    want, wz, ws, _ = run("pytorch", None)
    got, gz, gs, seen = run("b200", "exact")
    served = {k.split(".")[-1]: v["served_host_calls"] for k, v in seen.items()}
    assert served["transition_pair"] == {"b200": 1} and served["single_transition"] == {"b200": 1}
    assert served["tri_multi_outgoing"] == {"pytorch": 1}
    assert set(got) == set(want)
    for name in want:
        # both runs round: the op's own roundings, and once more for the ops after it that see rounded inputs
        assert rel(got[name], want[name]) < 2 * TOL, name
    assert rel(gz, wz) < 2 * TOL and rel(gs, ws) < 2 * TOL


@pytest.mark.parametrize("d,n,shape", [(128, 4, (1, 9, 9)), (384, 4, (1, 9)), (64, 4, (3, 5))])
def test_a_training_step_sees_weights_changed_through_data(d, n, shape):
    """``p.data`` leaves a parameter's address and version as they were; an optimiser's step changes the
    version. Both reach the next forward pass, and the next one without gradients."""
    def fresh(state):
        m = Transition(d, n).cuda()
        m.load_state_dict(state)
        m.set_backend("b200")
        m.set_checkpoint("exact")
        return m

    op = fresh(randomised(Transition(d, n), 3).state_dict())
    x = torch.randn(*shape, d, generator=torch.Generator().manual_seed(4)).to(BF16).cuda()
    first = op(x)
    op.squeeze.weight.data.mul_(-2.0)
    second = op(x)
    assert not torch.equal(first, second)
    assert torch.equal(second, fresh(op.state_dict())(x))
    with torch.no_grad():
        assert torch.equal(op(x), second)
    second.float().sum().backward()
    torch.optim.SGD(op.parameters(), lr=0.1).step()
    assert torch.equal(op(x), fresh(op.state_dict())(x))


def test_a_captured_training_step_calls_the_kernels():
    """Autograd under capture is refused; the same step from the kernels' functions is captured, replayed
    on new inputs, and agrees with autograd's."""
    module = randomised(factories.layer_norm(128), 7)
    module.set_backend("b200")
    module.set_checkpoint("mxfp8")
    g = torch.Generator(device="cuda").manual_seed(8)
    x = torch.randn(500, 128, device="cuda", generator=g).to(BF16)
    dy = torch.randn(500, 128, device="cuda", generator=g).to(BF16)

    def step():
        y, saved = kernels.layer_norm_train(x, module.weight, module.bias, module.eps, checkpoint=True)
        return [y, *kernels.layer_norm_backward(dy, saved, module.weight)]

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    refused = []
    with torch.cuda.graph(graph):
        try:
            module(x.detach().requires_grad_())
        except BackendUnsupported as exc:
            refused.append(str(exc))
        out = step()
    assert refused and "not captured" in refused[0]
    x.copy_(torch.randn(500, 128, device="cuda", generator=g))
    graph.replay()
    xa = x.clone().requires_grad_()
    y = module(xa)
    y.backward(dy)
    for a, b in zip(out, (y, xa.grad, module.weight.grad, module.bias.grad)):
        assert torch.equal(a, b)
