"""Gradients of the engine ops without a GPU: the ``checkpoint`` setting, what is refused, and the
backward pass's formulas with the kernels' plain forms in their place."""

from __future__ import annotations

import pytest
import torch

import training_reference as ref
from foldforge_b200 import kernels
from foldforge_b200.engine import factories, modules, training
from foldforge_b200.engine.modules import BackendUnsupported, LayerNorm, Transition
from foldforge_b200.engine.pairformer import pairformer_block

DOUBLE = torch.float64


def test_set_checkpoint_reaches_the_ops_that_have_gradients():
    block = pairformer_block(d_pair=128, triangle_model="af3", d_single=384, precision="fp32")
    names = training.set_checkpoint(block, "mxfp8")
    assert "transition_pair" in names and "transition_pair.ln_in" in names and "tri_multi_outgoing" not in names
    assert block.transition_pair.checkpoint == "mxfp8" and block.single_transition.ln_in.checkpoint == "mxfp8"
    training.set_checkpoint(block, None)
    assert block.transition_pair.checkpoint is None
    with pytest.raises(ValueError, match="checkpoint must be"):
        training.set_checkpoint(block, "int4")
    with pytest.raises(ValueError, match="checkpoint must be"):
        LayerNorm(8).set_checkpoint("fp8")


@pytest.fixture
def on_device(monkeypatch):
    """CPU tensors pass for ones on an sm_100 device."""
    monkeypatch.setattr(modules, "_device_reason", lambda *ts: None)
    monkeypatch.setattr(modules, "_library_reason", lambda: None)


def test_a_gradient_is_refused_without_a_checkpoint(on_device):
    """What was refused before stays refused: only ``checkpoint`` opens it."""
    for module, x in ((factories.layer_norm(64), torch.randn(4, 64)),
                      (factories.transition(64, 4), torch.randn(1, 4, 64, dtype=torch.bfloat16))):
        module.set_backend("b200")
        assert module.unsupported(x) is None
        x = x.requires_grad_()
        assert "inference only" in module.unsupported(x)
        with pytest.raises(BackendUnsupported, match="inference only"):
            module(x)
        module.set_checkpoint("exact")
        assert module.unsupported(x) is None
        with torch.no_grad():
            assert module.unsupported(x) is None and not module._trains(x)


def test_gradients_out_of_range_are_refused(on_device, monkeypatch):
    norm = factories.layer_norm(8200)
    norm.set_backend("b200")
    norm.set_checkpoint("mxfp8")
    assert "at most 8192" in norm.unsupported(torch.randn(2, 8200).requires_grad_())
    with torch.no_grad():
        assert norm.unsupported(torch.randn(2, 8200)) is None
    tr = Transition(64, 4)
    tr.set_backend("b200")
    tr.set_checkpoint("exact")
    assert "bf16" in tr.unsupported(torch.randn(1, 4, 64).requires_grad_())
    odd = Transition(20, 3)
    odd.set_backend("b200")
    odd.set_checkpoint("exact")
    assert "multiple of 8" in odd.unsupported(torch.randn(1, 4, 20, dtype=torch.bfloat16).requires_grad_())
    monkeypatch.setattr(training, "capture_reason", lambda: "captured")
    assert tr.unsupported(torch.randn(1, 4, 64, dtype=torch.bfloat16).requires_grad_()) == "captured"
    with torch.no_grad():
        assert tr.unsupported(torch.randn(1, 4, 64, dtype=torch.bfloat16)) is None


# --------------------------------------------------------------------------- the formulas, in 64 bits
def _rows(t):
    return t.reshape(-1, t.shape[-1])


@pytest.fixture
def plain_kernels(monkeypatch, on_device):
    """The kernels' definitions in 64 bits in place of the kernels (a checkpoint keeps the rounded values)."""

    def pack(x):
        return kernels.Checkpoint8(ref.rounded_to_8_bits(_rows(x)).reshape(x.shape), x.shape, x.dtype)

    def unpack(kept):
        return kept.data

    def values(kept):
        return unpack(kept) if isinstance(kept, kernels.Checkpoint8) else kept

    def norm(x, weight, bias, eps=1e-5, *, checkpoint=False):
        (y, *_), _ = ref.layer_norm(_rows(x), torch.zeros_like(_rows(x)), weight, bias, eps, False)
        mean = _rows(x).mean(1)
        stats = torch.stack([mean, ((_rows(x) - mean[:, None]).square().mean(1) + eps).rsqrt()])
        return y.view(x.shape), kernels.LayerNormSaved(pack(x) if checkpoint else x, stats)

    def norm_backward(dy, saved, weight, *, bias=True, residual=None):
        g = _rows(dy)
        mean, rstd = saved.stats[:, :, None]
        xh = (_rows(values(saved.x)) - mean) * rstd
        gw = g if weight is None else g * weight
        dx = rstd * (gw - gw.mean(1, keepdim=True) - xh * (gw * xh).mean(1, keepdim=True))
        dx = dx.view(dy.shape) + (0 if residual is None else residual)
        return dx, None if weight is None else (g * xh).sum(0), g.sum(0) if bias else None

    def gate_backward(dh, ab, *, output=False):
        (h, dab, _), _ = ref.swiglu(ab, dh, False)
        return (dab, h) if output else dab

    for name, f in {"checkpoint_pack": pack, "checkpoint_unpack": unpack, "layer_norm_train": norm,
                    "layer_norm_backward": norm_backward, "swiglu_backward": gate_backward,
                    "weight_grad": lambda dy, x: _rows(dy).t() @ _rows(x),
                    "gemm_nt": lambda a, b: a @ b.t()}.items():
        monkeypatch.setattr(kernels, name, f)
    monkeypatch.setattr(Transition, "unsupported", lambda self, x, mask=None: None)  # 64 bits run only here
    monkeypatch.setattr(Transition, "_run_b200", lambda self, x, mask: reference_transition(self, x, mask))


def reference_transition(module, x, mask):
    v = torch.nn.functional.layer_norm(x, (module.d,), module.ln_in.weight, module.ln_in.bias, module.ln_in.eps)
    a, b = v @ module.expand_a.weight.t(), v @ module.expand_b.weight.t()
    delta = (torch.nn.functional.silu(a) * b) @ module.squeeze.weight.t()
    if mask is not None and module.masked_update == "zero":
        m = mask[:, :, None] & mask[:, None, :] if x.dim() == 4 else mask
        delta = torch.where(m[..., None], delta, 0.0)
    return x + delta


@pytest.mark.parametrize("kind", ["exact", "mxfp8"])
@pytest.mark.parametrize("shape,masked,policy", [((2, 5, 16), False, "zero"), ((2, 5, 16), True, "zero"),
                                                 ((2, 4, 4, 16), True, "zero"), ((2, 4, 4, 16), True, "compute")])
def test_transition_gradients(plain_kernels, monkeypatch, shape, masked, policy, kind):
    """Against automatic differentiation in 64 bits; with an 8-bit checkpoint, of the input it stands for.
    Rows are worked on seven at a time, so that sums run over chunks with a last shorter one."""
    monkeypatch.setattr(training, "CHUNK_ROWS", 7)
    g = torch.Generator().manual_seed(1)
    module = Transition(16, 2).to(DOUBLE)
    module.masked_update = policy
    for m in (module.ln_in, module):  # LayerNorm keeps fp32 parameters under a cast
        for p in m.parameters(recurse=m is module):
            p.data = torch.randn(p.shape, generator=g, dtype=DOUBLE) * 0.5
    module.set_backend("b200")
    module.set_checkpoint(kind)
    x = torch.randn(shape, generator=g, dtype=DOUBLE)
    mask = None
    if masked:
        mask = torch.rand(shape[:2], generator=g) > 0.4
        mask[0] = False  # a whole example masked
    dy = torch.randn(shape, generator=g, dtype=DOUBLE)
    xa = x.clone().requires_grad_()
    out = module(xa, mask)
    params = list(module.parameters())
    got = torch.autograd.grad(out, [xa, *params], dy)
    base = ref.rounded_to_8_bits(_rows(x)).view(shape) if kind == "mxfp8" else x
    xb = base.clone().requires_grad_()
    want = torch.autograd.grad(reference_transition(module, xb, mask), [xb, *params], dy)
    torch.testing.assert_close(out, reference_transition(module, x, mask))
    for a, b in zip(got, want):
        torch.testing.assert_close(a, b.to(a.dtype))


@pytest.mark.parametrize("affine,bias", [(True, True), (True, False), (False, False)])
@pytest.mark.parametrize("kind", ["exact", "mxfp8"])
def test_layer_norm_gradients(plain_kernels, kind, affine, bias):
    g = torch.Generator().manual_seed(2)
    norm = LayerNorm(40, elementwise_affine=affine, bias=bias)
    for p in norm.parameters():
        p.data = torch.randn(p.shape, generator=g, dtype=DOUBLE)
    norm.set_backend("b200")
    norm.set_checkpoint(kind)
    x = torch.randn(3, 7, 40, generator=g, dtype=DOUBLE)
    dy = torch.randn(3, 7, 40, generator=g, dtype=DOUBLE)
    xa = x.clone().requires_grad_()
    # dtype checks are the kernels' business; 64 bits run only here
    out = training.layer_norm(xa, norm.weight, norm.bias, norm.eps, kind)
    got = torch.autograd.grad(out, [xa, *norm.parameters()], dy)
    w = None if norm.weight is None else norm.weight.detach()
    b = None if norm.bias is None else norm.bias.detach()
    (y, dx, dw, db), _ = ref.layer_norm(_rows(x), _rows(dy), w, b, norm.eps, kind == "mxfp8")
    torch.testing.assert_close(_rows(out), y)
    for a, want in zip(got, [dx.view(x.shape), *([dw] if affine else []), *([db] if bias else [])]):
        torch.testing.assert_close(a, want)


def test_masked_rows_may_hold_anything(plain_kernels):
    module = Transition(16, 2).to(DOUBLE)
    for p in module.parameters():
        p.data = p.data.double()
    module.set_backend("b200")
    module.set_checkpoint("exact")
    g = torch.Generator().manual_seed(3)
    mask = torch.tensor([[True, False, True, False]])
    x, dy = torch.randn(1, 4, 16, generator=g, dtype=DOUBLE), torch.randn(1, 4, 16, generator=g, dtype=DOUBLE)
    clean = torch.autograd.grad(module(x.requires_grad_(), mask), [x, *module.parameters()], dy)
    spoilt = x.detach().clone()
    spoilt[0, 1], spoilt[0, 3, 2] = float("nan"), float("inf")
    got = torch.autograd.grad(module(spoilt.requires_grad_(), mask), [spoilt, *module.parameters()], dy)
    for a, b in zip(got, clean):
        assert torch.equal(a, b)
    assert torch.equal(got[0][0, 1], dy[0, 1])


def test_a_backward_pass_is_not_captured(plain_kernels, monkeypatch):
    x = torch.randn(2, 16, dtype=DOUBLE, requires_grad=True)
    y = training.layer_norm(x, None, None, 1e-5, "exact")
    monkeypatch.setattr(training, "capture_reason", lambda: "captured")
    with pytest.raises(RuntimeError, match="captured"):
        y.sum().backward()


def test_an_input_changed_before_the_backward_pass_is_noticed(plain_kernels):
    x = torch.randn(2, 16, dtype=DOUBLE, requires_grad=True)
    z = x * 1.0
    y = training.layer_norm(z, None, None, 1e-5, "exact")
    z.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
