"""Dropout of the engine ops' updates and the norm of queries and keys, without a GPU."""

from __future__ import annotations

import copy

import pytest
import torch

import attention_reference as ref
from foldforge_b200.engine import backends, training
from foldforge_b200.engine.modules import (MSAPairWeightedAveraging, PairformerBlock, PairformerConfig, QKNorm, TriangleAttention,
                                           TriangleMultiplication)


def randomised(module, seed=0):
    g = torch.Generator().manual_seed(seed)
    for p in module.parameters():
        p.data = torch.randn(p.shape, generator=g) * 0.3
    return module


@pytest.mark.parametrize("shape,shared", [((7, 9), ()), ((2, 5, 4, 3), (1,)), ((2, 5, 4, 3), (2,)), ((3, 4, 5), (1, 2))])
def test_masks_are_the_definition(shape, shared):
    for seed, offset in ((3, 0), (-5, 2**40)):
        got = training.dropout_keep(shape, 0.3, seed, offset, shared)
        assert torch.equal(got, ref.kept(shape, 0.3, seed, offset, shared, device="cpu"))


OPS = [
    (lambda: TriangleMultiplication(16, p_drop=0.25), -3), (lambda: TriangleMultiplication(16, outgoing=False, p_drop=0.25), -3),
    (lambda: TriangleAttention(16, 2, d_hidden=8, starting=True, p_drop=0.25), -3),
    (lambda: TriangleAttention(16, 2, d_hidden=8, starting=False, p_drop=0.25), -2),
]


@pytest.mark.parametrize("make,axis", OPS)
def test_an_update_is_dropped_in_training_mode_once_it_is_asked_for(make, axis):
    op = randomised(make())
    x = torch.randn(2, 6, 6, 16, generator=torch.Generator().manual_seed(1))
    mask = torch.ones(2, 6, dtype=torch.bool)
    mask[1, 4:] = False
    plain = op(x, mask)
    assert op.training and op.dropout == 0  # off, whatever p_drop says
    op.set_dropout()
    assert op.dropout == 0.25
    torch.manual_seed(7)
    got = op(x, mask)
    torch.manual_seed(7)
    seed = int(torch.empty((), dtype=torch.int64).random_())
    keep = ref.kept(x.shape, 0.25, seed, 0, (axis % 4,), device="cpu")
    # what is kept is the update over 1 - p: fp32 roundings of the update, the product and the sum
    want = x + torch.where(keep, (plain - x) / 0.75, 0.0)
    assert torch.allclose(got, want, rtol=0, atol=32 * 2.0**-24 * float((plain - x).detach().abs().max() + x.abs().max()))
    assert torch.equal(got[~keep], x[~keep]) and torch.equal(got[1, 4:], x[1, 4:])
    assert not torch.equal(got, op(x, mask))  # another call, another mask
    op.eval()
    assert torch.equal(op(x, mask), plain)
    op.train()
    op.set_dropout(0.0)
    assert torch.equal(op(x, mask), plain)
    for bad in (-0.1, 1.5, float("nan")):
        with pytest.raises(ValueError):
            op.set_dropout(bad)


def test_msa_rows_share_a_mask():
    op = randomised(MSAPairWeightedAveraging(8, 16, n_head=2, p_drop=0.15))
    g = torch.Generator().manual_seed(2)
    msa, pair = torch.randn(1, 5, 7, 8, generator=g), torch.randn(1, 7, 7, 16, generator=g)
    plain = op(msa, pair)
    op.set_dropout(0.5)
    changed = op(msa, pair) != msa
    dropped = ~changed.any(1)  # positions and channels whose update is gone from every row
    assert 0 < dropped.sum() < dropped.numel()
    assert torch.equal(changed.any(1), changed.all(1)) and bool((plain != msa).all())


def test_gradients_follow_the_mask_and_recomputation_repeats_it():
    from torch.utils.checkpoint import checkpoint

    op = randomised(TriangleMultiplication(16, p_drop=0.25))
    op.set_dropout()
    x = torch.randn(1, 6, 6, 16, generator=torch.Generator().manual_seed(3), requires_grad=True)
    torch.manual_seed(11)
    out = op(x)
    out.square().sum().backward()
    want = [x.grad.clone()] + [p.grad.clone() for p in op.parameters()]
    x.grad = None
    op.zero_grad()
    torch.manual_seed(11)
    again = checkpoint(op, x, use_reentrant=False)
    assert torch.equal(again, out)
    again.square().sum().backward()
    for a, b in zip([x.grad] + [p.grad for p in op.parameters()], want, strict=True):
        assert torch.equal(a, b)
    # the definition's gradient: residual plus kept update over 1 - p
    y = x.detach().clone().requires_grad_()
    plain = copy.deepcopy(op)
    plain.set_dropout(0.0)
    torch.manual_seed(11)
    seed = int(torch.empty((), dtype=torch.int64).random_())
    keep = ref.kept(x.shape, 0.25, seed, 0, (1,), device="cpu")
    loss = (y + torch.where(keep, (plain(y) - y) / 0.75, 0.0)).square().sum()
    loss.backward()
    # the same numbers but for the order of fp32 roundings; a lost or doubled mask would be off by a quarter
    assert torch.allclose(y.grad, want[0], rtol=1e-3, atol=1e-3 * float(want[0].abs().max()))


def test_set_dropout_of_a_block():
    block = PairformerBlock(PairformerConfig(d_pair=16, d_hidden_tri_multi=16, d_hidden_tri_attention=8, n_head_tri_attention=2, d_single=0,
                                             p_drop=0.25))
    names = training.set_dropout(block)
    assert names == ["tri_multi_outgoing", "tri_multi_incoming", "tri_atten_starting", "tri_atten_ending"]
    assert all(block.get_submodule(n).dropout == 0.25 for n in names)
    assert training.set_dropout(block, 0.1) == names and block.tri_atten_ending.dropout == 0.1
    block.set_backend("b200")
    x = torch.randn(1, 4, 4, 16)
    for n in names:
        assert block.get_submodule(n).unsupported(x) is not None


# --------------------------------------------------------------------------- norm of queries and keys
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_qk_norm_on_pytorch(dtype, interleaved):
    g = torch.Generator().manual_seed(5)
    f, axes = [1.0, 0.3, 0.1, 0.05, 0.01], [0, 0, 1, 1, 1]
    module = QKNorm(24, frequencies=f, axes=axes, interleaved=interleaved)
    module.q_weight.data = 1 + 0.2 * torch.randn(24, generator=g)
    q, k = (torch.randn(2, 7, h, 24, generator=g).to(dtype) for h in (4, 2))
    positions = torch.randint(0, 1000, (2, 7, 2), generator=g)
    got = module(q, k, positions)
    angle = ref.angles(positions, f, axes)
    for x, y, w in zip((q, k), got, (module.q_weight, module.k_weight), strict=True):
        (want,), (bound,) = ref.heads(x, angle, interleaved, w.detach(), 1e-6)
        assert y.dtype == dtype
        from training_reference import worst

        assert worst(y.detach(), want, bound, dtype) <= 1
    shared = module(q, k, positions[:1].expand(2, 7, 2))
    assert torch.equal(module(q, k, positions[0])[0], shared[0])


def test_qk_norm_without_positions_and_its_checks():
    module = QKNorm(8, elementwise_affine=False)
    q = torch.randn(3, 2, 8)
    y, _ = module(q, q)
    assert torch.allclose(y.square().mean(-1), torch.ones(3, 2), atol=1e-4)
    assert list(module.parameters()) == []
    with pytest.raises(ValueError):
        module(q, q, torch.zeros(3, 1))
    turning = QKNorm(8, frequencies=[1.0, 0.1])
    with pytest.raises(ValueError):
        turning(q, q)
    for bad in (dict(frequencies=[1.0] * 5), dict(frequencies=[1.0], axes=[0, 1])):
        with pytest.raises(ValueError):
            QKNorm(8, **bad)
    assert QKNorm(8).bfloat16().q_weight.dtype == torch.float32
    assert backends.op_of(turning) == "layernorm"
    turning.set_backend("b200")
    assert "CUDA" in turning.unsupported(q, q, torch.zeros(3, 1))
    again = copy.deepcopy(turning)
    assert again.frequencies == turning.frequencies and again.q_weight is not turning.q_weight
    assert training.set_checkpoint(turning, "exact") == [""] and turning.checkpoint == "exact"
