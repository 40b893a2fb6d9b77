"""Outputs of the caller of the norm and rotation of queries and keys (B200 only)."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

from foldforge_b200 import _lib, kernels  # noqa: E402
from foldforge_b200.engine.modules import QKNorm  # noqa: E402

BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    torch.cuda.synchronize()
    assert _lib.device_error() == 0


def gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def turning(b, t, d):
    table = kernels.rotary_table(kernels.rotary_frequencies(d))
    return 3 * torch.arange(t, device="cuda")[:, None].expand(b, t, 1), table


# --------------------------------------------------------------------------- autograd sees what is written
@pytest.mark.parametrize("write", ["rotary", "qk_norm_rotary", "qk_norm_rotary_backward"])
def test_a_call_over_what_a_backward_pass_reads_is_seen(write):
    """q and k that a norm keeps for its backward pass, written in place meanwhile: the backward pass refuses to run."""
    module = QKNorm(48, frequencies=kernels.rotary_frequencies(48)).cuda()
    module.set_backend("b200")
    module.set_checkpoint("exact")
    rows = torch.randn(2, 30, 6, 48, device="cuda", generator=gen(1)).bfloat16()
    positions, table = turning(2, 30, 48)
    q, k = rows[:, :, :4], rows[:, :, 4:]
    y, z = module(q, k, positions)
    again = rows[:, :, :4], rows[:, :, 4:]  # other views of the same memory
    if write == "rotary":
        kernels.rotary(q, k, positions, table, out=again)
    elif write == "qk_norm_rotary":
        kernels.qk_norm_rotary(q, None, positions, table, None, None, out=(again[0], None))
    else:
        kernels.qk_norm_rotary_backward(y.detach(), z.detach(), q, k, positions, table, None, None, out=again)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        (y.float().sum() + z.float().sum()).backward()


def test_versions_of_outputs():
    """A call counts each of the caller's outputs once as written, its inputs not at all; new outputs start afresh.
    Inference tensors, which count nothing, are taken as well."""
    g = gen(2)
    positions, table = turning(2, 30, 48)
    q, k = torch.randn(2, 30, 4, 48, device="cuda", generator=g), torch.randn(2, 30, 2, 48, device="cuda", generator=g)
    out = torch.empty_like(q), torch.empty_like(k)
    before = [t._version for t in (q, k, *out)]
    got = kernels.rotary(q, k, positions, table, out=out)
    assert [t._version for t in (q, k, *out)] == [before[0], before[1], before[2] + 1, before[3] + 1]
    assert got[0]._version == out[0]._version and kernels.rotary(q, k, positions, table)[0]._version == 0
    want = out[0].clone()
    leaf = torch.empty_like(q, requires_grad=True)
    with torch.no_grad():
        kernels.rotary(q, None, positions, table, out=(leaf, None))
    assert leaf._version == 1 and torch.equal(leaf, want)
    with torch.inference_mode():
        other = torch.empty_like(q)
        kernels.rotary(q, None, positions, table, out=(other, None))
        assert torch.equal(other, want)


# --------------------------------------------------------------------------- outputs that lie between others
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("d", [48, 37])
@pytest.mark.parametrize("order", [(0, 2, 1, 3), (1, 2, 0, 3), (2, 0, 1, 3), (2, 1, 0, 3), (0, 1, 2, 3)])
def test_parts_of_one_tensor(order, d, dtype):
    """q and k as parts of one tensor of a batch, its axes in any order in memory (head-major among them), and as
    channels side by side in the same heads: in place and into another such tensor, the rest left as it was."""
    b, t = 3, 21
    positions, table = turning(b, t, 24)
    g = gen(d)

    def made(heads, channels):
        sizes = (b, t, heads, channels)
        memory = torch.randn([sizes[a] for a in order], device="cuda", generator=g).to(dtype)
        return memory.permute([order.index(a) for a in range(4)])

    for x, at in ((made(9, d), lambda x: (x[:, :, :4], x[:, :, 4:6], x[:, :, 6:])),
                  (made(3, 3 * d), lambda x: (x[..., 2 * d:], x[..., :d], x[..., d:2 * d]))):
        q, k, rest = at(x)
        w = 1 + 0.2 * torch.randn(d, device="cuda", generator=g)
        kept = rest.clone()
        want = kernels.qk_norm_rotary(q.contiguous(), k.contiguous(), positions, table, w, w)
        target = torch.empty_like(x).copy_(x)
        assert target.stride() == x.stride()
        kernels.qk_norm_rotary(q, k, positions, table, w, w, out=at(target)[:2])
        dq, dk = kernels.qk_norm_rotary_backward(*want, q, k, positions, table, w, w)[:2]
        gradients = torch.empty_like(x).copy_(x)
        kernels.qk_norm_rotary_backward(*want, q, k, positions, table, w, w, out=at(gradients)[:2])
        kernels.qk_norm_rotary(q, k, positions, table, w, w, out=(q, k))
        for got, parts in ((at(x), want), (at(target), want), (at(gradients), (dq, dk))):
            assert torch.equal(got[0], parts[0]) and torch.equal(got[1], parts[1]) and torch.equal(got[2], kept)
