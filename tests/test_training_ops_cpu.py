"""Refusals and the plain forms of the training operators, without a GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

import training_reference as ref
from foldforge_b200 import _lib, kernels

F32, BF16 = 1, 0


def checkpoint(rows: int, c: int, dtype: torch.dtype) -> kernels.Checkpoint8:
    size = -(-rows * c // 16) * 16 + rows * -(-c // 32)
    return kernels.Checkpoint8(torch.zeros(size, dtype=torch.uint8), torch.Size((rows, c)), dtype)


def test_checkpoint_parts():
    kept = checkpoint(3, 65, torch.bfloat16)
    assert kept.codes.shape == (3, 65) and kept.codes.dtype == torch.float8_e4m3fn
    assert kept.scales.shape == (3, 3) and kept.scales.dtype == torch.uint8
    assert (kept.scales.data_ptr() - kept.codes.data_ptr()) == 208  # 195 codes, to the next 16 bytes
    assert kept.data.numel() == 208 + 9


needs_library = pytest.mark.skipif(not (_lib.LIBRARY.exists() and (_lib.LIBRARY.parent / "_binding.so").exists()),
                                   reason="library not built")


@needs_library
def test_cpu_tensors_are_refused():
    x = torch.randn(4, 64)
    w = torch.ones(64)
    saved = kernels.LayerNormSaved(x, torch.ones(2, 4))
    for call in (lambda: kernels.layer_norm_train(x, w, w), lambda: kernels.layer_norm_backward(x, saved, w),
                 lambda: kernels.checkpoint_pack(x), lambda: kernels.weight_grad(x.bfloat16(), x.bfloat16()),
                 lambda: kernels.swiglu_train(x), lambda: kernels.swiglu_backward(x, torch.randn(4, 128)),
                 lambda: kernels.checkpoint_unpack(checkpoint(4, 64, torch.float32))):
        with pytest.raises(_lib.UnsupportedCall, match="CUDA device"):
            call()


@needs_library
def test_dtypes_and_shapes_are_refused():
    """The checks of shapes and dtypes come before the one of the device, so CPU tensors meet them."""
    x, w = torch.randn(4, 64), torch.ones(64)
    saved = kernels.LayerNormSaved(x, torch.ones(2, 4))
    kept = checkpoint(4, 64, torch.float32)
    bad = [
        lambda: kernels.layer_norm_train(x.half(), w, w),
        lambda: kernels.layer_norm_train(x, w[:63], w),
        lambda: kernels.layer_norm_train(x, w, torch.ones(1, 64)),
        lambda: kernels.layer_norm_train(torch.tensor(1.0), None, None),
        lambda: kernels.layer_norm_train(torch.empty(4, 0), None, None),
        lambda: kernels.layer_norm_backward(x[:3], saved, w),
        lambda: kernels.layer_norm_backward(x.bfloat16(), saved, w),
        lambda: kernels.layer_norm_backward(x, saved._replace(stats=torch.zeros(2, 5)), w),
        lambda: kernels.layer_norm_backward(x, saved._replace(stats=torch.ones(2, 4).double()), w),
        lambda: kernels.layer_norm_backward(x, saved, w, residual=x[:, :32]),
        lambda: kernels.layer_norm_backward(x, saved._replace(x=kept._replace(data=kept.data[:-1])), w),
        lambda: kernels.layer_norm_backward(x, saved._replace(x=kept._replace(dtype=torch.bfloat16)), w),
        lambda: kernels.checkpoint_pack(x.to(torch.int32)),
        lambda: kernels.checkpoint_unpack(kept._replace(data=kept.data[:200])),
        lambda: kernels.checkpoint_unpack(kept._replace(dtype=torch.float16)),
        lambda: kernels.checkpoint_unpack(kept._replace(data=kept.data.view(torch.int8))),
        lambda: kernels.checkpoint_unpack(kept._replace(shape=torch.Size((4, 32)))),
        lambda: kernels.checkpoint_unpack(kept._replace(shape=torch.Size(()))),
        lambda: kernels.weight_grad(x.bfloat16(), checkpoint(5, 64, torch.bfloat16)),
        lambda: kernels.weight_grad(x, x),
        lambda: kernels.weight_grad(x.bfloat16(), x),
        lambda: kernels.weight_grad(x.bfloat16(), x[:3].bfloat16()),
        lambda: kernels.weight_grad(x.bfloat16(), kept),  # a checkpoint of fp32 values
        lambda: kernels.weight_grad(x.bfloat16(), torch.empty(4, 0, dtype=torch.bfloat16)),
        lambda: kernels.swiglu_train(torch.randn(4, 63)),
        lambda: kernels.swiglu_backward(x, torch.randn(4, 64)),
        lambda: kernels.swiglu_backward(x, torch.randn(4, 128).bfloat16()),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(_lib.UnsupportedCall) as refusal:
            call()
        assert "CUDA device" not in str(refusal.value), i


@needs_library
def test_sizes_past_the_entry_points_are_refused():
    """Rows wider than the entry points' 32-bit counts, from a single element (nothing is copied or made)."""
    def of(*shape, dtype=torch.bfloat16):
        return torch.zeros(1, dtype=dtype).expand(*shape)

    wide, tall, norm = 2**32 + 128, 2**31, torch.ones(128)
    byte = torch.zeros(1, dtype=torch.uint8)
    refused = [
        lambda: kernels.checkpoint_pack(of(1, wide)),
        lambda: kernels.checkpoint_unpack(kernels.Checkpoint8(byte, torch.Size((1, wide)), torch.bfloat16)),
        lambda: kernels.layer_norm_train(of(1, wide), None, None),
        lambda: kernels.layer_norm_train(of(wide), None, None, checkpoint=True),
        lambda: kernels.layer_norm_backward(of(1, wide), kernels.LayerNormSaved(of(1, wide), torch.zeros(2, 1)), norm),
        lambda: kernels.swiglu_train(of(1, wide, dtype=torch.float32)),
        lambda: kernels.swiglu_backward(of(1, wide), of(1, 2 * wide)),
        lambda: kernels.weight_grad(of(4, wide), of(4, 8)),
        lambda: kernels.weight_grad(of(4, 8), of(4, wide)),
        lambda: kernels.weight_grad(of(4, 8), of(4, 2**20 + 1)),
        lambda: kernels.weight_grad(of(4, 2**20 + 1), of(4, 8)),
        lambda: kernels.weight_grad(of(tall, 8), of(tall, 8)),
    ]
    for i, call in enumerate(refused):
        with pytest.raises(_lib.UnsupportedCall) as refusal:
            call()
        assert "channels" in str(refusal.value), i
    size = _lib.load().ffb_weight_grad_workspace_bytes
    assert size(100, 2**31 - 1, 64, 0) == size(100, 64, 2**31 - 1, 1) == size(2**62, 64, 64, 0) == 0


@needs_library
def test_entry_points_check_their_arguments():
    """Bad arguments come back as a status before anything is launched (no GPU is touched)."""
    lib = _lib.load()
    p = ctypes.c_void_p(0x10000)
    q = ctypes.c_void_p(0x20000)
    r = ctypes.c_void_p(0x30000)
    odd = ctypes.c_void_p(0x10001)
    z = None
    eps = ctypes.c_float(1e-5)
    size = ctypes.c_size_t
    train = lib.ffb_layernorm_train_fwd
    assert train(p, q, z, z, r, r, z, z, -1, 8, eps, BF16, z) == 1
    assert train(p, q, z, z, r, r, z, z, 1, 0, eps, BF16, z) == 1
    assert train(p, q, z, z, r, r, z, z, 1, 8193, eps, BF16, z) == 2
    assert train(p, q, z, z, r, r, z, z, 1, 8, eps, 7, z) == 2
    assert train(z, q, z, z, r, r, z, z, 1, 8, eps, BF16, z) == 1
    assert train(p, p, z, z, r, r, z, z, 1, 8, eps, BF16, z) == 1
    assert train(odd, q, z, z, r, r, z, z, 1, 8, eps, BF16, z) == 1
    assert train(p, q, z, z, r, r, p, z, 1, 8, eps, BF16, z) == 1  # codes without scales
    assert train(z, z, z, z, z, z, z, z, 0, 8, eps, BF16, z) == 0  # no rows: nothing to do
    bwd = lib.ffb_layernorm_bwd
    need = lib.ffb_layernorm_bwd_workspace_bytes(1000, 8, BF16)
    assert need > 0 and lib.ffb_layernorm_bwd_workspace_bytes(0, 8, BF16) == 0
    assert bwd(p, q, z, z, r, r, z, z, ctypes.c_void_p(0x40000), r, r, p, size(need - 1), 1000, 8, BF16, z) == 1
    assert bwd(p, z, z, z, r, r, z, z, q, z, z, z, size(0), 1000, 8, BF16, z) == 1  # neither x nor a checkpoint
    assert bwd(p, q, r, r, r, r, z, z, p, z, z, z, size(0), 1000, 8, BF16, z) == 1  # both
    assert bwd(p, q, z, z, r, r, z, z, p, z, z, z, size(0), 1000, 8, BF16, z) == 1  # dx is dy
    assert bwd(p, q, z, z, r, r, z, z, odd, z, z, z, size(0), 1000, 8, F32, z) == 1
    assert lib.ffb_checkpoint_pack(p, z, q, 4, 8, BF16, z) == 1
    assert lib.ffb_checkpoint_pack(p, q, r, 4, 8, 3, z) == 2
    assert lib.ffb_checkpoint_unpack(z, q, p, 4, 8, BF16, z) == 1
    assert lib.ffb_checkpoint_unpack(p, q, odd, 4, 8, F32, z) == 1
    wg = lib.ffb_weight_grad
    need = lib.ffb_weight_grad_workspace_bytes(100000, 64, 64, 0)
    assert need > 0
    assert wg(p, q, z, z, r, z, size(0), 100000, 64, 64, z) == 1
    assert wg(p, q, z, z, r, p, size(need - 1), 100000, 64, 64, z) == 1
    assert wg(p, q, z, z, r, p, size(need), 100000, 0, 64, z) == 1
    assert wg(p, q, z, z, r, p, size(need), 1 << 31, 64, 64, z) == 2
    assert wg(p, q, r, z, r, p, size(need), 100000, 64, 64, z) == 1
    assert wg(p, q, z, z, z, p, size(need), 100000, 64, 64, z) == 1
    assert wg(ctypes.c_void_p(0x10002), q, z, z, r, p, size(need), 100000, 64, 64, z) == 1
    # rows that are padded into the workspace
    padded = lib.ffb_weight_grad_workspace_bytes(100000, 65, 64, 0)
    assert padded > 100000 * 72 * 2 and lib.ffb_weight_grad_workspace_bytes(100000, 64, 72, 1) > 100000 * 72 * 2
    assert wg(p, q, z, z, r, p, size(padded - 1), 100000, 65, 64, z) == 1
    assert lib.ffb_swiglu_train_fwd(p, p, z, z, 4, 8, BF16, z) == 1
    assert lib.ffb_swiglu_train_fwd(p, q, z, r, 4, 8, BF16, z) == 1
    assert lib.ffb_swiglu_bwd(p, q, z, z, q, z, 4, 8, BF16, z) == 1
    assert lib.ffb_swiglu_bwd(p, z, z, z, q, z, 4, 8, BF16, z) == 1
    assert lib.ffb_swiglu_bwd(p, q, z, z, r, z, 4, 0, BF16, z) == 1


def test_reference_forms_are_gradients():
    """The definitions the kernels are held to, against automatic differentiation in 64 bits."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(5, 40, generator=g, dtype=torch.float64, requires_grad=True)
    w = torch.randn(40, generator=g, dtype=torch.float64, requires_grad=True)
    b = torch.randn(40, generator=g, dtype=torch.float64, requires_grad=True)
    dy = torch.randn(5, 40, generator=g, dtype=torch.float64)
    y = torch.nn.functional.layer_norm(x, (40,), w, b, 1e-5)
    want = (y, *torch.autograd.grad(y, (x, w, b), dy))
    got, _ = ref.layer_norm(x.detach(), dy, w.detach(), b.detach(), 1e-5, False)
    for u, v in zip(got, want):
        torch.testing.assert_close(u, v)
    ab = torch.randn(5, 40, generator=g, dtype=torch.float64, requires_grad=True)
    dh = torch.randn(5, 20, generator=g, dtype=torch.float64)
    h = torch.nn.functional.silu(ab[:, :20]) * ab[:, 20:]
    (dab,) = torch.autograd.grad(h, ab, dh)
    got, _ = ref.swiglu(ab.detach(), dh, False)
    torch.testing.assert_close(got[0], h)
    torch.testing.assert_close(got[1], dab)


def test_reference_checkpoint_is_the_nearest_value():
    """Within half a step of e4m3: 2^-4 of the value, or half the smallest step of the block's scale."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(50, 70, generator=g) * torch.exp(3 * torch.randn(50, 70, generator=g))
    got = ref.rounded_to_8_bits(x)
    for first in range(0, 70, 32):
        v, q = x[:, first:first + 32].double(), got[:, first:first + 32]
        top = v.abs().amax(1, keepdim=True)
        scale = torch.exp2(torch.ceil(torch.log2(top / 448)))
        assert ((v - q).abs() <= torch.maximum(2.0**-4 * v.abs(), 2.0**-10 * scale)).all()
    assert torch.equal(ref.rounded_to_8_bits(got.float()), got)  # values that fit stay as they are
