"""Outputs of the caller of the norm and rotation of queries and keys: what is refused, without a GPU."""

from __future__ import annotations

import ctypes
import random

import pytest
import torch

from foldforge_b200 import _lib, kernels

needs_library = pytest.mark.skipif(not (_lib.LIBRARY.exists() and (_lib.LIBRARY.parent / "_binding.so").exists()),
                                   reason="library not built")


# --------------------------------------------------------------------------- outputs that autograd follows
@needs_library
@pytest.mark.parametrize("leaf", [True, False])
def test_outputs_that_require_a_gradient_are_refused(leaf):
    """The calls record nothing: written in place, such a tensor would keep the gradient of what it held before."""
    table = kernels.rotary_table(kernels.rotary_frequencies(16), device="cpu")
    positions = torch.zeros(5, 1, dtype=torch.int64)
    q, k = torch.randn(5, 4, 16), torch.randn(5, 2, 16)
    followed = torch.randn(5, 4, 16, requires_grad=True)
    followed = followed if leaf else followed * 2
    other = torch.randn(5, 2, 16, requires_grad=True)

    def calls(q_out, k_out):
        return [lambda: kernels.rotary(q, k, positions, table, out=(q_out, k_out)),
                lambda: kernels.qk_norm_rotary(q, k, positions, table, None, None, out=(q_out, k_out)),
                lambda: kernels.qk_norm_rotary_backward(q, k, q, k, positions, table, None, None, out=(q_out, k_out))]

    for out in ((followed, None), (followed[:, :, :], torch.empty_like(k)), (None, other)):
        for call in calls(*out):
            with pytest.raises(_lib.UnsupportedCall, match="requires a gradient"):
                call()
        with torch.no_grad():  # nothing is recorded: only the device is missing here
            for call in calls(*out):
                with pytest.raises(_lib.UnsupportedCall, match="CUDA device"):
                    call()


# --------------------------------------------------------------------------- outputs that lie between others
class HeadsView(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("batch_stride", ctypes.c_int64), ("token_stride", ctypes.c_int64),
                ("head_stride", ctypes.c_int64), ("heads", ctypes.c_int64)]


class Rotary(ctypes.Structure):
    _fields_ = [("positions", ctypes.c_void_p), ("batch_stride", ctypes.c_int64), ("token_stride", ctypes.c_int64),
                ("axis_stride", ctypes.c_int64), ("quarters", ctypes.c_void_p), ("pair_axes", ctypes.c_void_p),
                ("position_type", ctypes.c_int), ("axes", ctypes.c_int), ("pairs", ctypes.c_int), ("interleaved", ctypes.c_int),
                ("inverse", ctypes.c_int)]


BASE = 0x1000000
no_gpu = pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses: only where no launch can follow")


def taken(q, k, batch, tokens, channels, dtype):
    """Whether q and k, each ``(first element, strides of batch, token and head, heads)`` of memory at an address that is
    never read, may both be written in place: True where all checks passed and no device was found."""
    size = 4 if dtype == 1 else 2
    views = [HeadsView(BASE + size * v[0], *v[1:]) for v in (q, k)]
    at = [ctypes.cast(ctypes.pointer(v), ctypes.c_void_p) for v in views]
    rotary = Rotary()
    status = _lib.load().ffb_rotary_fwd(*at, *at, ctypes.cast(ctypes.pointer(rotary), ctypes.c_void_p), batch, tokens, channels, dtype, None)
    assert status in (1, 3)
    return status == 3


def elements(view, batch, tokens, channels):
    start, sb, st, sh, heads = view
    return [start + b * sb + t * st + h * sh + c for b in range(batch) for t in range(tokens) for h in range(heads) for c in range(channels)]


def strides(order, sizes):
    """Dense strides of axes named from the outermost in; those of the letters b, t, h"""
    step, found = 1, {}
    for axis in reversed(order):
        found[axis] = step
        step *= sizes[axis]
    return tuple(found[a] for a in "bth")


@needs_library
@no_gpu
@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("batch,tokens", [(1, 1), (1, 5), (3, 1), (3, 5)])
@pytest.mark.parametrize("order", ["bthd", "bhtd", "tbhd", "thbd", "hbtd", "htbd"])
def test_parts_of_one_tensor_are_taken(order, batch, tokens, dtype):
    """q and k as parts of one dense tensor, its axes in any order (head-major [batch, heads, tokens, d] among them): other
    heads, or other channels of the same heads, at the front or at the back."""
    d = 8
    for heads, q, k in ((9, (0, 4), (4, 2)), (9, (6, 3), (2, 4)), (2, (0, 1), (1, 1))):
        s = strides(order, {"b": batch, "t": tokens, "h": heads, "d": d})
        assert taken((q[0] * s[2], *s, q[1]), (k[0] * s[2], *s, k[1]), batch, tokens, d, dtype)
        assert not taken((q[0] * s[2], *s, q[1]), (q[0] * s[2] + d // 2, *s, q[1]), batch, tokens, d, dtype)
    s = strides(order, {"b": batch, "t": tokens, "h": 4, "d": 2 * d})
    assert taken((0, *s, 4), (d, *s, 4), batch, tokens, d, dtype) and taken((d, *s, 4), (0, *s, 2), batch, tokens, d, dtype)
    assert not taken((0, *s, 4), (d - 1, *s, 4), batch, tokens, d, dtype)
    assert not taken((0, *s, 4), (d + 1, *s, 4), batch, tokens, d, dtype)


@needs_library
@no_gpu
def test_what_is_taken_shares_no_element():
    """Small views of any strides: one that is taken was found to share nothing, element by element."""
    rng = random.Random(3)
    found = {True: 0, False: 0}
    for _ in range(20000):
        batch, tokens, channels = rng.choice([1, 2, 3]), rng.choice([1, 2, 3]), rng.choice([1, 2, 4])

        def view():
            heads = rng.choice([1, 2, 3])
            sizes = {"b": batch + rng.choice([0, 0, 1]), "t": tokens + rng.choice([0, 0, 1]), "h": rng.choice([heads, 6]),
                     "d": channels * rng.choice([1, 1, 2])}
            return (rng.randrange(40), *strides(rng.choice(["bthd", "bhtd", "tbhd", "thbd", "hbtd", "htbd"]), sizes), heads)

        q = view()
        k = view() if rng.random() < 0.5 else (rng.randrange(40), *q[1:4], rng.choice([1, 2, 3]))
        one, other = elements(q, batch, tokens, channels), elements(k, batch, tokens, channels)
        if taken(q, k, batch, tokens, channels, 1):
            assert not set(one) & set(other), (q, k, batch, tokens, channels)
        found[not set(one) & set(other)] += 1
    assert min(found.values()) > 2000
