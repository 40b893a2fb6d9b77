"""Refusals of the operators around an attention, their tables and their plain forms, without a GPU."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import attention_reference as ref
from foldforge_b200 import _lib, kernels

needs_library = pytest.mark.skipif(not (_lib.LIBRARY.exists() and (_lib.LIBRARY.parent / "_binding.so").exists()),
                                   reason="library not built")
BF16, F32 = 0, 1


# --------------------------------------------------------------------------- the generator
def test_philox_known_answers():
    """The published test vectors of Philox4x32-10 (Random123's known answers)."""
    ones = 0xFFFFFFFF
    assert ref.philox((0, 0, 0, 0), (0, 0)) == (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)
    assert ref.philox((ones,) * 4, (ones,) * 2) == (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)
    assert ref.philox((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0)) == \
        (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)


def test_words_are_philox():
    index = torch.tensor([0, 1, 2, 3, 4, 11, 2**34 - 1, 2**34, 2**36 + 5])
    for seed, offset in ((0, 0), (2**40 + 3, 7), (-1, 2**33 + 1)):
        got = ref.words(index, seed, offset).tolist()
        s, o = seed % 2**64, offset % 2**64
        for i, w in zip(index.tolist(), got, strict=True):
            g = i // 4
            assert w == ref.philox((g % 2**32, g >> 32, o % 2**32, o >> 32), (s % 2**32, s >> 32))[i % 4]


# --------------------------------------------------------------------------- tables and plain forms
def test_rotary_table():
    f = kernels.rotary_frequencies(8)
    assert f == [1.0, 0.1, 0.01, pytest.approx(0.001)]
    table = kernels.rotary_table(f, [0, 0, 2, 1], device="cpu")
    assert table.axes == 3 and not table.interleaved and table.pair_axes.dtype == torch.int32
    assert torch.allclose(table.quarters, torch.tensor(f, dtype=torch.float64) * 2 / math.pi, rtol=1e-15, atol=0)
    assert kernels.rotary_table([], device="cpu").axes == 1
    for bad in ((f, [0, 0, 0]), (f, [0, 0, 0, 16]), (f, [0, 0, 0, -1]), ([float("nan")], None), ([[1.0]], None), ([math.inf], None)):
        with pytest.raises(ValueError):
            kernels.rotary_table(*bad, device="cpu")


@pytest.mark.parametrize("interleaved", [False, True])
def test_reference_gradients_against_differences(interleaved):
    g = torch.Generator().manual_seed(1)
    x, w = torch.randn(2, 4, 3, 10, generator=g, dtype=torch.float64), torch.randn(10, generator=g, dtype=torch.float64)
    dy = torch.randn(2, 4, 3, 10, generator=g, dtype=torch.float64)
    angle = ref.angles(torch.randint(0, 99, (2, 4, 2), generator=g), [1.0, 0.3, 0.01, 0.5], [0, 1, 1, 0])

    def loss(x, w):
        return (ref.heads(x, angle, interleaved, w, 1e-6)[0][0] * dy).sum()

    (_, dx, dw), _ = ref.heads(x, angle, interleaved, w, 1e-6, dy)
    for _ in range(5):
        ax, aw = torch.randn(x.shape, generator=g, dtype=torch.float64), torch.randn(10, generator=g, dtype=torch.float64)
        h = 1e-6
        difference = (loss(x + h * ax, w + h * aw) - loss(x - h * ax, w - h * aw)) / (2 * h)
        assert abs(difference - (dx * ax).sum() - (dw * aw).sum()) < 1e-6


# --------------------------------------------------------------------------- refusals of the torch-facing calls
def heads_call(**changes):
    table = kernels.rotary_table(kernels.rotary_frequencies(16), device="cpu")
    args = dict(q=torch.randn(2, 5, 4, 16), k=torch.randn(2, 5, 2, 16), positions=torch.zeros(2, 5, 1, dtype=torch.int64), table=table,
                q_weight=torch.ones(16), k_weight=torch.ones(16))
    args.update(changes)
    return args


@needs_library
def test_cpu_tensors_are_refused():
    a = heads_call()
    x = torch.randn(4, 8)
    for call in (lambda: kernels.qk_norm_rotary(**a), lambda: kernels.rotary(a["q"], a["k"], a["positions"], a["table"]),
                 lambda: kernels.qk_norm_rotary_backward(a["q"], a["k"], *a.values()), lambda: kernels.dropout_train(x, 0.5, 1),
                 lambda: kernels.dropout_backward(x, kernels.DropoutSaved(0.5, 1, 0, (), x.shape, x.dtype, x.dtype))):
        with pytest.raises(_lib.UnsupportedCall, match="CUDA device"):
            call()


@needs_library
def test_shapes_and_dtypes_of_heads_are_refused():
    a = heads_call()
    t = a["table"]
    bad = [
        dict(q=a["q"].half()), dict(k=a["k"].bfloat16()), dict(q=torch.randn(5, 16)), dict(q=torch.randn(2, 2, 5, 4, 16)),
        dict(k=torch.randn(2, 6, 2, 16)), dict(k=torch.randn(2, 5, 2, 15)), dict(k=torch.randn(5, 2, 16)), dict(k=torch.randn(1, 5, 2, 16)),
        dict(q=torch.randn(2, 5, 4, 0)), dict(q=torch.randn(2, 5, 4, 513), k=None, k_weight=None, q_weight=None),
        dict(positions=None), dict(table=None), dict(positions=torch.zeros(2, 5, dtype=torch.int64)), dict(positions=torch.zeros(2, 5, 1).double()),
        dict(positions=torch.zeros(2, 5, 1, dtype=torch.bool)), dict(positions=torch.zeros(2, 6, 1)), dict(positions=torch.zeros(3, 5, 1)),
        dict(positions=torch.zeros(1, 1, 1)), dict(positions=torch.zeros(2, 5, 0)), dict(positions=torch.zeros(2, 5, 1, 1)),
        dict(table=t._replace(axes=2)), dict(table=t._replace(axes=0)), dict(table=t._replace(quarters=t.quarters.float())),
        dict(table=t._replace(pair_axes=t.pair_axes.long())), dict(table=t._replace(pair_axes=t.pair_axes[:7])),
        dict(table=kernels.rotary_table([1.0] * 9, device="cpu")), dict(table=t._replace(quarters=torch.zeros(16, dtype=torch.float64)[::2])),
        dict(q_weight=torch.ones(15)), dict(k_weight=torch.ones(2, 16)), dict(q_weight=torch.ones(16, dtype=torch.int32)), dict(k=None),
        dict(out=(torch.empty(2, 5, 4, 16), None, None)[:2], k=None), dict(out=(torch.empty(2, 5, 4, 15), torch.empty(2, 5, 2, 16))),
        dict(out=(torch.empty(2, 5, 4, 16).bfloat16(), torch.empty(2, 5, 2, 16))), dict(out=(torch.empty(2, 5, 4, 32)[..., ::2], None)),
        dict(out=(None, torch.empty(2, 5, 3, 16))),
    ]
    for changes in bad:
        with pytest.raises(_lib.UnsupportedCall):
            kernels.qk_norm_rotary(**heads_call(**changes))
    q, k = a["q"], a["k"]
    rest = (q, k, a["positions"], t, a["q_weight"], a["k_weight"])
    for call in (lambda: kernels.qk_norm_rotary_backward(q[:, :4], k, *rest), lambda: kernels.qk_norm_rotary_backward(q.bfloat16(), k, *rest),
                 lambda: kernels.qk_norm_rotary_backward(q, None, *rest), lambda: kernels.qk_norm_rotary_backward(q, k[:, :, :1], *rest),
                 lambda: kernels.qk_norm_rotary_backward(q, k, *rest, out=(torch.empty(2, 5, 4, 15), None)),
                 lambda: kernels.qk_norm_rotary_backward(q, k, q, None, *rest[2:])):
        with pytest.raises(_lib.UnsupportedCall):
            call()
    with pytest.raises(TypeError):
        kernels.rotary(q, k, None, t)


@needs_library
def test_dropout_refusals():
    x = torch.randn(3, 4, 5)
    for args, kwargs in [((x.half(), 0.1, 1), {}), ((x.int(), 0.1, 1), {}), ((x, -0.1, 1), {}), ((x, 1.1, 1), {}), ((x, float("nan"), 1), {}),
                         ((x, 0.1, 1), dict(residual=x[:2])), ((x, 0.1, 1), dict(residual=x.half())), ((x, 0.1, 1), dict(shared=3)),
                         ((x, 0.1, 1), dict(shared=-4)), ((x, 0.1, 1), dict(shared=(0, 2))), ((x, 0.1, 1), dict(shared=(1, 1))),
                         ((x, 0.1, torch.zeros(2)), {}), ((x, 0.1, torch.zeros(3, dtype=torch.int64)), {}),
                         ((x, 0.1, torch.zeros(4, dtype=torch.int64)[::2]), {}), ((torch.tensor(1.0), 0.1, 1), dict(shared=0))]:
        with pytest.raises(_lib.UnsupportedCall):
            kernels.dropout_train(*args, **kwargs)
    for seed in (1.5, "1", None):
        with pytest.raises(TypeError):
            kernels.dropout_train(x, 0.1, seed)
    saved = kernels.DropoutSaved(0.1, 1, 0, (), x.shape, torch.bfloat16, x.dtype)
    for dout in (x[:2], x.bfloat16(), x.reshape(12, 5)):
        with pytest.raises(_lib.UnsupportedCall):
            kernels.dropout_backward(dout, saved)


# --------------------------------------------------------------------------- refusals of the C ABI
class HeadsView(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("batch_stride", ctypes.c_int64), ("token_stride", ctypes.c_int64),
                ("head_stride", ctypes.c_int64), ("heads", ctypes.c_int64)]


class Rotary(ctypes.Structure):
    _fields_ = [("positions", ctypes.c_void_p), ("batch_stride", ctypes.c_int64), ("token_stride", ctypes.c_int64),
                ("axis_stride", ctypes.c_int64), ("quarters", ctypes.c_void_p), ("pair_axes", ctypes.c_void_p),
                ("position_type", ctypes.c_int), ("axes", ctypes.c_int), ("pairs", ctypes.c_int), ("interleaved", ctypes.c_int),
                ("inverse", ctypes.c_int)]


def view(address, batch, token, head, heads):
    return HeadsView(address, batch, token, head, heads)


def turning(**changes):
    r = dict(positions=0x1000, batch_stride=0, token_stride=1, axis_stride=1, quarters=0x2000, pair_axes=0x3000, position_type=1, axes=1,
             pairs=8, interleaved=0, inverse=0)
    r.update(changes)
    return Rotary(*r.values())


def ref_to(s):
    return None if s is None else ctypes.cast(ctypes.pointer(s), ctypes.c_void_p)


Q, K, QO, KO = 0x100000, 0x200000, 0x300000, 0x400000


def norm_status(q=None, k=None, qo=None, ko=None, r=None, batch=2, tokens=5, channels=16, dtype=F32, eps=1e-6, qw=None, kw=None):
    """The status of a call at addresses that are never read: a refusal (1 or 2), or 3 where all checks passed and
    no device was found."""
    q = q or view(Q, 320, 64, 16, 4)
    qo = qo or view(QO, 320, 64, 16, 4)
    lib = _lib.load()
    return lib.ffb_qk_norm_rotary_fwd(ref_to(q), ref_to(k), ref_to(qo), ref_to(ko), qw, kw, eps, ref_to(r or turning()), batch, tokens,
                                      channels, dtype, None)


no_gpu = pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses: only where no launch can follow")


@needs_library
@no_gpu
def test_c_abi_takes_good_calls():
    assert norm_status() not in (0, 1, 2)
    assert norm_status(k=view(K, 160, 32, 16, 2), ko=view(KO, 160, 32, 16, 2)) not in (0, 1, 2)
    assert norm_status(qo=view(Q, 320, 64, 16, 4)) not in (0, 1, 2)  # in place
    # q and k of packed rows, each in place, and written side by side to others
    assert norm_status(q=view(Q, 960, 192, 16, 4), k=view(Q + 256, 960, 192, 16, 4), qo=view(Q, 960, 192, 16, 4),
                       ko=view(Q + 256, 960, 192, 16, 4)) not in (0, 1, 2)
    # tokens before the batch in memory
    assert norm_status(q=view(Q, 192, 384, 16, 4), k=view(Q + 256, 192, 384, 16, 4), qo=view(Q, 192, 384, 16, 4),
                       ko=view(Q + 256, 192, 384, 16, 4)) not in (0, 1, 2)
    assert norm_status(tokens=0) == 0 and norm_status(batch=0) == 0
    assert norm_status(r=turning(pairs=0, positions=None, quarters=None, pair_axes=None)) not in (0, 1, 2)


@needs_library
@no_gpu
@pytest.mark.parametrize("status,changes", [
    (1, dict(batch=-1)), (1, dict(tokens=-1)), (1, dict(channels=0)), (2, dict(channels=513)), (2, dict(dtype=2)),
    (2, dict(batch=2**16, tokens=2**16)), (2, dict(batch=2**40)), (1, dict(eps=-1.0)), (1, dict(eps=float("nan"))), (1, dict(eps=float("inf"))),
    (1, dict(q=view(0, 320, 64, 16, 4))), (1, dict(q=view(Q + 2, 320, 64, 16, 4))), (1, dict(q=view(Q, -320, 64, 16, 4))),
    (1, dict(q=view(Q, 320, 2**60, 16, 4))), (1, dict(q=view(Q, 320, 64, 16, -1), qo=view(QO, 320, 64, 16, -1))),
    (2, dict(q=view(Q, 0, 0, 16, 2**21), qo=view(QO, 0, 0, 16, 2**21))),
    (1, dict(qo=view(QO, 320, 64, 16, 3))), (1, dict(qo=view(QO, 320, 64, 8, 4))), (1, dict(qo=view(QO, 0, 64, 16, 4))),
    (1, dict(qo=view(QO, 320, 63, 16, 4))), (1, dict(qo=view(Q + 64, 320, 64, 16, 4))), (1, dict(qo=view(Q, 320, 64, 16, 4), q=view(Q, 640, 64, 16, 4))),
    (1, dict(k=view(K, 160, 32, 16, 2))), (1, dict(ko=view(KO, 160, 32, 16, 2))),
    (1, dict(k=view(K, 160, 32, 16, 2), ko=view(QO, 160, 32, 16, 2))), (1, dict(k=view(K, 160, 32, 16, 2), ko=view(Q, 160, 32, 16, 2))),
    # packed rows, k's output over the last head of q's
    (1, dict(k=view(K, 160, 32, 16, 2), qo=view(QO, 960, 192, 16, 4), ko=view(QO + 192, 960, 192, 16, 2))),
    # rows whose parts reach into the next row
    (1, dict(k=view(K, 160, 32, 16, 2), qo=view(QO, 400, 80, 16, 4), ko=view(QO + 256, 400, 80, 16, 2))),
    # rows that interleave with the batch's
    (1, dict(k=view(K, 160, 32, 16, 2), qo=view(QO, 500, 192, 16, 4), ko=view(QO + 256, 500, 192, 16, 4))),
    (1, dict(qw=0x1004)), (1, dict(kw=0x1008)),
    (1, dict(r=turning(pairs=-1))), (1, dict(r=turning(pairs=9))), (2, dict(r=turning(axes=0))), (2, dict(r=turning(axes=17))),
    (2, dict(r=turning(position_type=3))), (1, dict(r=turning(positions=None))), (1, dict(r=turning(quarters=None))),
    (1, dict(r=turning(pair_axes=None))), (1, dict(r=turning(positions=0x1004))), (1, dict(r=turning(quarters=0x2004))),
    (1, dict(r=turning(token_stride=-1))), (1, dict(r=turning(token_stride=2**60))),
])
def test_c_abi_refuses(status, changes):
    assert norm_status(**changes) == status


@needs_library
@no_gpu
def test_c_abi_refuses_a_backward_pass():
    lib = _lib.load()
    x, dy, dx = view(Q, 320, 64, 16, 4), view(QO, 320, 64, 16, 4), view(KO, 320, 64, 16, 4)

    def status(dy=dy, x=x, dx=dx, dqw=0x5000, dkw=None, ws=0x6000, size=None, dk=None):
        need = lib.ffb_qk_norm_rotary_bwd_workspace_bytes(2, 5, 4, 0, 16, F32)
        return lib.ffb_qk_norm_rotary_bwd(ref_to(dy), dk, ref_to(x), None, ref_to(dx), None, None, None, dqw, dkw, 1e-6,
                                          ref_to(turning()), ws, need if size is None else size, 2, 5, 16, F32, None)

    assert status() not in (0, 1, 2) and status(dqw=None, ws=None, size=0) not in (0, 1, 2)
    assert status(dx=x) not in (0, 1, 2) and status(dx=dy) not in (0, 1, 2)  # over what the same places are read from
    assert status(dqw=0x5002) == 1 and status(dkw=0x7000) == 1 and status(dy=None) == 1 and status(dx=None) == 1 and status(x=None) == 1
    assert status(dx=view(QO + 4, 320, 64, 16, 4)) == 1 and status(dx=view(Q + 128, 320, 64, 16, 4)) == 1
    assert status(dk=ref_to(dy)) == 1
    if lib.ffb_qk_norm_rotary_bwd_workspace_bytes(2, 5, 4, 0, 16, F32) > 0:
        assert status(ws=None) == 1 and status(size=1) == 1 and status(ws=0x6004) == 1
    for sizes in ((-1, 5, 4, 0, 16), (2, -5, 4, 0, 16), (2, 5, -4, 0, 16), (2, 5, 4, 0, 0), (2, 5, 4, 0, 513), (2**31, 2, 1, 1, 16)):
        assert lib.ffb_qk_norm_rotary_bwd_workspace_bytes(*sizes, F32) == 0


@needs_library
@no_gpu
def test_c_abi_of_dropout():
    lib = _lib.load()

    def status(x=0x10000, xt=BF16, residual=None, out=0x20000, ot=BF16, outer=1, shared=1, inner=64, p=0.5, device=None):
        return lib.ffb_dropout(x, xt, residual, out, ot, outer, shared, inner, p, 1, 0, device, None)

    assert status() not in (0, 1, 2) and status(out=0x10000) not in (0, 1, 2) and status(residual=0x20000) not in (0, 1, 2)
    for n in (dict(outer=0), dict(shared=0), dict(inner=0)):
        assert status(**n) == 0
    for bad in (dict(outer=-1), dict(shared=-1), dict(inner=-1), dict(p=-0.1), dict(p=1.01), dict(p=float("nan")), dict(x=None),
                dict(out=None), dict(x=0x10001), dict(out=0x20001), dict(residual=0x30001), dict(device=0x7004), dict(out=0x10002),
                dict(out=0x10000, ot=F32), dict(residual=0x20004), dict(out=0x10000 + 126)):
        assert status(**bad) == 1, bad
    for bad in (dict(xt=2), dict(ot=-1), dict(outer=2**40, shared=2**40), dict(inner=2**47), dict(outer=2**45, inner=4)):
        assert status(**bad) == 2, bad
