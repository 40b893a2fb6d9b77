"""The norm and rotation of queries and keys against their definitions in 64 bits (B200 only)."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

import attention_reference as ref  # noqa: E402
from foldforge_b200 import _lib, kernels  # noqa: E402
from training_reference import worst  # noqa: E402

BF16, F32 = torch.bfloat16, torch.float32
EPS = 1e-6


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    torch.cuda.synchronize()
    assert _lib.device_error() == 0


def gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def values(g, *shape, dtype=BF16, size=1.0):
    spread = torch.exp(torch.randn(shape[-1], device="cuda", generator=g))
    return (size * (torch.randn(shape, device="cuda", generator=g) * spread + 0.3)).to(dtype)


def weights(g, c):
    return 1 + 0.3 * torch.randn(c, device="cuda", generator=g)


class Turn:
    """Frequencies on ``axes`` axes over ``pairs`` pairs, and positions."""

    def __init__(self, g, batch, tokens, pairs, axes=1, interleaved=False, kind="line", start=0):
        self.pair_axes = [i * axes // max(1, pairs) for i in range(pairs)]
        self.frequencies = [10000.0 ** (-i / max(1, pairs)) for i in range(pairs)]
        self.interleaved = interleaved
        self.table = kernels.rotary_table(self.frequencies, self.pair_axes, interleaved=interleaved)
        if kind == "points":
            self.positions = 30 * torch.randn(batch, tokens, axes, device="cuda", generator=g)
        else:
            self.positions = (start + torch.arange(tokens, device="cuda")[:, None] * 3
                              + 1000 * torch.arange(axes, device="cuda")).expand(batch, tokens, axes)
            self.positions = self.positions + 17 * torch.arange(batch, device="cuda")[:, None, None]

    def angles(self, dims=4):
        positions = self.positions if dims == 4 else self.positions[0]
        return ref.angles(positions, self.frequencies, self.pair_axes)


def check(got, want, bounds, dtypes, what=""):
    for i, (a, b, e, t) in enumerate(zip(got, want, bounds, dtypes, strict=True)):
        assert a.dtype == t and a.shape == b.shape, (what, i)
        assert worst(a, b, e, t) <= 1, (what, i)


def run_norm(q, k, dq, dk, turn, qw, kw, out=None, grads=None):
    got = list(kernels.qk_norm_rotary(q, k, turn.positions, turn.table, qw, kw, EPS, out=out))
    got += kernels.qk_norm_rotary_backward(dq, dk, q, k, turn.positions, turn.table, qw, kw, EPS, out=grads)
    want, bounds = [None] * 6, [None] * 6
    for i, (x, dy, w) in enumerate(((q, dq, qw), (k, dk, kw))):
        (y, dx, dw), (ey, edx, edw) = ref.heads(x, turn.angles(), turn.interleaved, w, EPS, dy)
        want[i::2], bounds[i::2] = [y, dx, dw], [ey, edx, edw]
    t = q.dtype
    check(got, want, bounds, [t, t, t, t, F32, F32])


SIZES = [
    # batch, tokens, q heads, k heads, channels, pairs, axes
    (1, 1, 1, 1, 1, 0, 1), (1, 1, 1, 1, 2, 1, 1), (1, 1, 16, 16, 48, 24, 1), (1, 1, 32, 8, 128, 64, 1), (3, 7, 2, 1, 3, 1, 1),
    (2, 5, 4, 2, 16, 8, 2), (2, 65, 3, 3, 17, 6, 3), (1, 130, 16, 16, 24, 12, 1), (5, 33, 4, 4, 32, 15, 3),
    (2, 100, 7, 1, 40, 20, 2), (1, 77, 5, 5, 64, 32, 1), (1, 77, 5, 5, 64, 8, 1), (3, 41, 6, 2, 80, 25, 2), (2, 50, 3, 2, 96, 48, 3),
    (1, 200, 12, 4, 128, 64, 3), (1, 60, 8, 8, 128, 0, 1), (1, 9, 40, 10, 120, 60, 1), (2, 31, 3, 3, 151, 75, 2),
    (1, 1000, 4, 2, 160, 80, 1), (1, 20, 6, 3, 192, 96, 1), (1, 65, 2, 2, 256, 128, 2), (4, 64, 1, 1, 256, 64, 1), (2, 19, 3, 1, 257, 128, 1),
    (1, 33, 2, 2, 320, 160, 1), (1, 21, 2, 1, 511, 255, 1), (1, 300, 2, 2, 512, 256, 1), (64, 1, 32, 8, 64, 32, 1), (1, 5001, 8, 8, 48, 24, 1),
]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("b,t,hq,hk,d,pairs,axes", SIZES)
def test_norm_and_rotation(b, t, hq, hk, d, pairs, axes, dtype, interleaved):
    g = gen(d * 1009 + t)
    turn = Turn(g, b, t, pairs, axes, interleaved)
    q, k = values(g, b, t, hq, d, dtype=dtype), values(g, b, t, hk, d, dtype=dtype)
    dq, dk = values(g, b, t, hq, d, dtype=dtype, size=1e-2), values(g, b, t, hk, d, dtype=dtype, size=1e-2)
    run_norm(q, k, dq, dk, turn, weights(g, d), weights(g, d))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("b,t,hq,hk,d,pairs,axes", SIZES)
def test_rotation(b, t, hq, hk, d, pairs, axes, dtype, interleaved):
    g = gen(d * 1013 + t)
    turn = Turn(g, b, t, pairs, axes, interleaved, kind="points")
    q, k = values(g, b, t, hq, d, dtype=dtype), values(g, b, t, hk, d, dtype=dtype)
    got = kernels.rotary(q, k, turn.positions, turn.table)
    back = kernels.rotary(q, k, turn.positions, turn.table, inverse=True)
    for x, y, z in zip((q, k), got, back, strict=True):
        want, bounds = ref.heads(x, turn.angles(), interleaved, dy=x)
        check([y, z], want, bounds, [dtype, dtype])
        assert torch.equal(y[..., 2 * pairs:], x[..., 2 * pairs:])  # what is not turned stays bit for bit


@pytest.mark.parametrize("d", [48, 37])
@pytest.mark.parametrize("position_dtype", [torch.int32, torch.int64, F32])
@pytest.mark.parametrize("start", [0, 2**20, 2**23])
def test_far_positions(position_dtype, start, d):
    g = gen(1)
    turn = Turn(g, 2, 50, d // 2, 2, start=start)
    turn.positions = turn.positions.to(position_dtype)
    q, k = values(g, 2, 50, 4, d, dtype=F32), values(g, 2, 50, 2, d, dtype=F32)
    got = kernels.rotary(q, k, turn.positions, turn.table)
    for x, y in zip((q, k), got, strict=True):
        check([y], *ref.heads(x, turn.angles(), False), [F32])
    negative = kernels.rotary(q, k, -turn.positions, turn.table)
    back = kernels.rotary(q, k, turn.positions, turn.table, inverse=True)
    assert all(torch.equal(a, b) for a, b in zip(negative, back, strict=True))


def test_quarter_turns_are_exact():
    """A frequency of a quarter turn: cosine and sine are 0 and 1 at every whole position, far ones too."""
    table = kernels.rotary_table([torch.pi / 2] * 4)._replace(quarters=torch.ones(4, dtype=torch.float64, device="cuda"))
    positions = torch.tensor([0, 1, 2, 3, 4, 5, 2**40 + 1, -1, -2, -3], device="cuda")[:, None]
    q = values(gen(2), 10, 3, 8, dtype=F32)
    y, _ = kernels.rotary(q, None, positions, table)
    for i, turns in enumerate((0, 1, 2, 3, 0, 1, 1, 3, 2, 1)):
        a, b = q[i, :, :4], q[i, :, 4:]
        for _ in range(turns):
            a, b = -b, a
        assert torch.equal(y[i], torch.cat([a, b], -1)), i


@pytest.mark.parametrize("d", [24, 48, 64, 67, 128])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_layouts(d, dtype):
    """Views of packed rows, head-major tensors, heads that repeat, rows off 16 bytes, channels apart."""
    g = gen(d)
    b, t = 2, 35
    turn = Turn(g, b, t, d // 2, 2)
    qw, kw = weights(g, d), weights(g, d)
    packed = values(g, b, t, 9, d, dtype=dtype)
    head_major = values(g, b, 5, t, d, dtype=dtype).transpose(1, 2)
    flat = values(g, 1, b * t * 3 * d + 1, dtype=dtype)[0, 1:].view(b, t, 3, d)
    for q, k in ((packed[:, :, :4], packed[:, :, 4:6]), (head_major, packed[:, :, 6:]), (flat, flat[:, :, :1].expand(b, t, 4, d)),
                 (values(g, t, b, 3, d, dtype=dtype).transpose(0, 1), values(g, b, t, 2, 2 * d, dtype=dtype)[..., ::2]),
                 (values(g, 1, t, 3, d, dtype=dtype).expand(b, t, 3, d), values(g, b, t, 3, d + 3, dtype=dtype)[..., 3:])):
        dq, dk = (values(g, *x.shape, dtype=dtype, size=1e-2) for x in (q, k))
        run_norm(q, k, dq, dk.transpose(1, 2).contiguous().transpose(1, 2), turn, qw, kw)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("d", [48, 50, 128])
def test_outputs_of_the_caller(d, dtype):
    """In place, side by side in packed rows, in a cache's slots; what lies around them stays."""
    g = gen(7)
    b, t = 3, 20
    turn = Turn(g, b, t, d // 2)
    qw, kw = weights(g, d), weights(g, d)
    rows = values(g, b, t, 8, d, dtype=dtype)
    q, k = rows[:, :, :4], rows[:, :, 4:6]
    want = kernels.qk_norm_rotary(q, k, turn.positions, turn.table, qw, kw, EPS)
    target = torch.full_like(rows, 7.0)
    got = kernels.qk_norm_rotary(q, k, turn.positions, turn.table, qw, kw, EPS, out=(target[:, :, :4], target[:, :, 4:6]))
    assert got[0].data_ptr() == target.data_ptr()
    assert torch.equal(target[:, :, :4], want[0]) and torch.equal(target[:, :, 4:6], want[1]) and bool((target[:, :, 6:] == 7).all())
    cache = torch.full((b, 2, 64, d), 5.0, device="cuda", dtype=dtype)  # [batch, heads, places, channels]
    kernels.qk_norm_rotary(q, k, turn.positions, turn.table, qw, kw, EPS, out=(target[:, :, :4], cache[:, :, 30:30 + t].transpose(1, 2)))
    assert torch.equal(cache[:, :, 30:30 + t].transpose(1, 2), want[1])
    assert bool((cache[:, :, :30] == 5).all()) and bool((cache[:, :, 30 + t:] == 5).all())
    dq, dk = values(g, *q.shape, dtype=dtype), values(g, *k.shape, dtype=dtype)
    gradients = kernels.qk_norm_rotary_backward(dq, dk, q, k, turn.positions, turn.table, qw, kw, EPS)
    again = kernels.qk_norm_rotary_backward(dq, dk, q, k, turn.positions, turn.table, qw, kw, EPS, out=(target[:, :, :4], target[:, :, 4:6]))
    assert all(torch.equal(x, y) for x, y in zip(gradients, again, strict=True))
    assert torch.equal(target[:, :, :4], gradients[0]) and bool((target[:, :, 6:] == 7).all())
    kept = rows.clone()
    turned = kernels.rotary(q, k, turn.positions, turn.table)
    kernels.rotary(q, k, turn.positions, turn.table, out=(q, k))
    assert torch.equal(q, turned[0]) and torch.equal(k, turned[1]) and torch.equal(rows[:, :, 6:], kept[:, :, 6:])


def test_without_weights_positions_or_k():
    g = gen(9)
    q, k = values(g, 30, 4, 64), values(g, 30, 2, 64)
    turn = Turn(g, 1, 30, 32)
    turn.positions = turn.positions[0]
    dq, dk = values(g, 30, 4, 64), values(g, 30, 2, 64)
    got = kernels.qk_norm_rotary(q, k, None, None, None, None, EPS)
    none = torch.zeros(30, 1, 0, device="cuda", dtype=torch.float64)
    for x, y in zip((q, k), got, strict=True):
        check([y], *ref.heads(x, none, False, None, EPS), [BF16])
    y, nothing = kernels.qk_norm_rotary(q, None, turn.positions, turn.table, None, None, EPS)
    assert nothing is None
    angle = ref.angles(turn.positions, turn.frequencies, turn.pair_axes)
    check([y], *ref.heads(q, angle, False, None, EPS), [BF16])
    out = kernels.qk_norm_rotary_backward(dq, dk, q, k, turn.positions, turn.table, None, None, EPS)
    assert out[2] is None and out[3] is None
    (_, dx, _), (_, edx, _) = ref.heads(q, angle, False, None, EPS, dq)
    check([out[0]], [dx], [edx], [BF16])
    w = weights(g, 64).bfloat16()  # of another type, on one side alone
    out = kernels.qk_norm_rotary_backward(dq, dk, q, k, turn.positions, turn.table, None, w, EPS)
    assert out[2] is None and out[3].dtype == F32
    (_, dx, dw), (_, edx, edw) = ref.heads(k, angle, False, w, EPS, dk)
    check([out[1], out[3]], [dx, dw], [edx, edw], [BF16, F32])
    frozen = kernels.qk_norm_rotary_backward(dq, dk, q, k, turn.positions, turn.table, None, w, EPS, weight_gradient=False)
    assert frozen[3] is None and torch.equal(frozen[0], out[0]) and torch.equal(frozen[1], out[1])
    only = kernels.qk_norm_rotary_backward(dk, None, k, None, turn.positions, turn.table, w, None, EPS)
    assert torch.equal(only[0], out[1]) and only[1] is None
    # alone, k's heads are shared out in another way, so its sums have another order: both lie within the sums' bound
    check([only[2]], [dw], [edw], [F32])


@pytest.mark.parametrize("shape", [(0, 4, 64), (2, 0, 4, 64), (0, 5, 4, 64), (5, 0, 64)])
def test_nothing_to_do(shape):
    q = torch.empty(shape, device="cuda", dtype=BF16)
    tokens = shape[-3]
    table = kernels.rotary_table(kernels.rotary_frequencies(64))
    positions = torch.zeros(tokens, 1, dtype=torch.int64, device="cuda")
    w = torch.ones(64, device="cuda")
    y, z = kernels.qk_norm_rotary(q, q, positions, table, w, w)
    assert y.shape == z.shape == shape
    dq, dk, dqw, dkw = kernels.qk_norm_rotary_backward(q, q, q, q, positions, table, w, w)
    assert dq.shape == shape and not dqw.any() and not dkw.any()


def test_heads_of_zeros_and_values_that_are_not_finite():
    """A head of zeros gives zeros; infinities and NaN stay in their own head (or pair, where only turned)."""
    g = gen(11)
    turn = Turn(g, 1, 12, 24)
    q = values(g, 1, 12, 4, 48)
    w = weights(g, 48)
    dq = values(g, 1, 12, 4, 48)
    clean = kernels.qk_norm_rotary(q, None, turn.positions, turn.table, w, None, EPS)[0]
    clean_dx = kernels.qk_norm_rotary_backward(dq, None, q, None, turn.positions, turn.table, w, None, EPS)[0]
    q[0, 3, 1], q[0, 4, 2, 5], q[0, 5, 0, 7], q[0, 6, 3, 40] = 0, float("nan"), float("inf"), -float("inf")
    y = kernels.qk_norm_rotary(q, None, turn.positions, turn.table, w, None, EPS)[0]
    dx = kernels.qk_norm_rotary_backward(dq, None, q, None, turn.positions, turn.table, w, None, EPS)[0]
    touched = torch.zeros(1, 12, 4, dtype=torch.bool, device="cuda")
    for at in ((3, 1), (4, 2), (5, 0), (6, 3)):
        touched[0, at[0], at[1]] = True
    assert not y[0, 3, 1].any() and bool(torch.isfinite(dx[0, 3, 1]).all())
    assert torch.equal(y[~touched], clean[~touched]) and torch.equal(dx[~touched], clean_dx[~touched])
    assert bool(y[0, 4, 2].isnan().all())
    turned = kernels.rotary(q, None, turn.positions, turn.table)[0]
    bad = ~torch.isfinite(turned)
    assert set(torch.nonzero(bad[0, 4, 2]).flatten().tolist()) == {5, 29}
    positions = turn.positions.to(F32).clone()
    positions[0, 2, 0] = float("nan")
    one = kernels.rotary(q, None, positions, turn.table)[0]
    assert bool(one[0, 2].isnan().all())
    rest = [i for i in range(12) if i != 2]
    assert torch.equal(one[0, rest].nan_to_num(), turned[0, rest].nan_to_num())


def test_an_axis_that_is_not_there():
    """A table made by hand whose axis is past the positions': the pair is NaN, the others are right."""
    q = values(gen(3), 5, 2, 16, dtype=F32)
    table = kernels.rotary_table([1.0] * 8)
    axes = table.pair_axes.clone()
    axes[3], axes[5] = 7, -1
    positions = torch.arange(5, device="cuda")[:, None]
    good = kernels.rotary(q, None, positions, table)[0]
    got = kernels.rotary(q, None, positions, table._replace(pair_axes=axes))[0]
    bad = [3, 5, 11, 13]
    rest = [i for i in range(16) if i not in bad]
    assert bool(got[..., bad].isnan().all()) and torch.equal(got[..., rest], good[..., rest])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_positions_of_several_forms(dtype):
    """Positions shared by the batch, with axes apart or in another order of memory, or without strides."""
    g = gen(21)
    q = values(g, 3, 40, 4, 48, dtype=dtype)
    table = kernels.rotary_table(kernels.rotary_frequencies(48), [0] * 12 + [2] * 12)
    positions = torch.randint(0, 5000, (40, 3), device="cuda", generator=g)
    want = kernels.rotary(q, None, positions.expand(3, 40, 3).contiguous(), table)[0]
    for p in (positions, positions[None], positions.expand(3, 40, 3), positions.t().contiguous().t(), positions.int(), positions.float(),
              torch.cat([positions, positions], 1), positions.expand(3, 40, 3).transpose(0, 1).contiguous().transpose(0, 1)):
        assert torch.equal(kernels.rotary(q, None, p, table)[0], want)
    one = positions[:1].expand(40, 3)
    assert torch.equal(kernels.rotary(q, None, one, table)[0], kernels.rotary(q, None, one.contiguous(), table)[0])


def test_offsets_past_32_bits():
    """Tokens more than 2^31 elements apart, in q and in the output."""
    buffer = torch.empty(2**32 + 2**10, device="cuda", dtype=BF16)
    g = gen(5)
    step = 2**31 + 64
    for d in (48, 33):
        far = buffer.as_strided((2, 3, d), (step, d, 1))
        q = values(g, 2, 3, d)
        far.copy_(q)
        turn = Turn(g, 1, 2, d // 2)
        w = weights(g, d)
        want = kernels.qk_norm_rotary(q, None, turn.positions[0], turn.table, w, None, EPS)[0]
        assert torch.equal(kernels.qk_norm_rotary(far, None, turn.positions[0], turn.table, w, None, EPS)[0], want)
        kernels.qk_norm_rotary(q, None, turn.positions[0], turn.table, w, None, EPS, out=(far, None))
        assert torch.equal(far, want)


@pytest.mark.parametrize("t,hq,hk,d,pairs,axes", [(70001, 1, 1, 16, 8, 1), (70001, 2, 1, 24, 12, 1), (40009, 4, 4, 32, 16, 3),
                                                  (40009, 4, 4, 32, 15, 5), (40009, 3, 1, 7, 3, 9), (1, 3, 3, 16, 8, 2), (33, 0, 2, 32, 16, 1),
                                                  (40009, 16, 16, 48, 24, 1), (30011, 9, 4, 24, 8, 2), (20011, 10, 3, 128, 64, 3),
                                                  (20011, 7, 5, 80, 40, 1), (20011, 6, 6, 56, 28, 1)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_tokens_that_share_a_warp(t, hq, hk, d, pairs, axes, dtype, interleaved):
    """Many tokens: several a warp, a number of them that leaves lanes without one."""
    g = gen(t + d)
    turn = Turn(g, 1, t, pairs, axes, interleaved)
    q, k = values(g, 1, t, hq, d, dtype=dtype), values(g, 1, t, hk, d, dtype=dtype)
    dq, dk = values(g, 1, t, hq, d, dtype=dtype, size=1e-2), values(g, 1, t, hk, d, dtype=dtype, size=1e-2)
    run_norm(q, k, dq, dk, turn, weights(g, d), weights(g, d))


@pytest.mark.parametrize("d", [24, 48, 64, 33])
def test_many_tokens_in_place(d):
    """q and k of packed rows over themselves, a batch with positions of its own, tokens before the batch in memory."""
    g = gen(d + 1)
    b, t = 3, 9001
    turn = Turn(g, b, t, d // 2, 2)
    qw, kw = weights(g, d), weights(g, d)
    rows = values(g, t, b, 7, d).transpose(0, 1)
    q, k = rows[:, :, :4], rows[:, :, 4:6]
    kept = rows.clone()
    want = kernels.qk_norm_rotary(q, k, turn.positions, turn.table, qw, kw, EPS)
    for x, y, w in zip((q, k), want, (qw, kw), strict=True):
        check([y], *ref.heads(x, turn.angles(), False, w, EPS), [BF16])
    got = kernels.qk_norm_rotary(q, k, turn.positions, turn.table, qw, kw, EPS, out=(q, k))
    assert got[0].data_ptr() == rows.data_ptr()
    assert torch.equal(rows[:, :, :4], want[0]) and torch.equal(rows[:, :, 4:6], want[1]) and torch.equal(rows[:, :, 6:], kept[:, :, 6:])
    rows.copy_(kept)
    dq, dk = values(g, b, t, 4, d, size=1e-2), values(g, b, t, 2, d, size=1e-2)
    want = kernels.qk_norm_rotary_backward(dq, dk, q, k, turn.positions, turn.table, qw, kw, EPS)
    got = kernels.qk_norm_rotary_backward(dq, dk, q, k, turn.positions, turn.table, qw, kw, EPS, out=(dq, dk))  # over the gradients
    assert all(torch.equal(x, y) for x, y in zip(got, want, strict=True)) and torch.equal(dq, want[0])


def test_more_tokens_than_a_grid_takes_at_once():
    g = gen(6)
    turn = Turn(g, 1, 120000, 8)
    q, k = values(g, 1, 120000, 2, 16), values(g, 1, 120000, 1, 16)
    dq, dk = values(g, 1, 120000, 2, 16, size=1e-2), values(g, 1, 120000, 1, 16, size=1e-2)
    run_norm(q, k, dq, dk, turn, weights(g, 16), weights(g, 16))


def test_results_repeat_and_replay():
    """The same call twice, on another stream, and captured: bit for bit the same; two graphs that take turns keep
    their own workspaces."""
    g = gen(8)
    turn = Turn(g, 2, 700, 24)
    qw, kw = weights(g, 48), weights(g, 48)
    sets = []
    for _ in range(2):
        q, k = values(g, 2, 700, 6, 48), values(g, 2, 700, 2, 48)
        sets.append((q, k, values(g, *q.shape, size=1e-2), values(g, *k.shape, size=1e-2)))

    def step(q, k, dq, dk):
        return [*kernels.qk_norm_rotary(q, k, turn.positions, turn.table, qw, kw, EPS),
                *kernels.qk_norm_rotary_backward(dq, dk, q, k, turn.positions, turn.table, qw, kw, EPS),
                *kernels.rotary(q, k, turn.positions, turn.table)]

    want = [step(*s) for s in sets]
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        again = step(*sets[0])
    torch.cuda.current_stream().wait_stream(other)
    assert all(torch.equal(a, b) for a, b in zip(again, want[0], strict=True))
    graphs, results = [], []
    for s in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(step(*s))
        graphs.append(graph)
    for _ in range(2):
        for graph in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for got, w in zip(results, want, strict=True):
        assert all(torch.equal(a, b) for a, b in zip(got, w, strict=True))


def test_gradients_are_those_of_the_plain_form():
    """Against autograd over the definition, and against differences of the loss along a direction."""
    g = gen(12)
    turn = Turn(g, 2, 9, 10, 2, interleaved=True)
    q = values(g, 2, 9, 3, 24, dtype=F32)
    w = weights(g, 24)
    dy = values(g, 2, 9, 3, 24, dtype=F32)
    x64, w64 = q.double().requires_grad_(), w.double().requires_grad_()

    def loss(x, weight):
        rstd = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
        return (ref.rotate(x * rstd * weight, turn.angles(), True) * dy.double()).sum()

    loss(x64, w64).backward()
    dx, _, dw, _ = kernels.qk_norm_rotary_backward(dy, None, q, None, turn.positions, turn.table, w, None, EPS)
    (_, _, _), (_, edx, edw) = ref.heads(q, turn.angles(), True, w, EPS, dy)
    check([dx, dw], [x64.grad, w64.grad], [edx, edw], [F32, F32])
    along_x, along_w = torch.randn_like(x64), torch.randn_like(w64)
    h = 1e-5
    with torch.no_grad():
        difference = (loss(x64 + h * along_x, w64 + h * along_w) - loss(x64 - h * along_x, w64 - h * along_w)) / (2 * h)
    slope = (dx.double() * along_x).sum() + (dw.double() * along_w).sum()
    # the bounds above along the direction, fp32's own rounding, and the difference's error of second order: each
    # value depends on h^2 / 6 of third derivatives below 100 of the values' size
    allowed = ((edx + ref.STEP * dx.abs()) * along_x.abs()).sum() + ((edw + ref.STEP * dw.abs()) * along_w.abs()).sum()
    allowed = allowed + h * h * 100 * (dy.double().abs().sum() + 1)
    assert abs(float(difference - slope)) <= float(allowed)
