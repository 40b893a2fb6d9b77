"""Operators around an attention, and their plain forms: what is timed and what it is compared with.

Three operators of a training or serving step on either side of an attention:

* ``qk_norm_rotary``: queries and keys of each head divided by their root mean square, scaled by a weight
  and turned by their positions' angles, and the backward pass (the gradients of q and k, and of the two
  weights reduced over tokens and heads).
* ``rotary``: the rotation alone, positions on one or several axes, and its backward pass (the rotation
  by the opposite angles).
* ``dropout``: an update dropped by a counter-based generator, scaled and added to its residual, the mask
  drawn again in the backward pass; one mask for all positions of an axis where ``shared`` names it.

Where ``own`` is false ``run`` computes the plain form from elementary torch operations; where it is true
it calls ``foldforge_b200.kernels``. ``exact`` is each operator's definition in 64 bits.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-6
LARGEST_HEADS = 65536 * 40 * 128  # elements of the q and k of the largest case listed
LARGEST_DROPOUT = 16384 * 4096  # elements of the largest dropout listed


def listed():
    return [
        # one new token of one sequence, 16 heads of 48: the smallest call, all latency
        _heads("qkn_step", "qk_norm_rotary", "forward", b=1, t=1, hq=16, hk=16, d=48, widths=[48]),
        # the token transformer's attention in training: 5 samples of 512 tokens, q and k views of a
        # projection's [q | k | v] rows
        _heads("qkn_tokens", "qk_norm_rotary", "train", b=5, t=512, hq=16, hk=16, d=48, widths=[48], packed=True),
        # a long sequence far from its beginning, four query heads for each key head
        _heads("qkn_long", "qk_norm_rotary", "train", b=1, t=65536, hq=32, hk=8, d=128, widths=[128], start=2**20),
        # fp32, odd length, two axes over a part of the channels, neighbouring channels paired
        _heads("qkn_odd_fp32", "qk_norm_rotary", "train", b=3, t=1237, hq=6, hk=2, d=80, widths=[26, 24], dtype="fp32",
               interleaved=True),
        # one new token for each of 64 sequences at positions of their own
        _heads("rot_step_batch", "rotary", "forward", b=64, t=1, hq=32, hk=8, d=64, widths=[64], start=30000),
        # atoms (3584 of them) by their coordinates, three axes, four heads of 32
        _heads("rot_atoms", "rotary", "train", b=1, t=3584, hq=4, hk=4, d=32, widths=[10, 10, 10], places="points"),
        # frames of a video: time, height and width
        _heads("rot_video", "rotary", "train", b=2, t=16 * 30 * 52, hq=24, hk=24, d=128, widths=[44, 42, 42],
               places="grid", interleaved=True),
        # one token's single row (c_s = 384): the smallest call
        _dropout("drop_one_row", [1, 384], 0.1),
        # the update of triangle multiplication over a 512-token crop, one mask for all rows
        _dropout("drop_pair_rows", [1, 512, 512, 128], 0.25, shared=1),
        # the ending node's update in fp32 beside a bf16 pair of 300 tokens, one mask for all columns
        _dropout("drop_pair_columns", [1, 300, 300, 128], 0.25, shared=2, dtype="fp32"),
        # a few sequences' wide activations, each element for itself
        _dropout("drop_wide", [16384, 4096], 0.1),
        # fp32 rows of an odd width, without a residual
        _dropout("drop_odd_fp32", [20011, 197], 0.15, dtype="fp32", residual=None),
    ]


def _heads(name, op, step, *, b, t, hq, hk, d, widths, dtype="bf16", interleaved=False, packed=False, start=0,
           places="line"):
    """A case of heads: ``widths`` are the channels turned by each axis, ``places`` what the positions are."""
    case = {"op": op, "step": step, "b": b, "t": t, "hq": hq, "hk": hk, "d": d,
            "widths": ",".join(str(w) for w in widths), "dtype": dtype, "interleaved": interleaved, "packed": packed,
            "start": start, "places": places}
    return dict(case, name=name) if name else case


def _dropout(name, shape, p, *, shared=None, dtype="bf16", residual="bf16"):
    case = {"op": "dropout", "shape": ",".join(str(n) for n in shape), "p": p, "shared": -1 if shared is None else shared,
            "dtype": dtype, "residual": residual or "none"}
    return dict(case, name=name) if name else case


def _numbers(text):
    return [int(n) for n in text.split(",")]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["qk_norm_rotary", "qk_norm_rotary", "rotary", "dropout", "dropout"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if op == "dropout":
        most = LARGEST_DROPOUT // (2 if dtype == "fp32" else 1)
        p = rng.choice([0.05, 0.1, 0.15, 0.25, 0.5])
        residual = rng.choice(["bf16", "fp32", None]) if dtype == "fp32" else rng.choice(["bf16", None])
        if rng.random() < 0.5:  # rows of any width
            c = _spread(rng, 1, 8192)
            c = max(8, c // 8 * 8) if rng.random() < 2 / 3 else c
            return _dropout(None, [_spread(rng, 1, most // c), c], p, dtype=dtype, residual=residual)
        c = rng.choice([32, 64, 128, 128, 33])  # a pair of any length
        n = _spread(rng, 2, int(math.sqrt(most / 2 / c)))
        return _dropout(None, [1, n, n, c], p, shared=rng.choice([None, 1, 2]), dtype=dtype, residual=residual)
    d = _spread(rng, 8, 256)
    if rng.random() < 2 / 3:
        d = max(16, d // 16 * 16)
    axes = rng.choice([1, 1, 2, 3])
    turned = d // 2 if rng.random() < 2 / 3 else rng.randint(axes, max(axes, d // 2))  # pairs
    widths = [2 * (turned // axes + (1 if i < turned % axes else 0)) for i in range(axes)]
    hk = _spread(rng, 1, 16)
    hq = hk * rng.choice([1, 1, 2, 4])
    most = LARGEST_HEADS // (2 if dtype == "fp32" else 1) // ((hq + hk) * d)
    tokens = _spread(rng, 1, min(most, 100000))
    b = min(tokens, rng.choice([1, 1, 2, 5, 16]))
    return _heads(None, op, rng.choice(["forward", "train", "train"]), b=b, t=max(1, tokens // b), hq=hq, hk=hk, d=d,
                  widths=widths, dtype=dtype, interleaved=rng.random() < 0.4, packed=rng.random() < 0.4,
                  start=rng.choice([0, 0, 30000, 2**20]), places=rng.choice(["line", "line", "points"]))


# --------------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _activation(gen, shape, dtype):
    """Channels of different spread, a few of them large, an offset."""
    c = shape[-1]
    spread = torch.exp(0.7 * torch.randn(c, device="cuda", generator=gen))
    offset = 0.3 * torch.randn(c, device="cuda", generator=gen)
    return torch.randn(shape, device="cuda", generator=gen).mul_(spread).add_(offset).to(dtype)


def _gradient(gen, shape, dtype):
    """A loss's gradient: small, its rows of different sizes."""
    size = 1e-3 * torch.exp(0.5 * torch.randn(*shape[:-1], 1, device="cuda", generator=gen))
    return torch.randn(shape, device="cuda", generator=gen).mul_(size).to(dtype)


def _ladder(case):
    """Each pair's frequency and axis: a geometric ladder from 1 down to nearly 1 / 10000 on every axis."""
    frequencies, axes = [], []
    for axis, width in enumerate(_numbers(case["widths"])):
        frequencies += [10000.0 ** (-2.0 * i / width) for i in range(width // 2)]
        axes += [axis] * (width // 2)
    return frequencies, axes


def _positions(gen, case):
    """``[b, t, axes]``: places on a line (each sequence's own beginning), points or a grid's coordinates."""
    b, t, n = case["b"], case["t"], len(_numbers(case["widths"]))
    if case["places"] == "points":
        return 20.0 * torch.randn(b, t, n, device="cuda", generator=gen)
    at = torch.arange(t, device="cuda")
    if case["places"] == "grid":
        grid = torch.stack([at // (30 * 52), at // 52 % 30, at % 52], -1)
        return grid.expand(b, t, 3)  # the samples share the grid
    first = case["start"] + torch.randint(0, 1000, (b, 1, 1), device="cuda", generator=gen)
    return first + at[:, None] + 1000 * torch.arange(n, device="cuda")


def prepare(case, seed):
    gen = _generator(seed)
    dtype = DTYPES[case["dtype"]]
    state = {"op": case["op"]}
    if case["op"] == "dropout":
        shape = _numbers(case["shape"])
        out_dtype = dtype if case["residual"] == "none" else DTYPES[case["residual"]]
        state.update(x=_activation(gen, shape, dtype), dout=_gradient(gen, shape, out_dtype), p=case["p"],
                     residual=None if case["residual"] == "none" else _activation(gen, shape, out_dtype),
                     shared=None if case["shared"] < 0 else case["shared"], seed=9021 * seed + 12345678901, offset=seed)
        return state
    b, t, hq, hk, d = (case[k] for k in ("b", "t", "hq", "hk", "d"))
    if case["packed"]:  # a projection's rows [q | k | v]
        rows = _activation(gen, (b, t, hq + 2 * hk, d), dtype)
        q, k = rows[:, :, :hq], rows[:, :, hq:hq + hk]
    else:
        q, k = _activation(gen, (b, t, hq, d), dtype), _activation(gen, (b, t, hk, d), dtype)
    state.update(q=q, k=k, positions=_positions(gen, case), train=case["step"] == "train")
    if state["train"]:
        state.update(dq=_gradient(gen, (b, t, hq, d), dtype), dk=_gradient(gen, (b, t, hk, d), dtype))
    if case["op"] == "qk_norm_rotary":
        state.update(q_weight=1.0 + 0.2 * torch.randn(d, device="cuda", generator=gen),
                     k_weight=1.0 + 0.2 * torch.randn(d, device="cuda", generator=gen))
    frequencies, axes = _ladder(case)
    if own:
        from foldforge_b200 import kernels

        state["table"] = kernels.rotary_table(frequencies, axes, interleaved=case["interleaved"], device="cuda")
    else:
        state["table"] = (torch.tensor(frequencies, dtype=torch.float64, device="cuda"),
                          torch.tensor(axes, device="cuda"), case["interleaved"])
    return state


def run(state):
    return _run_own(state) if own else _run_plain(state)


# --------------------------------------------------------------------------- the framework's calls
def _run_own(state):
    from foldforge_b200 import kernels

    if state["op"] == "dropout":
        out, saved = kernels.dropout_train(state["x"], state["p"], state["seed"], offset=state["offset"],
                                           residual=state["residual"], shared=state["shared"])
        return [out, kernels.dropout_backward(state["dout"], saved)]
    q, k, positions, table = state["q"], state["k"], state["positions"], state["table"]
    if state["op"] == "rotary":
        out = list(kernels.rotary(q, k, positions, table))
        if state["train"]:
            out += kernels.rotary(state["dq"], state["dk"], positions, table, inverse=True)
        return out
    weights = state["q_weight"], state["k_weight"]
    out = list(kernels.qk_norm_rotary(q, k, positions, table, *weights, EPS))
    if state["train"]:
        out += kernels.qk_norm_rotary_backward(state["dq"], state["dk"], q, k, positions, table, *weights, EPS)
    return out


# --------------------------------------------------------------------------- the plain forms
def _turned(x, cos, sin, interleaved):
    """fp32 ``x [b, t, heads, d]`` with its first pairs turned; ``cos, sin [b, t, 1, pairs]``."""
    n = cos.shape[-1]
    rest = x[..., 2 * n:]
    if interleaved:
        a, b = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
        both = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :n], x[..., n:2 * n]
        both = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([both, rest], -1)


def _run_plain(state):
    if state["op"] == "dropout":
        return _dropout_plain(state)
    frequencies, axes, interleaved = state["table"]
    # angles of far positions lose their last digits in 32 bits
    angle = (state["positions"].double()[..., axes] * frequencies)[:, :, None]
    cos, sin = angle.cos().float(), angle.sin().float()
    heads = [(state["q"], "q"), (state["k"], "k")]
    out, gradients, weight_gradients = [], [], []
    for x, name in heads:
        v = x.float()
        if state["op"] == "qk_norm_rotary":
            weight = state[name + "_weight"]
            rstd = torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS)
            out.append(_turned(v * rstd * weight, cos, sin, interleaved).to(x.dtype))
        else:
            out.append(_turned(v, cos, sin, interleaved).to(x.dtype))
        if state["train"]:
            g = _turned(state["d" + name].float(), cos, -sin, interleaved)
            if state["op"] == "qk_norm_rotary":
                xhat = v * rstd
                weight_gradients.append((g * xhat).sum((0, 1, 2)))
                g = g * weight
                g = rstd * (g - xhat * (g * xhat).mean(-1, keepdim=True))
            gradients.append(g.to(x.dtype))
    return out + gradients + weight_gradients


def _words(count, seed, offset):
    """``count`` 32-bit words of Philox4x32-10 (Salmon et al., "Parallel random numbers: as easy as 1, 2, 3",
    2011): key = the seed's two halves, counter = (word // 4 in two halves, the offset's two halves). Products of
    two 32-bit numbers wrap in 64-bit integers and keep their bits."""
    low = 0xFFFFFFFF
    group = torch.arange(-(-count // 4), dtype=torch.int64, device="cuda")
    c0, c1 = group & low, group >> 32
    c2, c3 = torch.full_like(group, offset & low), torch.full_like(group, offset >> 32 & low)
    k0, k1 = seed & low, seed >> 32 & low
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (p1 >> 32 & low) ^ c1 ^ k0, p1 & low, (p0 >> 32 & low) ^ c3 ^ k1, p0 & low
        k0, k1 = k0 + 0x9E3779B9 & low, k1 + 0xBB67AE85 & low
    return torch.stack([c0, c1, c2, c3], -1).flatten()[:count]


def _dropout_plain(state):
    x, p, shared = state["x"], state["p"], state["shared"]
    shape = list(x.shape)
    if shared is not None:
        shape[shared] = 1
    words = _words(math.prod(shape), state["seed"], state["offset"])
    keep = (words >= round(p * 2**32)).view(shape)
    scale = 1.0 / (1.0 - p)
    out = torch.where(keep, x.float() * scale, 0.0)
    if state["residual"] is not None:
        out = out + state["residual"].float()
    dx = torch.where(keep, state["dout"].float() * scale, 0.0)
    return [out.to(state["dout"].dtype), dx.to(x.dtype)]


# --------------------------------------------------------------------------- the definitions, in 64 bits
def _complex(x, n, interleaved):
    """The first n pairs of the last axis as complex numbers."""
    if interleaved:
        return torch.view_as_complex(x[..., :2 * n].unflatten(-1, (n, 2)).contiguous())
    return torch.complex(x[..., :n].contiguous(), x[..., n:2 * n].contiguous())


def _rotation(x, turn, interleaved):
    n = turn.shape[-1]
    z = torch.view_as_real(_complex(x, n, interleaved) * turn)
    y = x.clone()
    if interleaved:
        y[..., :2 * n] = z.flatten(-2)
    else:
        y[..., :n], y[..., n:2 * n] = z[..., 0], z[..., 1]
    return y


def _heads_exact(case, state):
    frequencies, axes = _ladder(case)
    frequencies = torch.tensor(frequencies, dtype=torch.float64, device="cuda")
    place = torch.stack([state["positions"][..., a] for a in axes], -1).double()
    angle = (place * frequencies)[:, :, None]
    turn, back = torch.polar(torch.ones_like(angle), angle), torch.polar(torch.ones_like(angle), -angle)
    norm, interleaved = case["op"] == "qk_norm_rotary", case["interleaved"]
    out, gradients, weight_gradients = [], [], []
    for name in ("q", "k"):
        v = state[name].double()
        if norm:
            w = state[name + "_weight"].double()
            sigma = (v.square().sum(-1, keepdim=True) / case["d"] + EPS).sqrt()
            normal = v / sigma
            out.append(_rotation(normal * w, turn, interleaved))
        else:
            out.append(_rotation(v, turn, interleaved))
        if case["step"] == "train":
            g = _rotation(state["d" + name].double(), back, interleaved)
            if norm:
                weight_gradients.append(torch.einsum("bthd,bthd->d", g, normal))
                along = torch.einsum("bthd,bthd->bth", g * w, normal)[..., None] / case["d"]
                g = (g * w - normal * along) / sigma
            gradients.append(g)
    return out + gradients + weight_gradients


def _halves(a, m):
    """The upper and lower 32 bits of ``a m`` by products of 16-bit parts."""
    a1, a0, m1, m0 = a >> 16, a & 0xFFFF, m >> 16, m & 0xFFFF
    low, middle = a0 * m0, a1 * m0 + (a0 * m0 >> 16)
    other = a0 * m1 + (middle & 0xFFFF)
    return a1 * m1 + (middle >> 16) + (other >> 16), (other & 0xFFFF) << 16 | low & 0xFFFF


def _kept(index, p, seed, offset):
    """Whether the elements with these mask indices stay: each one's own word, from its own counter."""
    counter = [(index // 4) % 2**32, (index // 4) // 2**32, offset % 2**32, offset // 2**32 % 2**32]
    counter = [torch.as_tensor(c, device="cuda") + torch.zeros_like(index) for c in counter]
    for r in range(10):
        key = [((seed >> 32 * i) + r * bump) % 2**32 for i, bump in enumerate((0x9E3779B9, 0xBB67AE85))]
        high_a, low_a = _halves(counter[0], 0xD2511F53)
        high_b, low_b = _halves(counter[2], 0xCD9E8D57)
        counter = [high_b ^ counter[1] ^ key[0], low_b, high_a ^ counter[3] ^ key[1], low_a]
    word = torch.stack(counter).gather(0, (index % 4)[None])[0]
    return word >= int(p * 2**32 + 0.5)


def _dropout_exact(case, state):
    shape, shared = _numbers(case["shape"]), case["shared"]
    x, dout = state["x"].reshape(-1), state["dout"].reshape(-1)
    residual = None if state["residual"] is None else state["residual"].reshape(-1)
    out = torch.empty(x.numel(), dtype=torch.float64, device="cuda")
    dx = torch.empty_like(out)
    inner = math.prod(shape[shared + 1:]) if shared >= 0 else 1
    size = shape[shared] if shared >= 0 else 1
    for first in range(0, x.numel(), 1 << 24):
        part = slice(first, min(first + (1 << 24), x.numel()))
        index = torch.arange(part.start, part.stop, device="cuda")
        if shared >= 0:  # the index without the shared axis
            index = index // (inner * size) * inner + index % inner
        kept = _kept(index, case["p"], state["seed"], state["offset"]).double()
        out[part] = kept * x[part].double() / (1.0 - case["p"])
        if residual is not None:
            out[part] += residual[part].double()
        dx[part] = kept * dout[part].double() / (1.0 - case["p"])
    return [out.view(shape), dx.view(shape)]


def exact(case, seed):
    global own
    held, own = own, False  # the inputs alone are wanted
    try:
        state = prepare(case, seed)
    finally:
        own = held
    return _dropout_exact(case, state) if case["op"] == "dropout" else _heads_exact(case, state)


def work(case):
    """Bytes and operations one pass cannot do without. A training pass reads its input in the forward pass
    and again (q and k, or nothing where the rotation or the mask alone is undone) in the backward pass: the
    two lie a whole model apart."""
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "dropout":
        n = math.prod(_numbers(case["shape"]))
        out = {"none": size, "bf16": 2, "fp32": 4}[case["residual"]]
        residual = 0 if case["residual"] == "none" else out
        # the generator's ten rounds of two products, four exclusive ors and two additions, for four elements
        masks = n // _numbers(case["shape"])[case["shared"]] if case["shared"] >= 0 else n
        return {"bytes": n * (size + residual + out) + n * (out + size), "flops": 5 * n + 2 * 20 * masks}
    tokens, heads, d = case["b"] * case["t"], case["hq"] + case["hk"], case["d"]
    n = tokens * heads * d
    norm, train = case["op"] == "qk_norm_rotary", case["step"] == "train"
    width = 4 if case["places"] == "points" else 8
    places = width * len(_numbers(case["widths"])) * (case["t"] if case["places"] == "grid" else tokens)
    passes = 2 + ((3 if norm else 2) if train else 0)
    weights = (8 * d * (3 if train else 1)) if norm else 0
    return {"bytes": n * size * passes + places * (2 if train else 1) + weights,
            "flops": n * ((7 if norm else 3) + ((14 if norm else 3) if train else 0))}
