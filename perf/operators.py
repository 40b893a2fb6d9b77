"""The training operators and their plain forms: what is timed and what it is compared with.

Four operators of a training step around the engine's norms and transitions:

* ``layer_norm``: LayerNorm forward and backward (dx, and the weight's and bias's gradients reduced
  over the rows), the backward pass reading either the input itself or its 8-bit checkpoint.
* ``checkpoint``: an activation quantised to 8 bits as it is kept (blocks of 32 channels, one
  power-of-two scale a block, e4m3 codes), and read back.
* ``weight_grad``: a linear layer's weight gradient dW = dY^T X over all rows, X as it is or kept in
  8 bits.
* ``swiglu``: the gated unit silu(a) b forward and backward, the backward pass reading the kept
  [a | b] as it is or in 8 bits.

Where ``own`` is false ``run`` computes the plain form from elementary torch operations in fp32;
where it is true it calls ``foldforge_b200.kernels``. ``exact`` is each operator's definition in
64 bits.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-5
BLOCK = 32  # channels that share a scale
LARGEST = 2**25  # elements of the largest activation listed (the pair tensor of 512 tokens)
LARGEST_PRODUCT = 2**34  # multiply-adds of the largest weight gradient listed


def listed():
    return [
        # one token's single row (c_s = 384): the smallest call, all latency
        {"name": "ln_one_row", "op": "layer_norm", "rows": 1, "c": 384, "dtype": "bf16", "kept": "exact"},
        # the pair norm of a 512-token crop, its input kept as it is
        {"name": "ln_pair_512", "op": "layer_norm", "rows": 512 * 512, "c": 128, "dtype": "bf16", "kept": "exact"},
        # the same with the input kept in 8 bits
        {"name": "ln_pair_512_mx", "op": "layer_norm", "rows": 512 * 512, "c": 128, "dtype": "bf16", "kept": "mxfp8"},
        # fp32 precision at an odd length and an odd width
        {"name": "ln_odd_fp32", "op": "layer_norm", "rows": 20011, "c": 197, "dtype": "fp32", "kept": "mxfp8"},
        # wide rows, a few thousand tokens
        {"name": "ln_wide", "op": "layer_norm", "rows": 4099, "c": 4096, "dtype": "bf16", "kept": "mxfp8"},
        # the single track of a short chain, fp32, a width that ends inside a block
        {"name": "checkpoint_small", "op": "checkpoint", "rows": 77, "c": 390, "dtype": "fp32"},
        # an MSA of 1024 rows x 512 columns, c_m = 64
        {"name": "checkpoint_msa", "op": "checkpoint", "rows": 1024 * 512, "c": 64, "dtype": "bf16"},
        # the single transition's expansion, 512 tokens, its input kept in 8 bits
        {"name": "wgrad_single_mx", "op": "weight_grad", "rows": 512, "n": 1536, "k": 384, "kept": "mxfp8"},
        # the pair transition's expansion, 512 tokens, its input kept in 8 bits
        {"name": "wgrad_pair_mx", "op": "weight_grad", "rows": 512 * 512, "n": 512, "k": 128, "kept": "mxfp8"},
        # a narrow head projection over the pair rows of 300 tokens, odd widths, bf16 input
        {"name": "wgrad_odd", "op": "weight_grad", "rows": 300 * 300, "n": 129, "k": 68, "kept": "exact"},
        # a single-track gate, 384 tokens, a hidden width of 2 x 384
        {"name": "swiglu_single", "op": "swiglu", "rows": 384, "h": 768, "dtype": "bf16", "kept": "exact"},
        # the pair transition's gate over the pair rows of 256 tokens, [a | b] kept in 8 bits
        {"name": "swiglu_pair_mx", "op": "swiglu", "rows": 256 * 256, "h": 512, "dtype": "bf16", "kept": "mxfp8"},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _width(rng, low, high):
    """A width spread over its logarithm: a multiple of 8 in two draws of three, else any number."""
    w = _spread(rng, low, high)
    return max(8, w // 8 * 8) if rng.random() < 2 / 3 else w


def draw(rng):
    op = rng.choice(["layer_norm", "layer_norm", "checkpoint", "weight_grad", "weight_grad", "swiglu"])
    case = {"op": op}
    if op == "weight_grad":
        n, k = _width(rng, 4, 2048), _width(rng, 4, 2048)
        most = min(LARGEST_PRODUCT // (n * k), LARGEST // max(n, k), 512 * 512)
        case.update(rows=_spread(rng, 1, most), n=n, k=k)
    elif op == "swiglu":
        h = _width(rng, 4, 4096)
        case.update(rows=_spread(rng, 1, LARGEST // h), h=h)
    else:
        c = _width(rng, 4, 8192)
        case.update(rows=_spread(rng, 1, LARGEST // c), c=c)
    if op != "weight_grad":
        case["dtype"] = rng.choice(["bf16", "bf16", "fp32"])
        if case["dtype"] == "fp32":
            case["rows"] = max(1, case["rows"] // 2)
    if op != "checkpoint":
        case["kept"] = rng.choice(["exact", "mxfp8"])
    return case


def _activation(gen, rows, c, dtype):
    """Rows as a residual stream holds them: channels of different spread, a few of them large, an offset."""
    spread = torch.exp(0.7 * torch.randn(c, device="cuda", generator=gen))
    offset = 0.3 * torch.randn(c, device="cuda", generator=gen)
    x = torch.randn(rows, c, device="cuda", generator=gen)
    return x.mul_(spread).add_(offset).to(dtype)


def _gradient(gen, rows, c, dtype):
    """A loss's gradient: small, its rows of different sizes."""
    size = 1e-3 * torch.exp(0.5 * torch.randn(rows, 1, device="cuda", generator=gen))
    return torch.randn(rows, c, device="cuda", generator=gen).mul_(size).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rows, op = case["rows"], case["op"]
    state = {"op": op, "kept": case.get("kept")}
    dtype = DTYPES[case.get("dtype", "bf16")]
    if op == "layer_norm":
        c = case["c"]
        state["x"] = _activation(gen, rows, c, dtype)
        state["dy"] = _gradient(gen, rows, c, dtype)
        state["weight"] = 1.0 + 0.2 * torch.randn(c, device="cuda", generator=gen)
        state["bias"] = 0.1 * torch.randn(c, device="cuda", generator=gen)
    elif op == "checkpoint":
        state["x"] = _activation(gen, rows, case["c"], dtype)
    elif op == "weight_grad":
        state["dy"] = _gradient(gen, rows, case["n"], dtype)
        x = _activation(gen, rows, case["k"], dtype)
        # in 8 bits, the backward pass has the checkpoint in hand that the forward pass left
        state["x"] = x if case["kept"] == "exact" else _keep(x)
    else:
        state["ab"] = _activation(gen, rows, 2 * case["h"], dtype)
        state["dh"] = _gradient(gen, rows, case["h"], dtype)
    return state


def _keep(x):
    """The 8-bit checkpoint a program holds: the library's own, or the plain form's (codes, scales)."""
    if own:
        from foldforge_b200 import kernels

        return kernels.checkpoint_pack(x)
    return _quantise(x)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# --------------------------------------------------------------------------- the framework's calls
def _run_own(state):
    from foldforge_b200 import kernels

    op = state["op"]
    if op == "layer_norm":
        y, saved = kernels.layer_norm_train(state["x"], state["weight"], state["bias"], EPS,
                                            checkpoint=state["kept"] == "mxfp8")
        dx, dweight, dbias = kernels.layer_norm_backward(state["dy"], saved, state["weight"])
        return [y, dx, dweight, dbias]
    if op == "checkpoint":
        return [kernels.checkpoint_unpack(kernels.checkpoint_pack(state["x"]))]
    if op == "weight_grad":
        return [kernels.weight_grad(state["dy"], state["x"])]
    h, saved = kernels.swiglu_train(state["ab"], checkpoint=state["kept"] == "mxfp8")
    return [h, kernels.swiglu_backward(state["dh"], saved)]


# --------------------------------------------------------------------------- the plain forms
def _quantise(x):
    """Codes and scales of ``x`` in blocks of 32 channels of a row: the scale is the smallest power of
    two that brings the block's largest finite value to at most 448 (e4m3's largest)."""
    rows, c = x.shape
    blocks = -(-c // BLOCK)
    v = torch.zeros(rows, blocks * BLOCK, device=x.device)
    v[:, :c] = x.float()
    v = v.view(rows, blocks, BLOCK)
    finite = torch.isfinite(v)
    largest = torch.where(finite, v.abs(), torch.zeros_like(v)).amax(-1, keepdim=True)
    mantissa, exponent = torch.frexp(largest)  # largest = mantissa 2^exponent, mantissa in [0.5, 1)
    exponent = exponent - 9 + (mantissa > 0.875).int()  # 448 = 0.875 2^9
    exponent = torch.where(largest > 0, exponent, torch.full_like(exponent, -127)).clamp_min(-127)
    codes = torch.where(finite, torch.ldexp(v, -exponent), torch.full_like(v, math.nan)).to(torch.float8_e4m3fn)
    return codes, exponent, c, x.dtype


def _values(kept):
    """The fp32 values a checkpoint stands for."""
    codes, exponent, c, _ = kept
    v = torch.ldexp(codes.float(), exponent)
    return v.reshape(v.shape[0], -1)[:, :c]


def _run_plain(state):
    op = state["op"]
    mx = state["kept"] == "mxfp8"
    if op == "layer_norm":
        x, dy, weight = state["x"], state["dy"], state["weight"]
        v = x.float()
        mean = v.mean(-1, keepdim=True)
        d = v - mean
        rstd = torch.rsqrt((d * d).mean(-1, keepdim=True) + EPS)
        y = (d * rstd * weight + state["bias"]).to(x.dtype)
        xhat = ((_values(_quantise(x)) if mx else v) - mean) * rstd
        g = dy.float()
        dweight, dbias = (g * xhat).sum(0), g.sum(0)
        g = g * weight
        dx = rstd * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
        return [y, dx.to(x.dtype), dweight, dbias]
    if op == "checkpoint":
        return [_values(_quantise(state["x"])).to(state["x"].dtype)]
    if op == "weight_grad":
        x = _values(state["x"]) if mx else state["x"].float()
        return [state["dy"].float().t() @ x]
    ab, dtype = state["ab"].float(), state["ab"].dtype
    half = ab.shape[-1] // 2
    a, b = ab[:, :half], ab[:, half:]
    h = (a / (1 + torch.exp(-a)) * b).to(dtype)
    if mx:
        ab = _values(_quantise(state["ab"]))
        a, b = ab[:, :half], ab[:, half:]
    s = 1 / (1 + torch.exp(-a))
    dh = state["dh"].float()
    da = dh * b * s * (1 + a * (1 - s))
    db = dh * a * s
    return [h, torch.cat([da, db], -1).to(dtype)]


# --------------------------------------------------------------------------- the definitions, in 64 bits
def _rounded(x):
    """What the 8-bit checkpoint makes of ``x``, by arithmetic on 64-bit values."""
    rows, c = x.shape
    out = torch.empty(rows, c, dtype=torch.float64, device=x.device)
    for first in range(0, c, BLOCK):
        block = x[:, first:first + BLOCK].double()
        top = block.abs().amax(1, keepdim=True)
        # the smallest power of two 2^e with top <= 448 2^e, at least 2^-127
        e = torch.ceil(torch.log2(top / 448)).nan_to_num(neginf=-127.0)
        e = torch.where(top > 448 * torch.exp2(e), e + 1, e)
        e = torch.where(top <= 448 * torch.exp2(e - 1), e - 1, e).clamp_min(-127)
        scaled = block / torch.exp2(e)
        # e4m3: steps of 2^(k - 3) in [2^k, 2^(k + 1)), of 2^-9 below 2^-6; ties to even
        k = torch.floor(torch.log2(scaled.abs().clamp_min(2.0**-6)))
        k = torch.where(scaled.abs() >= torch.exp2(k + 1), k + 1, k)
        step = torch.exp2(k.clamp_min(-6) - 3)
        out[:, first:first + BLOCK] = torch.round(scaled / step) * step * torch.exp2(e)
    return out


def _layer_norm_exact(x, dy, weight, bias, mx):
    v = x.double()
    c = v.shape[1]
    mean = v.sum(1, keepdim=True) / c
    sigma = ((v - mean).square().sum(1, keepdim=True) / c + EPS).sqrt()
    y = (v - mean) / sigma * weight + bias
    normal = ((_rounded(x) if mx else v) - mean) / sigma
    g = dy.double()
    gw = g * weight
    along = (gw * normal).sum(1, keepdim=True) / c
    dx = (gw - gw.sum(1, keepdim=True) / c - normal * along) / sigma
    return [y, dx, torch.einsum("rc,rc->c", g, normal), g.sum(0)]


def exact(case, seed):
    global own
    op, rows = case["op"], case["rows"]
    held, own = own, False  # the inputs alone are wanted, the plain checkpoint's codes with them
    try:
        state = prepare(dict(case, kept="exact"), seed)
    finally:
        own = held
    mx = case.get("kept") == "mxfp8"
    if op == "layer_norm":
        return _layer_norm_exact(state["x"], state["dy"], state["weight"].double(), state["bias"].double(), mx)
    if op == "checkpoint":
        return [_rounded(state["x"])]
    if op == "weight_grad":
        n, k = case["n"], case["k"]
        total = torch.zeros(n, k, dtype=torch.float64, device="cuda")
        for first in range(0, rows, 1 << 15):
            x = state["x"][first:first + (1 << 15)]
            total += state["dy"][first:first + (1 << 15)].double().t() @ (_rounded(x) if mx else x.double())
        return [total]
    half = case["h"]
    ab = state["ab"].double()
    h = ab[:, :half] * torch.sigmoid(ab[:, :half]) * ab[:, half:]
    if mx:
        ab = _rounded(state["ab"])
    a, b = ab[:, :half], ab[:, half:]
    dh = state["dh"].double()
    s = torch.sigmoid(a)
    return [h, torch.cat([dh * b * (s + a * s * torch.sigmoid(-a)), dh * a * s], 1)]


def work(case):
    """Bytes and operations one pass cannot do without. A training pass reads its input in the forward
    pass and what is kept of it in the backward pass: the two lie a whole model apart."""
    rows, op = case["rows"], case["op"]
    size = 4 if case.get("dtype") == "fp32" else 2

    def kept_bytes(c):
        return rows * (c + -(-c // BLOCK))

    mx = case.get("kept") == "mxfp8"
    if op == "layer_norm":
        c = case["c"]
        forward = rows * c * 2 * size + rows * 8 + (kept_bytes(c) if mx else 0)
        backward = rows * c * 2 * size + rows * 8 + (kept_bytes(c) if mx else rows * c * size)
        return {"bytes": forward + backward + 20 * c, "flops": rows * c * 22}
    if op == "checkpoint":
        c = case["c"]
        return {"bytes": 2 * rows * c * size + 2 * kept_bytes(c), "flops": rows * c * 4}
    if op == "weight_grad":
        n, k = case["n"], case["k"]
        return {"bytes": rows * n * 2 + (kept_bytes(k) if mx else rows * k * 2) + n * k * 4, "flops": 2 * rows * n * k}
    h = case["h"]
    forward = rows * 3 * h * size + (kept_bytes(2 * h) if mx else 0)
    backward = rows * 3 * h * size + (kept_bytes(2 * h) if mx else rows * 2 * h * size)
    return {"bytes": forward + backward, "flops": rows * h * 24}
