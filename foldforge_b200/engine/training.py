"""Gradients of the engine ops on the ``b200`` backend.

An op's ``checkpoint`` says what its forward pass keeps for the backward pass, and with that whether the
op has one on b200 at all:

* ``None`` (the default): nothing. The op is inference-only; a call that needs a gradient is refused.
* ``"exact"``: its input as it is.
* ``"mxfp8"``: its input in 8 bits (33 bytes for 32 channels, :class:`foldforge_b200.kernels.Checkpoint8`).

``LayerNorm`` and ``Transition`` have gradients; :func:`set_checkpoint` sets them for a whole model. A
transition's forward pass runs the kernels it runs without gradients and gives the same output; its backward
pass computes the hidden activations again from the kept input, in bf16 with sums in fp32 (the ``pytorch``
backend holds them in fp32). ``LayerNorm``'s forward pass is a kernel of its own, which keeps the rows'
statistics: its output is the one without gradients but for the order of its sums. Only the gradients that
are asked for are formed.

A backward pass is not captured into a CUDA graph: autograd keeps a leaf's accumulation on the stream of
the graph that made it first, and capturing another while that one lives ends the process. A captured
training step calls the functions of :mod:`foldforge_b200.kernels` itself.
"""

from __future__ import annotations

import torch
from torch import nn
from torch.autograd.function import once_differentiable

Tensor = torch.Tensor
CHECKPOINTS = (None, "exact", "mxfp8")
#: rows of a transition's backward pass worked on at a time (its hidden activations are as many rows)
CHUNK_ROWS = 1 << 18


def check_name(name: str | None) -> str | None:
    if name not in CHECKPOINTS:
        raise ValueError(f"checkpoint must be one of {CHECKPOINTS}, got {name!r}")
    return name


def set_checkpoint(model: nn.Module, name: str | None) -> list[str]:
    """Set ``checkpoint`` on every op under ``model`` that has gradients on b200; their names."""
    check_name(name)
    found = [(path, m) for path, m in model.named_modules() if hasattr(m, "set_checkpoint")]
    for _, m in found:
        m.set_checkpoint(name)
    return [path for path, _ in found]


def needs_gradient(module: nn.Module, *inputs: Tensor) -> bool:
    return torch.is_grad_enabled() and (
        any(t.requires_grad for t in inputs) or any(p.requires_grad for p in module.parameters()))


def capture_reason() -> str | None:
    if torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing():
        return "autograd's backward pass is not captured into a CUDA graph"
    return None


def _refuse_capture() -> None:
    reason = capture_reason()
    if reason:
        raise RuntimeError(reason)


def _keep(ctx, kind: str, x: Tensor, kept=None) -> tuple[Tensor, ...]:
    """What goes into ``save_for_backward`` of an input."""
    from foldforge_b200 import kernels

    ctx.shape, ctx.dtype = x.shape, x.dtype
    if kind == "exact":
        return (x,)
    return (kernels.checkpoint_pack(x).data if kept is None else kept.data,)


def _kept(ctx, kind: str, saved: Tensor):
    from foldforge_b200 import kernels

    return saved if kind == "exact" else kernels.Checkpoint8(saved, ctx.shape, ctx.dtype)


def _norm_backward(dy: Tensor, saved, weight: Tensor | None, want_weight: bool, want_bias: bool, **kwargs):
    from foldforge_b200 import kernels

    if weight is not None and not want_weight:
        kwargs["weight_gradient"] = False
    return kernels.layer_norm_backward(dy, saved, weight, bias=want_bias, **kwargs)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x: Tensor, weight: Tensor | None, bias: Tensor | None, eps: float, kind: str) -> Tensor:
        from foldforge_b200 import kernels

        y, saved = kernels.layer_norm_train(x, weight, bias, eps, checkpoint=kind == "mxfp8")
        ctx.kind, ctx.has_bias = kind, bias is not None
        kept = _keep(ctx, kind, x, saved.x)
        ctx.save_for_backward(*kept, saved.stats, weight)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy: Tensor):
        from foldforge_b200 import kernels

        _refuse_capture()
        kept, stats, weight = ctx.saved_tensors
        saved = kernels.LayerNormSaved(_kept(ctx, ctx.kind, kept), stats)
        wanted = ctx.needs_input_grad
        dx, dweight, dbias = _norm_backward(dy, saved, weight, wanted[1], ctx.has_bias and wanted[2])
        return dx if wanted[0] else None, dweight, dbias, None, None


def layer_norm(x: Tensor, weight: Tensor | None, bias: Tensor | None, eps: float, kind: str) -> Tensor:
    return _LayerNorm.apply(x, weight, bias, eps, kind)


class _Transition(torch.autograd.Function):
    """``x + m W_sq(silu(W_a v) * W_b v)``, ``v = LN(x)``. Backward, with ``g`` the output's gradient:
    ``dh = m g W_sq``, the gate's gradient ``[da | db]`` (``ab`` computed again), ``dW_sq = (m g)^T h``,
    ``dW_a = da^T v``, ``dW_b = db^T v``, ``dv = da W_a + db W_b``, ``dx = g + LN'(dv)``."""

    @staticmethod
    def forward(ctx, x: Tensor, mask: Tensor | None, run, kind: str, eps: float, ln_weight: Tensor, ln_bias: Tensor,
                expand_a: Tensor, expand_b: Tensor, squeeze: Tensor) -> Tensor:
        out = run(x)
        ctx.kind, ctx.eps, ctx.masked = kind, eps, mask is not None
        kept = _keep(ctx, kind, x)
        ctx.save_for_backward(*kept, mask, ln_weight, ln_bias, expand_a, expand_b, squeeze)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, g: Tensor):
        from foldforge_b200 import kernels

        _refuse_capture()
        kept, mask, ln_weight, ln_bias, expand_a, expand_b, squeeze = ctx.saved_tensors
        c, h = squeeze.shape
        x = kernels.checkpoint_unpack(_kept(ctx, ctx.kind, kept)) if ctx.kind == "mxfp8" else kept
        x = x.reshape(-1, c)
        rows = x.shape[0]
        g = g.to(x.dtype).reshape(rows, c).contiguous()
        keep = None if mask is None else mask.reshape(rows, 1)
        expand = torch.cat([expand_a, expand_b]).to(x.dtype)  # [2 h, c]
        expand_t, squeeze_t = expand.t().contiguous(), squeeze.t().to(x.dtype).contiguous()
        # the gradients that are asked for; the norm's kernel forms dx with its sums over the rows
        want_x, want_ln_weight, want_ln_bias, want_a, want_b, want_squeeze = (ctx.needs_input_grad[i] for i in (0, 5, 6, 7, 8, 9))
        want_expand, want_norm = want_a or want_b, want_x or want_ln_weight or want_ln_bias
        dx: list[Tensor] = []
        sums: dict[str, Tensor] = {}

        def add(name: str, part: Tensor | None) -> None:
            if part is not None:
                sums[name] = sums[name].add_(part) if name in sums else part

        for first in range(0, rows, CHUNK_ROWS):
            part = slice(first, min(first + CHUNK_ROWS, rows))
            xp, gd = x[part], g[part]
            if keep is not None:  # rows without an update: whatever they hold stays out of every sum
                xp, gd = torch.where(keep[part], xp, 0.0), torch.where(keep[part], gd, 0.0)
            v, saved = kernels.layer_norm_train(xp, ln_weight, ln_bias, ctx.eps)
            ab = kernels.gemm_nt(v, expand)
            dab = kernels.swiglu_backward(kernels.gemm_nt(gd, squeeze_t), ab, output=want_squeeze)
            del ab
            if want_squeeze:
                dab, hidden = dab
                add("squeeze", kernels.weight_grad(gd, hidden))
                del hidden
            if want_expand:
                add("expand", kernels.weight_grad(dab, v))
            if want_norm:
                dxp, dln_weight, dln_bias = _norm_backward(kernels.gemm_nt(dab, expand_t), saved, ln_weight, want_ln_weight,
                                                           want_ln_bias, residual=g[part] if want_x else None)
                add("ln_weight", dln_weight)
                add("ln_bias", dln_bias)
                if want_x:
                    dx.append(dxp)
        if rows == 0:
            dx = [torch.empty_like(x)]
            sums = {name: torch.zeros_like(t, dtype=torch.float32) for name, t in
                    (("ln_weight", ln_weight), ("ln_bias", ln_bias), ("expand", expand), ("squeeze", squeeze))}
        all_dx = (dx[0] if len(dx) == 1 else torch.cat(dx)).view(ctx.shape) if want_x else None
        dexpand = sums.get("expand")
        return (all_dx, None, None, None, None, sums.get("ln_weight") if want_ln_weight else None,
                sums.get("ln_bias") if want_ln_bias else None, dexpand[:h] if want_a else None,
                dexpand[h:] if want_b else None, sums.get("squeeze") if want_squeeze else None)


def transition(x: Tensor, mask: Tensor | None, run, kind: str, eps: float, *weights: Tensor) -> Tensor:
    """``run(x)`` with a gradient. ``mask`` (bool, the shape of x without its channels): where the update is
    kept; ``weights``: LayerNorm weight and bias, expand_a, expand_b, squeeze."""
    return _Transition.apply(x, mask, run, kind, eps, *weights)
