"""Layer norm and RMS norm of rows.

With mean and variance over the last axis,

  layer_norm   (x - mean) / sqrt(var + eps) * weight + bias
  rms_norm     x / sqrt(mean(x^2) + eps) * weight

in fp32 from one reading of the row, rounded once to x's type (``ops.rms_norm``, the block's
inference kernel, rounds before the weight as the reference's module does). The squares are summed as
they are: values up to 1e17 fit at any width, and those below 1e-18 count as 0 beside eps. Both are
differentiable in x, weight and bias: the gradients of weight and bias are sums over the rows in
fp32 and in a fixed order, so the same inputs give the same bits.
"""

from __future__ import annotations

import torch
from torch import Tensor

from .kernels import dense


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, layer):
        with dense.on(x):
            out, stats = dense.norm(x, weight, bias, eps, layer, True)
        ctx.save_for_backward(x, weight, stats)
        ctx.layer = layer
        ctx.dtype = x.dtype if bias is None else bias.dtype
        return out

    @staticmethod
    @dense.once
    def backward(ctx, g):
        x, weight, stats = ctx.saved_tensors
        need = ctx.needs_input_grad
        with dense.on(x):
            dx, dw, db = dense.norm_backward(x, weight, stats, dense.rows_of(g), ctx.layer,
                                             ctx.dtype if weight is None else weight.dtype, need[1],
                                             need[2])
        return dx, dw, db, None, None


def _norm(what: str, x: Tensor, weight: Tensor | None, bias: Tensor | None, eps: float,
          layer: bool) -> Tensor:
    weight, bias = dense.need_norm(what, x, weight, bias)
    eps = dense.need_eps(what, eps)
    dense.need_device(what, x, weight, bias)
    rows = dense.rows_of(x)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        out = _Norm.apply(rows, weight, bias, eps, layer)
    else:
        with dense.on(x):
            out, _ = dense.norm(rows, weight, bias, eps, layer, False)
    return out if x.dim() == 2 else out.view(x.shape)


def layer_norm(x: Tensor, weight: Tensor | None = None, bias: Tensor | None = None, *,
               eps: float = 1e-5) -> Tensor:
    """Layer norm (see the module's note) of ``x`` [..., H], float32 or bfloat16 of any row stride,
    H at most 16384; ``weight`` and ``bias`` [H] of x's type or both float32."""
    return _norm("layer_norm", x, weight, bias, eps, True)


def rms_norm(x: Tensor, weight: Tensor | None = None, *, eps: float = 1e-6) -> Tensor:
    """RMS norm (see the module's note) of ``x`` [..., H], types and limits as ``layer_norm``'s."""
    return _norm("rms_norm", x, weight, None, eps, False)
