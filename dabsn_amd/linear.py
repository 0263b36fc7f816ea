"""Linear layers whose bias, activation and residual are the product's epilogue, and the block's
MLP made of them.

  fused_linear  activation(x W^T + bias) + residual
  fused_mlp     x + activation(norm(x) W1^T + b1) W2^T + b2

Activations: ``none``, ``relu2`` (the squared ReLU of the reference's MLP), ``gelu`` (by the error
function) and ``silu``. (A plain ReLU is left out: its slope jumps at 0, so products of 16-bit
operands would differ by whole terms.) Products are fp32 sums; everything up to the result is fp32
and is rounded once. Both are differentiable in all their tensors. In the backward the products'
operands have the inputs' type: dz = g activation'(z) is rounded once to it. The slope is kept in
fp32, or with bfloat16 in 16 bits (2^-11 of itself or 2^-39 off); the squared ReLU's is 2 sqrt of its
output, which is kept itself.
"""

from __future__ import annotations

import torch
from torch import Tensor

from .kernels import dense
from .norm import layer_norm, rms_norm

_RELU2 = dense.ACTIVATIONS["relu2"]


def _cast(*tensors: Tensor | None):
    """All tensors in autocast's type, as ``F.linear`` casts its own."""
    dt = torch.get_autocast_dtype("cuda")
    return tuple(None if t is None else t.to(dt) for t in tensors)


def _weight(what: str, name: str, w: Tensor, x: Tensor, width: int) -> Tensor:
    if w.dim() != 2 or w.shape[1] != width or 0 in w.shape:
        raise ValueError(f"{what}: {name} {tuple(w.shape)} does not match width {width}")
    if w.shape[0] > dense.MOST or width > dense.MOST:
        raise ValueError(f"{what}: {name} {tuple(w.shape)} has over {dense.MOST} rows or columns")
    if w.dtype != x.dtype:
        raise TypeError(f"{what}: {name} must be {x.dtype} as x is, not {w.dtype}")
    return dense.rows_of(w)


def _keeps(x: Tensor, n: int, act: int, residual: bool):
    """(buffer for what the slope is made of or None, its kind) of an activated product's forward in
    training. The squared ReLU's output is at hand where no residual is added to it."""
    if act == 0 or (act == _RELU2 and not residual):
        return None, dense.FROM_SQUARE if act else 0
    return dense.padded(x.shape[0], n, x), dense.FROM_SQUARE if act == _RELU2 else dense.STORED


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        with dense.on(x):
            keep, ctx.kind = _keeps(x, weight.shape[0], act, residual is not None)
            out = dense.product(x, weight, bias, act, keep, residual)
        ctx.save_for_backward(x, weight, out if ctx.kind and keep is None else keep)
        return out

    @staticmethod
    @dense.once
    def backward(ctx, g):
        x, weight, slope = ctx.saved_tensors
        need = ctx.needs_input_grad
        with dense.on(x):
            grads = dense.product_backward(x, weight, dense.rows_of(g), slope, ctx.kind, need)
        return (*grads, g if need[3] else None, None)


def fused_linear(x: Tensor, weight: Tensor, bias: Tensor | None = None, *,
                 activation: str = "none", residual: Tensor | None = None) -> Tensor:
    """``activation(x @ weight.T + bias) + residual`` (see the module's note) of ``x`` [..., K],
    ``weight`` [N, K], ``bias`` [N] and ``residual`` [..., N], all float32 or all bfloat16, of any
    row strides. Inside autocast the product runs in its type, and a residual of another type is
    added afterwards, as ``F.linear(...) + residual`` would."""
    what = "fused_linear"
    act = dense.need_activation(what, activation)
    autocast = torch.is_autocast_enabled("cuda")
    if autocast:
        x, weight, bias = _cast(x, weight, bias)
    dense.need_float(what, "x", x)
    if x.dim() < 1:
        raise ValueError(f"{what}: expected x [..., K]")
    w = _weight(what, "weight", weight, x, int(x.shape[-1]))
    n = int(w.shape[0])
    bias = dense.need_vector(what, "bias", bias, n, x.dtype)
    shape = (*x.shape[:-1], n)
    if residual is not None:
        if residual.shape != shape:
            raise ValueError(f"{what}: residual {tuple(residual.shape)} does not match {shape}")
        if residual.dtype != x.dtype:
            if not autocast:
                raise TypeError(f"{what}: residual must be {x.dtype} as x is, not {residual.dtype}")
            dense.need_float(what, "residual", residual)
    dense.need_device(what, x, w, bias, residual)
    if residual is not None and residual.dtype != x.dtype:
        return fused_linear(x, w, bias, activation=activation) + residual
    rows = dense.rows_of(x)
    res = None if residual is None else dense.rows_of(residual)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad
                                       for t in (rows, w, bias, res)):
        out = _Linear.apply(rows, w, bias, res, act)
    else:
        with dense.on(x):
            out = dense.product(rows, w, bias, act, None, res)
    return out if x.dim() == 2 else out.view(shape)


class _MLP(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, nw, nb, w1, b1, w2, b2, act, layer, eps):
        leaves = nw, nb, w1, b1, w2, b2
        with dense.on(x):
            out, saved = dense.mlp(x, leaves, act, layer, eps, True)
        ctx.save_for_backward(x, *leaves, saved)
        ctx.args = act, layer, eps
        return out

    @staticmethod
    @dense.once
    def backward(ctx, g):
        x, *leaves, saved = ctx.saved_tensors
        with dense.on(x):
            grads = dense.mlp_backward(x, leaves, saved, dense.rows_of(g).contiguous(), *ctx.args,
                                       ctx.needs_input_grad)
        return (*grads, None, None, None)


def fused_mlp(x: Tensor, w1: Tensor, w2: Tensor, b1: Tensor | None = None,
              b2: Tensor | None = None, *, norm: str = "rms", norm_weight: Tensor | None = None,
              norm_bias: Tensor | None = None, eps: float | None = None,
              activation: str = "relu2") -> Tensor:
    """``x + activation(norm(x) @ w1.T + b1) @ w2.T + b2`` (see the module's note) of ``x`` [..., H],
    ``w1`` [F, H], ``w2`` [H, F], ``b1`` [F] and ``b2`` [H], all float32 or all bfloat16. ``norm`` is
    ``rms`` or ``layer`` (``eps`` 1e-6 or 1e-5 unless given; weight and bias as ``layer_norm``
    takes them). Inside autocast the products run in its type, the norm and the sum in x's."""
    what = "fused_mlp"
    act = dense.need_activation(what, activation)
    if norm not in ("rms", "layer"):
        raise ValueError(f"{what}: norm must be rms or layer, not {norm!r}")
    layer = norm == "layer"
    if norm_bias is not None and not layer:
        raise ValueError(f"{what}: the RMS norm has no bias")
    eps = dense.need_eps(what, (1e-5 if layer else 1e-6) if eps is None else eps)
    if torch.is_autocast_enabled("cuda"):
        w1, w2, b1, b2 = _cast(w1, w2, b1, b2)
        if x.dtype != w1.dtype:
            if w2.dim() == 2 and w2.shape[:1] != x.shape[-1:]:
                raise ValueError(f"{what}: w2 {tuple(w2.shape)} does not lead back to x {tuple(x.shape)}")
            normed = (layer_norm(x, norm_weight, norm_bias, eps=eps) if layer
                      else rms_norm(x, norm_weight, eps=eps))
            return fused_linear(fused_linear(normed, w1, b1, activation=activation), w2, b2,
                                residual=x)
    nw, nb = dense.need_norm(what, x, norm_weight, norm_bias)
    h = int(x.shape[-1])
    w1 = _weight(what, "w1", w1, x, h)
    w2 = _weight(what, "w2", w2, x, int(w1.shape[0]))
    if w2.shape[0] != h:
        raise ValueError(f"{what}: w2 {tuple(w2.shape)} does not lead back to width {h}")
    b1 = dense.need_vector(what, "b1", b1, int(w1.shape[0]), x.dtype)
    b2 = dense.need_vector(what, "b2", b2, h, x.dtype)
    dense.need_device(what, x, w1, w2, b1, b2, nw, nb)
    rows = dense.rows_of(x)
    leaves = (rows, nw, nb, w1, b1, w2, b2)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in leaves):
        out = _MLP.apply(*leaves, act, layer, eps)
    else:
        with dense.on(x):
            out, _ = dense.mlp(rows, leaves[1:], act, layer, eps, False)
    return out if x.dim() == 2 else out.view(x.shape)
