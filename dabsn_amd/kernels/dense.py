"""Calls of the norm and product kernels, shared by ``norm`` and ``linear``: argument checks,
types inside autocast, and the launches."""

from __future__ import annotations

import math

import torch
from torch import Tensor

from .. import _lib
from . import ops, vocab
from .vocab import need_device, need_float, on, stream  # noqa: F401

ACTIVATIONS = {"none": 0, "relu2": 1, "gelu": 2, "silu": 3}
MAX_WIDTH = 16384  # of a norm's rows
MOST = 2 ** 21 - 8  # of a product's rows, and of the strides between them
STORED, FROM_SQUARE = 1, 2


def once(backward):
    """A Function's backward that refuses to be differentiated itself."""

    def run(ctx, *grads):
        if torch.is_grad_enabled():  # create_graph=True
            raise RuntimeError("DABSN HIP operators of the MLP have no second derivative: run the "
                               "backward without create_graph")
        return backward(ctx, *grads)

    return run


def rows_of(x: Tensor) -> Tensor:
    """x [..., K] as [rows, K] with unit column stride and a row stride that the products take."""
    x = vocab.rows_of(x)
    return x.contiguous() if row_stride(x) > MOST >= x.shape[1] else x


def row_stride(x: Tensor) -> int:
    """The row stride of ``rows_of``'s result (a lone row's stride says nothing)."""
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def need_activation(what: str, name: str) -> int:
    try:
        return ACTIVATIONS[name]
    except (KeyError, TypeError):
        raise ValueError(f"{what}: activation must be one of {', '.join(ACTIVATIONS)}, not "
                         f"{name!r}") from None


def need_eps(what: str, eps: float) -> float:
    eps = float(eps)
    if not 0.0 <= eps < math.inf:
        raise ValueError(f"{what}: eps must be finite and not negative, not {eps}")
    return eps


def need_vector(what: str, name: str, t: Tensor | None, n: int, *types: torch.dtype):
    """A vector [n] of one of the types (contiguous), or None."""
    if t is None:
        return None
    if tuple(t.shape) != (n,):
        raise ValueError(f"{what}: {name} {tuple(t.shape)} does not match width {n}")
    if t.dtype not in types:
        raise TypeError(f"{what}: {name} must be {' or '.join(str(x) for x in types)}, not {t.dtype}")
    return t if t.is_contiguous() else t.contiguous()


def need_norm(what: str, x: Tensor, weight: Tensor | None, bias: Tensor | None):
    """(weight, bias) for rows x [..., H]: x's type or float32, both the same."""
    need_float(what, "x", x)
    if x.dim() < 1 or not 0 < x.shape[-1] <= MAX_WIDTH:
        raise ValueError(f"{what}: expected x [..., H] with H in [1, {MAX_WIDTH}], got "
                         f"{tuple(x.shape)}")
    h = int(x.shape[-1])
    weight = need_vector(what, "weight", weight, h, x.dtype, torch.float32)
    types = (x.dtype, torch.float32) if weight is None else (weight.dtype,)
    return weight, need_vector(what, "bias", bias, h, *types)


def norm(x: Tensor, weight: Tensor | None, bias: Tensor | None, eps: float, layer: bool,
         keep: bool) -> tuple[Tensor, Tensor | None]:
    """(normed rows, their (mean, rstd)) of x [rows, H] as ``rows_of`` gives it."""
    rows, h = x.shape
    out = x.new_empty((rows, h))
    stats = x.new_empty((rows, 2), dtype=torch.float32) if keep else None
    w = weight if weight is not None else bias
    tk = ops.KernelTimer.begin("norm", x)
    _lib.check(_lib.load().dabsn_hip_norm_fwd(
        ops._code(x.dtype), ops._code(x.dtype if w is None else w.dtype), layer, rows, h,
        x.data_ptr(), row_stride(x), ops._p(weight), ops._p(bias), eps, out.data_ptr(),
        ops._p(stats), stream(x)), "norm")
    ops.KernelTimer.end(tk)
    return out, stats


def norm_backward(x: Tensor, weight: Tensor | None, stats: Tensor, g: Tensor, layer: bool,
                  dtype: torch.dtype, need_weight: bool, need_bias: bool):
    """(dx, dweight, dbias); ``dtype`` is that of weight and bias."""
    lib, (rows, h) = _lib.load(), x.shape
    dx = x.new_empty((rows, h))
    dw = x.new_empty(h, dtype=dtype) if need_weight else None
    db = x.new_empty(h, dtype=dtype) if need_bias else None
    nbytes = (lib.dabsn_hip_norm_workspace_bytes(ops._code(x.dtype), rows, h)
              if need_weight or need_bias else 0)
    ws = x.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    tk = ops.KernelTimer.begin("norm_bwd", x)
    _lib.check(lib.dabsn_hip_norm_bwd(
        ops._code(x.dtype), ops._code(dtype), layer, rows, h, x.data_ptr(), row_stride(x),
        ops._p(weight), stats.data_ptr(), g.data_ptr(), row_stride(g), None, dx.data_ptr(),
        ops._p(dw), ops._p(db), ops._p(ws), nbytes, stream(x)), "norm backward")
    ops.KernelTimer.end(tk)
    return dx, dw, db


def padded(rows: int, n: int, like: Tensor) -> Tensor:
    """Uninitialised [rows, n] of like's type whose rows start at 16-byte boundaries."""
    ld = -(-n // 8) * 8
    return like.new_empty((rows, ld))[:, :n]


def product(a: Tensor, b: Tensor, bias: Tensor | None = None, act: int = 0,
            keep: Tensor | None = None, residual: Tensor | None = None) -> Tensor:
    """act(a b^T + bias) + residual (see ``dabsn_hip_linear``) of a [M, K] and b [N, K]."""
    lib, (m, k), n = _lib.load(), a.shape, b.shape[0]
    out = a.new_empty((m, n))
    p, ld = ops._p, lambda t: 0 if t is None else row_stride(t)  # noqa: E731
    call = _lib.LinearCall(
        ops._code(a.dtype), 0, 0, 0, 0, 0, act, 0, m, n, k, a.data_ptr(), b.data_ptr(), p(bias),
        None, p(residual), row_stride(a), row_stride(b), 0, ld(residual), n, ld(keep),
        out.data_ptr(), p(keep))
    nbytes = lib.dabsn_hip_linear_workspace_bytes(call)
    if nbytes:
        ws = a.new_empty(nbytes, dtype=torch.uint8)
        call.workspace, call.workspace_bytes = ws.data_ptr(), nbytes
    tk = ops.KernelTimer.begin("linear", a)
    _lib.check(lib.dabsn_hip_linear(call, stream(a)), "linear")
    ops.KernelTimer.end(tk)
    return out


def product_backward(x: Tensor, w: Tensor, g: Tensor, slope: Tensor | None, slope_kind: int, need):
    """Gradients (None where not needed) of x, w and bias from g [M, N] of ``product`` without
    residual; ``slope`` is what was kept."""
    lib, (m, k), n, p = _lib.load(), x.shape, w.shape[0], ops._p
    dx = x.new_empty((m, k)) if need[0] else None
    dw = x.new_empty((n, k)) if need[1] else None
    db = x.new_empty(n) if need[2] else None
    call = _lib.LinearGradsCall(
        ops._code(x.dtype), slope_kind, m, n, k, x.data_ptr(), w.data_ptr(), g.data_ptr(), p(slope),
        row_stride(x), row_stride(w), row_stride(g), 0 if slope is None else row_stride(slope),
        p(dx), p(dw), p(db))
    nbytes = lib.dabsn_hip_linear_grads_workspace_bytes(call)
    if nbytes:
        ws = x.new_empty(nbytes, dtype=torch.uint8)
        call.workspace, call.workspace_bytes = ws.data_ptr(), nbytes
    tk = ops.KernelTimer.begin("linear_bwd", x)
    _lib.check(lib.dabsn_hip_linear_grads(call, stream(x)), "linear backward")
    ops.KernelTimer.end(tk)
    return dx, dw, db


def mlp(x: Tensor, leaves, act: int, layer: bool, eps: float, train: bool):
    """(out, what the backward needs or None) of x [M, H] and leaves, norm weight and bias, w1, b1,
    w2, b2 (see ``dabsn_hip_mlp_fwd``)."""
    lib, out = _lib.load(), x.new_empty(x.shape)
    call = _mlp_call(x, leaves, act, layer, eps, train)
    call.out = out.data_ptr()
    _lib.check(lib.dabsn_hip_mlp_plan(call, 0), "mlp")
    saved = x.new_empty(call.saved_bytes, dtype=torch.uint8) if train else None
    call.saved = ops._p(saved)
    ws = x.new_empty(call.workspace_bytes, dtype=torch.uint8)
    call.workspace = ws.data_ptr()
    tk = ops.KernelTimer.begin("mlp", x)
    _lib.check(lib.dabsn_hip_mlp_fwd(call, stream(x)), "mlp")
    ops.KernelTimer.end(tk)
    return out, saved


def mlp_backward(x: Tensor, leaves, saved: Tensor, g: Tensor, act: int, layer: bool, eps: float, need):
    """Gradients (None where not needed) of x and the leaves from g [M, H], contiguous."""
    lib, p = _lib.load(), ops._p
    grads = [t.new_empty(t.shape) if n else None for t, n in zip((x, *leaves), need)]
    call = _mlp_call(x, leaves, act, layer, eps, True)
    call.grad, call.saved = g.data_ptr(), saved.data_ptr()
    (call.dx, call.dnorm_weight, call.dnorm_bias, call.dw1, call.db1, call.dw2,
     call.db2) = map(p, grads)
    _lib.check(lib.dabsn_hip_mlp_plan(call, 1), "mlp backward")
    ws = x.new_empty(call.workspace_bytes, dtype=torch.uint8)
    call.workspace = ws.data_ptr()
    tk = ops.KernelTimer.begin("mlp_bwd", x)
    _lib.check(lib.dabsn_hip_mlp_bwd(call, stream(x)), "mlp backward")
    ops.KernelTimer.end(tk)
    return grads


def _mlp_call(x, leaves, act, layer, eps, train) -> _lib.MlpCall:
    nw, nb, w1, b1, w2, b2 = leaves
    p, vector = ops._p, nw if nw is not None else nb if nb is not None else x
    return _lib.MlpCall(
        ops._code(x.dtype), ops._code(vector.dtype), layer, act, train, eps, x.shape[0], x.shape[1],
        w1.shape[0], x.data_ptr(), p(nw), p(nb), w1.data_ptr(), p(b1), w2.data_ptr(), p(b2), None,
        row_stride(x), row_stride(w1), row_stride(w2))
