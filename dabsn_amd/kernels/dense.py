"""Calls of the norm and product kernels, shared by ``norm`` and ``linear``: argument checks,
types inside autocast, and the launches."""

from __future__ import annotations

import math

import torch
from torch import Tensor

from .. import _lib
from . import ops
from .vocab import need_device, need_float, on, row_stride, rows_of, stream  # noqa: F401

ACTIVATIONS = {"none": 0, "relu2": 1, "gelu": 2, "silu": 3}
MAX_WIDTH = 16384
_STORED, _FROM_SQUARE = 1, 2


def once(backward):
    """A Function's backward that refuses to be differentiated itself."""

    def run(ctx, *grads):
        if torch.is_grad_enabled():  # create_graph=True
            raise RuntimeError("DABSN HIP operators of the MLP have no second derivative: run the "
                               "backward without create_graph")
        return backward(ctx, *grads)

    return run


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
                  add: Tensor | None, dtype: torch.dtype, need_weight: bool, need_bias: bool):
    """(dx [+ add], dweight, dbias); ``dtype`` is that of weight and bias."""
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
        ops._p(weight), stats.data_ptr(), g.data_ptr(), row_stride(g), ops._p(add), dx.data_ptr(),
        ops._p(dw), ops._p(db), ops._p(ws), nbytes, stream(x)), "norm backward")
    ops.KernelTimer.end(tk)
    return dx, dw, db


def padded(rows: int, n: int, like: Tensor) -> Tensor:
    """Uninitialised [rows, n] of like's type whose rows start at 16-byte boundaries."""
    ld = -(-n // 8) * 8
    return like.new_empty((rows, ld))[:, :n]


def product(a: Tensor, b: Tensor, *, trans_a: bool = False, trans_b: bool = False,
            bias: Tensor | None = None, act: int = 0, keep: Tensor | None = None,
            slope: Tensor | None = None, slope_kind: int = 0, residual: Tensor | None = None,
            out: Tensor | None = None, pad_a: bool = False, pad_out: bool = False) -> Tensor:
    """act(a b^T + bias) * slope + residual (see ``dabsn_hip_linear``). a [M, K], or [K, M] with
    ``trans_a``; b [N, K], or [K, N] with ``trans_b``. ``pad_a``: a is a ``padded`` buffer that this
    module filled; ``pad_out``: out is to be one."""
    lib = _lib.load()
    k, m = a.shape if trans_a else a.shape[::-1]
    n = b.shape[1] if trans_b else b.shape[0]
    if out is None:
        out = padded(m, n, a) if pad_out else a.new_empty((m, n))
    p, ld = ops._p, lambda t: 0 if t is None else row_stride(t)  # noqa: E731
    call = _lib.LinearCall(
        ops._code(a.dtype), trans_a, trans_b, pad_a, False, pad_out, act, slope_kind, m, n, k,
        a.data_ptr(), b.data_ptr(), p(bias), p(slope), p(residual), row_stride(a), row_stride(b),
        ld(slope), ld(residual), row_stride(out), ld(keep), out.data_ptr(), p(keep))
    nbytes = lib.dabsn_hip_linear_workspace_bytes(call)
    if nbytes:
        ws = a.new_empty(nbytes, dtype=torch.uint8)
        call.workspace, call.workspace_bytes = ws.data_ptr(), nbytes
    tk = ops.KernelTimer.begin("linear", a)
    _lib.check(lib.dabsn_hip_linear(call, stream(a)), "linear")
    ops.KernelTimer.end(tk)
    return out


def slope_product(g: Tensor, slope: Tensor | None, slope_kind: int, need_rows: bool,
                  need_sums: bool) -> tuple[Tensor, Tensor | None]:
    """(g * slope, its column sums or None); g itself without a slope."""
    lib, (rows, n) = _lib.load(), g.shape
    code = ops._code(g.dtype)
    dz = padded(rows, n, g) if need_rows and slope is not None else None
    sums = g.new_empty(n) if need_sums else None
    if dz is None and sums is None:
        return g, None
    nbytes = lib.dabsn_hip_linear_slope_workspace_bytes(code, rows, n) if need_sums else 0
    ws = g.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    tk = ops.KernelTimer.begin("linear_slope", g)
    _lib.check(lib.dabsn_hip_linear_slope(
        code, rows, n, g.data_ptr(), row_stride(g), ops._p(slope),
        0 if slope is None else row_stride(slope), slope_kind, ops._p(dz),
        0 if dz is None else row_stride(dz), ops._p(sums), ops._p(ws), nbytes, stream(g)),
        "linear slope")
    ops.KernelTimer.end(tk)
    return g if dz is None else dz, sums
