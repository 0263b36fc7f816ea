"""Scaled token embedding: ``scale * weight[ids]`` and the gradient of the table.

The gradient of a word's row is ``scale`` times the sum of its tokens' gradient rows, in token
order and in fp32, rounded once to the table's type: the same inputs give the same bits, and a
frequent word's sum of thousands of bf16 rows loses nothing on the way.
"""

from __future__ import annotations

import math

import torch
from torch import Tensor

from . import _lib
from .kernels import ops, vocab

_WHAT = "embedding"
_NO_PADDING = -1  # not a word


def _lookup(ids: Tensor, w: Tensor, scale: float) -> Tensor:
    (V, H), n = w.shape, ids.numel()
    with vocab.on(w):
        out = w.new_empty((*ids.shape, H))
        word = vocab.ErrorWord(w.device)
        tk = ops.KernelTimer.begin("embedding", w)
        _lib.check(_lib.load().dabsn_hip_embedding_fwd(
            ops._code(w.dtype), n, V, H, ids.data_ptr(), w.data_ptr(), vocab.row_stride(w), scale,
            out.data_ptr(), word.word.data_ptr(), vocab.stream(w)), _WHAT)
        ops.KernelTimer.end(tk)
        word.check(_WHAT)
    return out


class _ScaledEmbedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale, padding):
        ctx.save_for_backward(ids)
        ctx.args = tuple(weight.shape), weight.dtype, scale, padding
        return _lookup(ids, weight, scale)

    @staticmethod
    @vocab.once
    def backward(ctx, grad):
        (ids,) = ctx.saved_tensors
        (V, H), dtype, scale, padding = ctx.args
        g = (grad if grad.dtype == dtype else grad.to(dtype)).contiguous()
        n, lib = ids.numel(), _lib.load()
        with vocab.on(g):
            out = g.new_empty((V, H))
            nbytes = lib.dabsn_hip_embedding_workspace_bytes(n, V, H)
            ws = g.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
            tk = ops.KernelTimer.begin("embedding_bwd", g)
            _lib.check(lib.dabsn_hip_embedding_bwd(
                ops._code(dtype), n, V, H, ids.data_ptr(), padding, g.data_ptr(), scale,
                out.data_ptr(), ops._p(ws), nbytes, vocab.stream(g)), _WHAT + " backward")
            ops.KernelTimer.end(tk)
        return None, out, None, None


def scaled_embedding(ids: Tensor, weight: Tensor, *, scale: float = 1.0,
                     padding_idx: int | None = None) -> Tensor:
    """``scale * weight[ids]`` [..., H] for int64 or int32 ``ids`` [...] and ``weight`` [V, H],
    float32 or bfloat16 (the product in fp32, one rounding). The tokens of ``padding_idx`` give
    the table no gradient, as in ``nn.Embedding``. An id outside [0, V) gives a row of NaN, no
    gradient, and sets the error word that ``kernels.check_errors()`` raises
    (``DABSN_HIP_ERROR_CHECK=sync``: raised here)."""
    vocab.need_float(_WHAT, "weight", weight)
    if weight.dim() != 2 or weight.shape[1] == 0 or weight.shape[1] >= 1 << 24:
        raise ValueError(f"{_WHAT}: expected weight [V, H], got {tuple(weight.shape)}")
    v = vocab.need_vocab(_WHAT, int(weight.shape[0]))
    scale = float(scale)
    if not math.isfinite(scale):
        raise ValueError(f"{_WHAT}: scale must be finite, not {scale}")
    padding = _NO_PADDING
    if padding_idx is not None:
        padding = int(padding_idx) + (v if padding_idx < 0 else 0)
        if not 0 <= padding < v:
            raise ValueError(f"{_WHAT}: padding_idx {padding_idx} of {v} words")
    ids = vocab.need_tokens(_WHAT, "ids", ids, ids.shape)
    vocab.need_device(_WHAT, weight, ids)
    w = vocab.rows_of(weight)
    if w.requires_grad and torch.is_grad_enabled():
        return _ScaledEmbedding.apply(ids, w, scale, padding)
    return _lookup(ids, w, scale)
