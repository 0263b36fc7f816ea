"""Distillation from a teacher's top logits.

A teacher's scoring pass leaves K tokens a row with their logits t_k (``token_logprobs`` with
``top=K``: log probabilities serve as logits). With u = t / T at temperature T and the student's
p = softmax(x / T), a row's loss is T^2 KL(q || p):

  teacher_lse None   q = softmax(u) over the row's listed tokens
  teacher_lse given  q_k = exp(u_k - teacher_lse), teacher_lse = the log-sum-exp of the teacher's
                     whole row / T (0 where the values are log probabilities at T = 1), and all
                     other tokens together are one event with q_r = 1 - sum q against the
                     student's mass on them, so that a list that leaves much out is not taken for
                     the whole

and the result the mean over the rows that have a listed token. The factor T^2 keeps the
gradient's size as T grows. Entries whose token is ``ignore_index`` or whose value is -inf are
absent, so rows of different lists, and padding rows, share one array; a token listed twice
counts with both weights. The student may rule words out with -inf; the rest is left out where
the student has no word for it, and a listed word with probability 0 makes the loss inf.

``distillation_from_logits`` takes the student's logits, ``chunked_linear_distillation`` the hidden
rows and the readout's weight and bias, whose logits [N, V] never exist at once.
"""

from __future__ import annotations

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _lib
from .kernels import ops, vocab
from .scoring import _at

_WHAT = "distillation"


def _rows(x, bias, values, tokens, lse, ignore, t, s, loss, coef, weights, scale, out, ldo, plane,
          word):
    rows, V = x.shape
    tk = ops.KernelTimer.begin("distill", x)
    _lib.check(_lib.load().dabsn_hip_distill(
        ops._code(x.dtype), rows, V, x.data_ptr(), vocab.row_stride(x), ops._p(bias),
        tokens.shape[1], ops._code(values.dtype), _at(values, s), _at(tokens, s), ignore, t,
        _at(lse, s), _at(loss, s), _at(coef, s), _at(weights, s), ops._p(scale), out, ldo, plane,
        word.word.data_ptr(), ops._stream(x)), _WHAT)
    ops.KernelTimer.end(tk)


def _mean(loss: Tensor, t: float) -> tuple[Tensor, Tensor]:
    """(mean loss, T / counted rows) of the rows' losses."""
    mean = torch.empty((), device=loss.device, dtype=torch.float32)
    factor = torch.empty((), device=loss.device, dtype=torch.float32)
    _lib.check(_lib.load().dabsn_hip_distill_mean(
        loss.shape[0], loss.data_ptr(), t, mean.data_ptr(), factor.data_ptr(), ops._stream(loss)),
        _WHAT)
    return mean, factor


class _FromLogits(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, values, tokens, lse, ignore, t):
        n, f32 = int(x.shape[0]), torch.float32
        need = ctx.needs_input_grad[0]
        with vocab.on(x):
            word = vocab.ErrorWord(x.device)
            loss = torch.empty((n, 2), device=x.device, dtype=f32)
            coef = torch.empty((n, 4), device=x.device, dtype=f32) if need else None
            weights = torch.empty(tokens.shape, device=x.device, dtype=f32) if need else None
            _rows(x, None, values, tokens, lse, ignore, t, 0, loss, coef, weights, None, None, 0, 0,
                  word)
            word.check(_WHAT)
            mean, factor = _mean(loss, t)
        ctx.save_for_backward(x, tokens, coef, weights, factor)
        ctx.t = t
        return mean

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        x, tokens, coef, weights, factor = ctx.saved_tensors
        rows, V = x.shape
        g = g.to(torch.float32)
        with vocab.on(x):
            out = torch.empty(x.shape, device=x.device, dtype=x.dtype)
            tk = ops.KernelTimer.begin("distill_bwd", x)
            _lib.check(_lib.load().dabsn_hip_distill_bwd(
                ops._code(x.dtype), rows, V, x.data_ptr(), vocab.row_stride(x), tokens.shape[1],
                tokens.data_ptr(), ctx.t, coef.data_ptr(), weights.data_ptr(),
                factor.data_ptr(), g.data_ptr(), out.data_ptr(), ops._stream(x)),
                _WHAT + " backward")
            ops.KernelTimer.end(tk)
        return out, None, None, None, None, None


class _Linear(torch.autograd.Function):
    """The gradients are formed in the forward, chunk by chunk, while the logits are at hand (the
    factor 1 / counted rows is known from the lists), and held in fp32: the backward scales and
    rounds them. Forming the logits again there would be a fourth product beside the three."""

    @staticmethod
    def forward(ctx, hidden, weight, bias, values, tokens, lse, ignore, t, chunk):
        n, dev = int(hidden.shape[0]), hidden.device
        need = ctx.needs_input_grad[:3]
        lib = _lib.load()
        with vocab.on(hidden), torch.autocast("cuda", enabled=False):
            r = vocab.Readout(hidden, weight, bias)
            word = vocab.ErrorWord(dev)
            loss = torch.empty((n, 2), device=dev, dtype=torch.float32)
            if any(need):
                _lib.check(lib.dabsn_hip_distill_rows(
                    n, r.V, tokens.shape[1], ops._code(values.dtype), values.data_ptr(),
                    tokens.data_ptr(), ignore, loss.data_ptr(), ops._stream(hidden)), _WHAT)
                _, scale = _mean(loss, t)
                acc = vocab.ReadoutGrads(r, need, chunk)
                for g0, g1 in acc.groups():
                    acc.begin(g0, g1)
                    for s in range(g0, g1, acc.chunk):
                        x = r.logits(s, min(g1, s + acc.chunk))
                        _rows(x, r.row_bias, values, tokens, lse, ignore, t, s, loss, None, None,
                              scale, *acc.rows(s), word)
                        del x
                    acc.end()
                ctx.save_for_backward(*acc.results())
            else:
                for s in range(0, n, chunk):
                    _rows(r.logits(s, min(n, s + chunk)), r.row_bias, values, tokens, lse, ignore, t,
                          s, loss, None, None, None, None, 0, 0, word)
            word.check(_WHAT)
            mean, _ = _mean(loss, t)
        ctx.dtype = hidden.dtype
        return mean

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        g = g.to(torch.float32)
        with vocab.on(g):
            grads = [vocab.scaled(x, g, ctx.dtype) for x in ctx.saved_tensors]
        return (*grads, None, None, None, None, None, None)


def _lists(shape, v: int, top_logits: Tensor, top_indices: Tensor, teacher_lse: Tensor | None):
    """The teacher's arrays as the kernels read them."""
    vocab.need_float(_WHAT, "top_logits", top_logits)
    if top_indices.dim() != len(shape) + 1 or tuple(top_indices.shape[:-1]) != tuple(shape):
        raise ValueError(f"{_WHAT}: top_indices {tuple(top_indices.shape)} does not match rows "
                         f"{tuple(shape)}")
    if top_logits.shape != top_indices.shape:
        raise ValueError(f"{_WHAT}: top_logits {tuple(top_logits.shape)} and top_indices "
                         f"{tuple(top_indices.shape)} do not match")
    k = int(top_indices.shape[-1])
    if not 1 <= k <= vocab.MAX_TOP:
        raise ValueError(f"{_WHAT}: 1 to {vocab.MAX_TOP} listed tokens a row, not {k}")
    tokens = vocab.need_tokens(_WHAT, "top_indices", top_indices, top_indices.shape).view(-1, k)
    values = top_logits.detach().reshape(-1, k).contiguous()
    lse = None
    if teacher_lse is not None:
        if v > vocab.MAX_REST_VOCAB:
            raise ValueError(f"{_WHAT}: teacher_lse goes with at most {vocab.MAX_REST_VOCAB} words")
        if tuple(teacher_lse.shape) != tuple(shape):
            raise ValueError(f"{_WHAT}: teacher_lse {tuple(teacher_lse.shape)} does not match rows "
                             f"{tuple(shape)}")
        if not teacher_lse.is_floating_point():
            raise TypeError(f"{_WHAT}: teacher_lse must be a float tensor")
        lse = teacher_lse.detach().to(torch.float32).reshape(-1).contiguous()
    return values, tokens, lse


def distillation_from_logits(logits: Tensor, top_logits: Tensor, top_indices: Tensor, *,
                             temperature: float = 1.0, teacher_lse: Tensor | None = None,
                             ignore_index: int = -100) -> Tensor:
    """Mean distillation loss (fp32 scalar; see the module's note) of the student's ``logits``
    [..., V], float32 or bfloat16 of any row stride, against the teacher's ``top_logits`` and
    ``top_indices`` [..., K], 1 <= K <= 128, and ``teacher_lse`` [...]. The gradient has the
    logits' type, one rounding; the teacher's arrays get none. A listed token outside [0, V)
    other than ``ignore_index`` makes the loss NaN and sets the error word that
    ``kernels.check_errors()`` raises (``DABSN_HIP_ERROR_CHECK=sync``: raised here)."""
    vocab.need_float(_WHAT, "logits", logits)
    if logits.dim() < 2:
        raise ValueError(f"{_WHAT}: expected logits [..., V] of one row or more")
    v = vocab.need_vocab(_WHAT, int(logits.shape[-1]))
    t = vocab.need_temperature(_WHAT, temperature)
    values, tokens, lse = _lists(logits.shape[:-1], v, top_logits, top_indices, teacher_lse)
    vocab.need_device(_WHAT, logits, values, tokens, lse)
    return _FromLogits.apply(vocab.rows_of(logits), values, tokens, lse, int(ignore_index), t)


def chunked_linear_distillation(hidden: Tensor, weight: Tensor, bias: Tensor | None,
                                top_logits: Tensor, top_indices: Tensor, *,
                                temperature: float = 1.0, teacher_lse: Tensor | None = None,
                                ignore_index: int = -100,
                                chunk_budget: int | None = None) -> Tensor:
    """``distillation_from_logits(F.linear(hidden, weight, bias), ...)`` in chunks of
    ``chunk_budget // V`` rows (``DABSN_LOSS_CHUNK_SCORES``, default 2**24 elements), the logits
    in fp32 whatever the type of ``hidden`` [..., H]. Where a gradient is needed it is formed
    with the loss, chunk by chunk, and held in fp32 until the backward, which scales it and
    rounds it once to the inputs' types."""
    shape = hidden.shape[:-1]
    h, w, b = vocab.need_readout(_WHAT, hidden, weight, bias)
    t = vocab.need_temperature(_WHAT, temperature)
    values, tokens, lse = _lists(shape, int(w.shape[0]), top_logits, top_indices, teacher_lse)
    vocab.need_device(_WHAT, h, w, b, values, tokens, lse)
    chunk = vocab.chunk_rows(int(h.shape[0]), int(w.shape[0]), chunk_budget)
    return _Linear.apply(h, w, b, values, tokens, lse, int(ignore_index), t, chunk)
