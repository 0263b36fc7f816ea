"""Log probabilities of given tokens, with the rows' entropy and top alternatives.

For a row of logits x over V words and a temperature T, z = x / T and p = softmax(z):

  logprobs       log p at the row's target token (0 where it is ``ignore_index``)
  entropy        -sum p log p, in nats
  top_logprobs   log p of the ``top`` most likely words, largest first; ``top_indices`` their
                 numbers (equal logits in the order of their numbers)

``token_logprobs`` takes logits, ``chunked_linear_token_logprobs`` the hidden rows and the
readout's weight and bias, whose logits [N, V] never exist at once (chunks as in
``chunked_linear_cross_entropy``). Both are differentiable in their float inputs, through the log
probabilities, the entropy and the alternatives' log probabilities: a policy gradient with an
entropy bonus needs the first two, and a teacher's alternatives are what ``distill`` learns from.

Words whose logit is -inf, or as low as masks set it (-1e9, the type's lowest value), have
probability 0 and take no part. A row of -inf only has log probabilities -inf, entropy 0, its first words as
alternatives and no gradient. A row with a NaN or +inf gives NaN. One kernel reads the logits
once (and the few vectors that hold an alternative again); sums are fp32, joined in 64 bits.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch import Tensor

from . import _lib
from .kernels import ops, vocab


class TokenLogprobs(NamedTuple):
    """Results of ``token_logprobs``; fields that were not asked for are None."""

    logprobs: Optional[Tensor]
    entropy: Tensor
    top_logprobs: Optional[Tensor]
    top_indices: Optional[Tensor]


_WHAT = "token log probabilities"


def _outputs(rows: int, top: int, device, targets: bool, stats: bool):
    ent = torch.empty(rows, device=device, dtype=torch.float32)
    lp = torch.empty_like(ent) if targets else None
    st = ent.new_empty((rows, 2)) if stats else None
    tl = ent.new_empty((rows, top)) if top else None
    ti = ent.new_empty((rows, top), dtype=torch.int64) if top else None
    return lp, ent, st, tl, ti


def _forward(x, bias, targets, ignore, temperature, top, outs, s, word, stream):
    lp, ent, st, tl, ti = outs
    rows, V = x.shape
    tk = ops.KernelTimer.begin("token_logprobs", x)
    _lib.check(_lib.load().dabsn_hip_token_logprobs(
        ops._code(x.dtype), rows, V, x.data_ptr(), vocab.row_stride(x), ops._p(bias),
        vocab.at(targets, s), ignore, temperature, top, vocab.at(lp, s), vocab.at(ent, s),
        vocab.at(st, s), vocab.at(tl, s), vocab.at(ti, s), word.word.data_ptr(), stream), _WHAT)
    ops.KernelTimer.end(tk)


def _backward(x, bias, targets, ignore, temperature, top, saved, grads, s, out, ldo, plane):
    st, ent, ti = saved
    gl, ge, gt = grads
    rows, V = x.shape
    tk = ops.KernelTimer.begin("token_logprobs_bwd", x)
    _lib.check(_lib.load().dabsn_hip_token_logprobs_bwd(
        ops._code(x.dtype), rows, V, x.data_ptr(), vocab.row_stride(x), ops._p(bias),
        vocab.at(targets, s), ignore, temperature, top, vocab.at(ti, s), vocab.at(st, s),
        vocab.at(ent, s), vocab.at(gl, s), vocab.at(ge, s), vocab.at(gt, s), out, ldo, plane,
        vocab.stream(x)), _WHAT + " backward")
    ops.KernelTimer.end(tk)


def _from_logits(x, targets, ignore, temperature, top, stats):
    word = vocab.ErrorWord(x.device)
    outs = _outputs(x.shape[0], top, x.device, targets is not None, stats)
    _forward(x, None, targets, ignore, temperature, top, outs, 0, word, vocab.stream(x))
    word.check(_WHAT)
    return outs


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, targets, ignore, temperature, top):
        with vocab.on(x):
            lp, ent, st, tl, ti = _from_logits(x, targets, ignore, temperature, top, True)
        ctx.save_for_backward(x, targets, st, ent, ti)
        ctx.args = ignore, temperature, top
        ctx.set_materialize_grads(False)
        if ti is not None:
            ctx.mark_non_differentiable(ti)
        return lp, ent, tl, ti

    @staticmethod
    @vocab.once
    def backward(ctx, gl, ge, gt, _):
        x, targets, st, ent, ti = ctx.saved_tensors
        grads = vocab.grads_of(gl), vocab.grads_of(ge), vocab.grads_of(gt)
        with vocab.on(x):
            out = x.new_empty(x.shape)
            _backward(x, None, targets, *ctx.args, (st, ent, ti), grads, 0, out.data_ptr(),
                      x.shape[1], 0)
        return out, None, None, None, None


class _LinearTokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, bias, targets, ignore, temperature, top, chunk, stats):
        n = int(hidden.shape[0])
        with vocab.on(hidden), vocab.no_autocast():
            r = vocab.Readout(hidden, weight, bias)
            word = vocab.ErrorWord(hidden.device)
            outs = _outputs(n, top, hidden.device, targets is not None, stats)
            stream = vocab.stream(hidden)
            for s in range(0, n, chunk):
                _forward(r.logits(s, min(n, s + chunk)), r.row_bias, targets, ignore, temperature,
                         top, outs, s, word, stream)
            word.check(_WHAT)
        lp, ent, st, tl, ti = outs
        ctx.save_for_backward(hidden, weight, bias, targets, st, ent, ti)
        ctx.args, ctx.chunk = (ignore, temperature, top), chunk
        ctx.set_materialize_grads(False)
        if ti is not None:
            ctx.mark_non_differentiable(ti)
        return lp, ent, tl, ti

    @staticmethod
    @vocab.once
    def backward(ctx, gl, ge, gt, _):
        hidden, weight, bias, targets, st, ent, ti = ctx.saved_tensors
        grads = vocab.grads_of(gl), vocab.grads_of(ge), vocab.grads_of(gt)
        with vocab.on(hidden), vocab.no_autocast():
            r = vocab.Readout(hidden, weight, bias)
            acc = vocab.ReadoutGrads(r, ctx.needs_input_grad[:3], ctx.chunk)
            for g0, g1 in acc.groups():
                acc.begin(g0, g1)
                for s in range(g0, g1, acc.chunk):
                    x = r.logits(s, min(g1, s + acc.chunk))
                    _backward(x, r.row_bias, targets, *ctx.args, (st, ent, ti), grads, s,
                              acc.rows(s), acc.ldo, acc.plane())
                    del x
                acc.end()
            gh, gw, gb = acc.results()
        to = lambda g, like: None if g is None else g.to(like.dtype)  # noqa: E731
        return (to(gh, hidden), to(gw, weight), to(gb, bias), None, None, None, None, None, None)


def _top(top: int, v: int) -> int:
    top = int(top)
    if not 0 <= top <= min(vocab.MAX_TOP, v):
        raise ValueError(f"{_WHAT}: top must lie in [0, {min(vocab.MAX_TOP, v)}], not {top}")
    return top


def _shaped(outs, shape, top) -> TokenLogprobs:
    lp, ent, tl, ti = outs
    if len(shape) == 1:
        return TokenLogprobs(lp, ent, tl, ti)
    view = lambda t, tail: None if t is None else t.view((*shape, *tail))  # noqa: E731
    return TokenLogprobs(view(lp, ()), view(ent, ()), view(tl, (top,)), view(ti, (top,)))


def token_logprobs(logits: Tensor, targets: Tensor | None = None, *, top: int = 0,
                   temperature: float = 1.0, ignore_index: int = -100) -> TokenLogprobs:
    """Log probabilities, entropy and alternatives (see the module's note) of ``logits``
    [..., V], float32 or bfloat16 of any row stride; ``targets`` [...] int64 or int32, or None
    for the entropy and alternatives alone. ``top`` is at most 128 and V. A target outside
    [0, V) other than ``ignore_index`` gives NaN and sets the error word that
    ``kernels.check_errors()`` raises (``DABSN_HIP_ERROR_CHECK=sync``: raised here). The
    gradient has the logits' type, one rounding."""
    vocab.need_float(_WHAT, "logits", logits)
    if logits.dim() < 1:
        raise ValueError(f"{_WHAT}: expected logits [..., V]")
    shape, v = logits.shape[:-1], vocab.need_vocab(_WHAT, int(logits.shape[-1]))
    top, t = _top(top, v), vocab.need_temperature(_WHAT, temperature)
    if targets is not None:
        targets = vocab.need_tokens(_WHAT, "targets", targets, shape)
    vocab.need_device(_WHAT, logits, targets)
    x = vocab.rows_of(logits)
    if targets is not None and targets.dim() != 1:
        targets = targets.view(-1)
    if x.requires_grad and torch.is_grad_enabled():
        return _shaped(_TokenLogprobs.apply(x, targets, int(ignore_index), t, top), shape, top)
    with vocab.on(x):
        lp, ent, _, tl, ti = _from_logits(x, targets, int(ignore_index), t, top, False)
    return _shaped((lp, ent, tl, ti), shape, top)


def chunked_linear_token_logprobs(hidden: Tensor, weight: Tensor, bias: Tensor | None,
                                  targets: Tensor | None = None, *, top: int = 0,
                                  temperature: float = 1.0, ignore_index: int = -100,
                                  chunk_budget: int | None = None) -> TokenLogprobs:
    """``token_logprobs(F.linear(hidden, weight, bias), targets, ...)`` in chunks of
    ``chunk_budget // V`` rows (``DABSN_LOSS_CHUNK_SCORES``, default 2**25 elements), the logits
    in fp32 whatever the type of ``hidden`` [..., H]. The backward forms each chunk's logits
    again and adds the gradient products in fp32, rounded once to the inputs' types."""
    shape = hidden.shape[:-1]
    h, w, b = vocab.need_readout(_WHAT, hidden, weight, bias)
    v = int(w.shape[0])
    top, t = _top(top, v), vocab.need_temperature(_WHAT, temperature)
    if targets is not None:
        targets = vocab.need_tokens(_WHAT, "targets", targets, shape).view(-1)
    vocab.need_device(_WHAT, h, w, b, targets)
    stats = torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in (h, w, b))
    chunk = vocab.chunk_rows(int(h.shape[0]), v, chunk_budget)
    outs = _LinearTokenLogprobs.apply(h, w, b, targets, int(ignore_index), t, top, chunk, stats)
    return _shaped(outs, shape, top)
