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
counts with both weights. The student may rule words out with -inf or a large negative number; the
rest is left out where the student has no word for it (a mass off the list of 0 in 64 bits, below
e^-745), and a listed word with probability 0 makes the loss inf.

``distillation_from_logits`` takes the student's logits, ``chunked_linear_distillation`` the hidden
rows and the readout's weight and bias, whose logits [N, V] never exist at once.
"""

from __future__ import annotations

import math

import torch
from torch import Tensor

from . import _lib
from .kernels import ops, vocab

_WHAT = "distillation"


# From this many logits on, the gradient is formed with the loss while a row's logits are in
# registers, and the backward only checks that its upstream factor is 1 (loss.backward()); another
# factor forms it again (``loss_weight`` keeps a mixed objective's share out of it). Kernels of
# forward and backward with 32 listed tokens and the rest, in two passes -> with the gradient formed
# ahead (and again for another factor), us: 8388 x 32000 bf16 330 -> 230 (440), 16777 x 16000 343 -> 255
# (466), 4129 x 65000 309 -> 244 (461), 33554 x 8000 365 -> 329 (509), 2097 x 32000 fp32 159 -> 126 (235).
# Rows of few words are read again from the caches (33554 x 2000 bf16 208 -> 231), rows of more do not
# fit the registers (2684 x 100000 313 -> 308, and 490 for another factor), and below 2^24 logits the
# launches that count the rows ahead cost as much as the second reading.
_FUSED_LOGITS = 1 << 24
_FUSED_WORDS = (4096, 65536)


def _rows(x, bias, values, tokens, lse, ignore, t, s, loss, coef, weights, scale, split, out, ldo,
          word, stream):
    rows, V = x.shape
    tk = ops.KernelTimer.begin("distill", x)
    _lib.check(_lib.load().dabsn_hip_distill(
        ops._code(x.dtype), rows, V, x.data_ptr(), vocab.row_stride(x), ops._p(bias),
        tokens.shape[1], ops._code(values.dtype), vocab.at(values, s), vocab.at(tokens, s), ignore, t,
        vocab.at(lse, s), loss, coef, weights, scale, split, out, ldo, word.word.data_ptr(), stream),
        _WHAT)
    ops.KernelTimer.end(tk)


def _counted(values, tokens, ignore, V, loss, t, weight, factor, stream):
    """factor = weight T / counted rows, from the lists alone."""
    n, lib = tokens.shape[0], _lib.load()
    _lib.check(lib.dabsn_hip_distill_rows(n, V, tokens.shape[1], ops._code(values.dtype),
                                          values.data_ptr(), tokens.data_ptr(), ignore, loss, stream),
               _WHAT)
    _lib.check(lib.dabsn_hip_distill_mean(n, loss, t, weight, None, factor, stream), _WHAT)


class _FromLogits(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, values, tokens, lse, ignore, t, weight, train):
        (n, V), K, dev = x.shape, tokens.shape[1], x.device
        need, lib = train and ctx.needs_input_grad[0], _lib.load()
        fused = need and n * V >= _FUSED_LOGITS and _FUSED_WORDS[0] <= V <= _FUSED_WORDS[1]
        with vocab.on(x):
            stream = vocab.stream(x)
            word = vocab.ErrorWord(dev)
            # The rows' losses [n, 2], coefficients [n, 3], listed words' gradients [n, K], the factor.
            aux = torch.empty(n * (5 + K) + 1 if need else 2 * n, device=dev, dtype=torch.float32)
            mean = aux.new_empty(())
            loss = aux.data_ptr()
            coef = weights = factor = ready = None
            if need:
                coef, weights, factor = loss + 8 * n, loss + 20 * n, loss + 4 * n * (5 + K)
            if fused:
                _counted(values, tokens, ignore, V, loss, t, weight, factor, stream)
                ready = x.new_empty((n, V))
            _rows(x, None, values, tokens, lse, ignore, t, 0, loss, coef, weights, factor, 0,
                  None if ready is None else ready.data_ptr(), V, word, stream)
            _lib.check(lib.dabsn_hip_distill_mean(n, loss, t, weight, mean.data_ptr(),
                                                  None if fused else factor, stream), _WHAT)
            word.check(_WHAT)
        if need:
            ctx.save_for_backward(x, tokens, aux)
            ctx.t = t
            ctx.ready = ready
            ctx.captured = ready is not None and torch.cuda.is_current_stream_capturing()
        return mean

    @staticmethod
    @vocab.once
    def backward(ctx, g):
        x, tokens, aux = ctx.saved_tensors
        (n, V), K = x.shape, tokens.shape[1]
        if g.dtype != torch.float32:
            g = g.float()
        # The rows formed ahead serve one backward (the caller owns what it returns), of the same
        # graph if one is being captured.
        out, ctx.ready = ctx.ready, None
        if out is not None and ctx.captured != torch.cuda.is_current_stream_capturing():
            out = None
        done = out is not None
        with vocab.on(x):
            if out is None:
                out = x.new_empty((n, V))
            aux_p = aux.data_ptr()
            tk = ops.KernelTimer.begin("distill_bwd", x)
            _lib.check(_lib.load().dabsn_hip_distill_bwd(
                ops._code(x.dtype), n, V, x.data_ptr(), vocab.row_stride(x), K, tokens.data_ptr(),
                ctx.t, aux_p + 8 * n, aux_p + 20 * n, aux_p + 4 * n * (5 + K), g.data_ptr(), done,
                out.data_ptr(), vocab.stream(x)), _WHAT + " backward")
            ops.KernelTimer.end(tk)
        return out, None, None, None, None, None, None, None


class _Linear(torch.autograd.Function):
    """The gradients are formed in the forward, chunk by chunk, while the logits are at hand (the
    factor 1 / counted rows is known from the lists), and held in fp32: the backward scales and
    rounds them. Forming the logits again there would be a fourth product beside the three."""

    @staticmethod
    def forward(ctx, hidden, weight, bias, values, tokens, lse, ignore, t, share, chunk, train):
        n, dev = int(hidden.shape[0]), hidden.device
        # (Under no_grad needs_input_grad tells of a parameter all the same.)
        need = [train and x for x in ctx.needs_input_grad[:3]]
        with vocab.on(hidden), vocab.no_autocast():
            stream = vocab.stream(hidden)
            r = vocab.Readout(hidden, weight, bias)
            word = vocab.ErrorWord(dev)
            aux = torch.empty(2 * n + 1, device=dev, dtype=torch.float32)
            loss, factor = aux.data_ptr(), aux.data_ptr() + 8 * n
            mean = torch.empty((), device=dev, dtype=torch.float32)

            def rows(x, s, scale=None, split=0, inverse=None, out=None, ldo=0):
                _rows(x, r.row_bias, values, tokens, lse, ignore, t, s, loss + 8 * s, inverse, None,
                      scale, split, out, ldo, word, stream)

            if any(need):
                _counted(values, tokens, ignore, r.V, loss, t, share, factor, stream)
                acc = vocab.ReadoutGrads(r, need, chunk, split=True)
                for g0, g1 in acc.groups():
                    acc.begin(g0, g1)
                    for s in range(g0, g1, acc.chunk):
                        rows(r.logits(s, min(g1, s + acc.chunk)), s, factor, acc.split,
                             acc.inverses(s), acc.rows(s), acc.ldo)
                    acc.end()
                # Split rows lack the factor T / counted rows.
                own = aux[2 * n:] if r.half else None
                ctx.save_for_backward(*acc.results(), own, acc.scale)
            else:
                for s in range(0, n, chunk):
                    rows(r.logits(s, min(n, s + chunk)), s)
            word.check(_WHAT)
            _lib.check(_lib.load().dabsn_hip_distill_mean(n, loss, t, share, mean.data_ptr(), None,
                                                          stream), _WHAT)
        ctx.dtype = hidden.dtype
        return mean

    @staticmethod
    @vocab.once
    def backward(ctx, g):
        g = g.to(torch.float32)
        gh, gw, gb, own, scale = ctx.saved_tensors
        with vocab.on(g):
            grads = [vocab.scaled(x, ctx.dtype, g, own, s)
                     for x, s in ((gh, scale), (gw, None), (gb, None))]
        return (*grads, None, None, None, None, None, None, None, None)


def _share(weight: float) -> float:
    weight = float(weight)
    if not math.isfinite(weight):
        raise ValueError(f"{_WHAT}: loss_weight must be finite, not {weight}")
    return weight


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
                             ignore_index: int = -100, loss_weight: float = 1.0) -> Tensor:
    """``loss_weight`` times the mean distillation loss (fp32 scalar; see the module's note) of the
    student's ``logits`` [..., V], float32 or bfloat16 of any row stride, against the teacher's
    ``top_logits`` and ``top_indices`` [..., K], 1 <= K <= 128, and ``teacher_lse`` [...]. The
    gradient has the logits' type, one rounding; the teacher's arrays get none. For many logits
    it is formed with the loss (and takes their memory from then on): give a share of a mixed
    objective, or one over the micro-batches, as ``loss_weight``; an upstream factor other than
    1 forms it again. A listed token outside [0, V) other than ``ignore_index``, or a
    ``teacher_lse`` that is not the row's (weights of more than 256 in sum), makes the loss NaN
    and sets the error word that ``kernels.check_errors()`` raises
    (``DABSN_HIP_ERROR_CHECK=sync``: raised here)."""
    vocab.need_float(_WHAT, "logits", logits)
    if logits.dim() < 2:
        raise ValueError(f"{_WHAT}: expected logits [..., V] of one row or more")
    v = vocab.need_vocab(_WHAT, int(logits.shape[-1]))
    t = vocab.need_temperature(_WHAT, temperature)
    values, tokens, lse = _lists(logits.shape[:-1], v, top_logits, top_indices, teacher_lse)
    vocab.need_device(_WHAT, logits, values, tokens, lse)
    return _FromLogits.apply(vocab.rows_of(logits), values, tokens, lse, int(ignore_index), t,
                             _share(loss_weight), torch.is_grad_enabled())


def chunked_linear_distillation(hidden: Tensor, weight: Tensor, bias: Tensor | None,
                                top_logits: Tensor, top_indices: Tensor, *,
                                temperature: float = 1.0, teacher_lse: Tensor | None = None,
                                ignore_index: int = -100, loss_weight: float = 1.0,
                                chunk_budget: int | None = None) -> Tensor:
    """``distillation_from_logits(F.linear(hidden, weight, bias), ...)`` in chunks of
    ``chunk_budget // V`` rows (``DABSN_LOSS_CHUNK_SCORES``, default 2**25 elements), the logits
    in fp32 whatever the type of ``hidden`` [..., H]. Where a gradient is needed it is formed
    with the loss, chunk by chunk, and held in fp32 until the backward, which scales it and
    rounds it once to the inputs' types."""
    shape = hidden.shape[:-1]
    h, w, b = vocab.need_readout(_WHAT, hidden, weight, bias)
    t = vocab.need_temperature(_WHAT, temperature)
    values, tokens, lse = _lists(shape, int(w.shape[0]), top_logits, top_indices, teacher_lse)
    vocab.need_device(_WHAT, h, w, b, values, tokens, lse)
    chunk = vocab.chunk_rows(int(h.shape[0]), int(w.shape[0]), chunk_budget)
    return _Linear.apply(h, w, b, values, tokens, lse, int(ignore_index), t, _share(loss_weight),
                         chunk, torch.is_grad_enabled())
