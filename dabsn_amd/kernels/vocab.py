"""Calls of the vocabulary-row and embedding kernels, shared by ``scoring``, ``distill`` and
``embedding``: argument checks, error words, and the readout products of the chunked forms.

Indices out of range are found by the kernels. These operators run once per token in serving and
inside captured training steps, so they do not wait for the device: the kernel sets the device's
sticky error word, which ``check_errors()`` (and the training read) raises, and the row in
question is NaN. ``DABSN_HIP_ERROR_CHECK=sync`` raises from the call instead.
"""

from __future__ import annotations

import contextlib
import os

import torch
from torch import Tensor

from .. import _lib
from . import ops

MAX_TOP = 128
MAX_REST_VOCAB = 480_000
MAX_VOCAB = (1 << 31) - 4097
_CHUNK_BUDGET = 1 << 25
_GROUP_LOGITS = 1 << 27
_TOKEN_ERROR = ("a token lies outside [0, V) and is not ignore_index, or a teacher_lse is not its "
                "row's")
_HERE = contextlib.nullcontext()


def on(t: Tensor):
    """The device of ``t`` as the current one (the library launches on the current device)."""
    return _HERE if t.get_device() == torch._C._cuda_getDevice() else torch.cuda.device(t.device)


def no_autocast():
    """Products in the operands' own types (the context costs 5 us, so only where one is on)."""
    return torch.autocast("cuda", enabled=False) if torch.is_autocast_enabled("cuda") else _HERE


def stream(t: Tensor) -> int:
    """The current stream's handle on the device of ``t``."""
    return torch._C._cuda_getCurrentRawStream(t.get_device())


def at(t: Tensor | None, s: int) -> int | None:
    """Pointer to row s of a contiguous tensor."""
    if t is None:
        return None
    return t.data_ptr() + s * t.stride(0) * t.element_size() if s else t.data_ptr()


def once(backward):
    """A Function's backward that refuses to be differentiated itself. (``once_differentiable``
    takes a gradient whose upstream needs none for a constant, though it depends on the inputs, and
    costs 4 us of a small call's 25.)"""

    def run(ctx, *grads):
        if torch.is_grad_enabled():  # create_graph=True
            raise RuntimeError("DABSN HIP operators of the vocabulary have no second derivative: "
                               "run the backward without create_graph")
        return backward(ctx, *grads)

    return run


def need_device(what: str, *tensors: Tensor | None) -> None:
    """All tensors on one ROCm device."""
    first = None
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError(f"{what}: DABSN HIP operators need ROCm device tensors")
        if first is None:
            first = t
        elif t.get_device() != first.get_device():
            raise RuntimeError(f"{what}: tensors on {first.device} and {t.device}")


def need_float(what: str, name: str, t: Tensor) -> None:
    if t.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"{what}: {name} must be float32 or bfloat16, not {t.dtype}")


def need_tokens(what: str, name: str, t: Tensor, shape) -> Tensor:
    """Token numbers of the given shape as contiguous int64."""
    if t.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"{what}: {name} must be int64 or int32, not {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{what}: {name} {tuple(t.shape)} does not match {tuple(shape)}")
    if t.dtype != torch.int64:
        t = t.to(torch.int64)
    return t if t.is_contiguous() else t.contiguous()


def need_temperature(what: str, t: float) -> float:
    t = float(t)
    if not 1e-6 <= t <= 1e6:  # nor NaN
        raise ValueError(f"{what}: temperature must lie in [1e-6, 1e6], not {t}")
    return t


def need_vocab(what: str, v: int) -> int:
    if not 0 < v <= MAX_VOCAB:
        raise ValueError(f"{what}: a vocabulary of {v} words")
    return v


def rows_of(x: Tensor) -> Tensor:
    """x [..., V] as [rows, V] with unit column stride and rows that do not overlap."""
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    if (x.stride(1) != 1 and x.shape[1] > 1) or (x.stride(0) < x.shape[1] and x.shape[0] > 1):
        x = x.contiguous()
    return x


def row_stride(x: Tensor) -> int:
    """The row stride of ``rows_of``'s result (a lone row's stride says nothing)."""
    return max(x.stride(0), x.shape[1])


def grads_of(g: Tensor | None) -> Tensor | None:
    if g is None:
        return None
    return (g if g.dtype == torch.float32 else g.float()).contiguous()


class ErrorWord:
    """The int32 word a call's kernels set for tokens out of range (see the module's note)."""

    __slots__ = ("word", "own")

    def __init__(self, device: torch.device):
        self.own = ops._sync_mode() == "sync"
        sticky = ops._STICKY.get(device.index)
        if sticky is None:
            # The graph would make the word, and clear it on every replay.
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("the first DABSN HIP call on a device cannot be captured into a "
                                   "graph: call the operator once before the capture")
            sticky = ops._sticky(device)
        self.word = torch.zeros(1, device=device, dtype=torch.int32) if self.own else sticky

    def check(self, what: str) -> None:
        if self.own:
            ops._record_error_word(self.word.view(torch.uint8), what, _TOKEN_ERROR)


def chunk_rows(rows: int, vocab: int, budget: int | None) -> int:
    """Rows a chunk, so that its logits stay within the element budget (that of the readout loss if
    one is set, ``DABSN_LOSS_CHUNK_SCORES``, else 2**25; not positive or ``off``: all rows at once):
    chunks of equal height, of whole tiles of 128 rows where they allow it. The default is twice the
    loss's: 128 MB of fp32 logits, which the row kernel still finds in the memory-side cache, and
    products of 1024 rows by 32000 words (4096 rows scored in 622 us of kernels; 668 with 2**24 and
    670 with 2**26)."""
    if budget is None:
        env = os.environ.get("DABSN_LOSS_CHUNK_SCORES", "")
        try:
            budget = int(env) if env else _CHUNK_BUDGET
        except ValueError:
            budget = 0 if env.lower() == "off" else _CHUNK_BUDGET
    rows = max(rows, 1)
    if budget <= 0:
        return rows
    most = max(1, min(rows, int(budget) // max(1, vocab)))
    even = -(-rows // -(-rows // most))
    tiles = -(-even // 128) * 128
    return tiles if tiles <= most else even


class Readout:
    """The readout of rows ``hidden`` [N, H] by ``weight`` [V, H] and ``bias`` [V]: logits of
    row ranges in fp32. A bf16 readout's product keeps its fp32 sums (a rounding of the logits to
    bf16, 2^-9 of values around 10, would show in every log probability) and leaves the bias to
    the row kernel; adding it in the product took 30% longer (8192 x 2048 x 32000: 846 against
    1135 TFLOP/s)."""

    def __init__(self, hidden: Tensor, weight: Tensor, bias: Tensor | None):
        self.hidden, self.weight, self.bias = hidden, weight, bias
        self.half = hidden.dtype == torch.bfloat16
        self.row_bias = bias if self.half else None
        self.V, self.H = int(weight.shape[0]), int(weight.shape[1])
        self.wt = weight.t()

    def logits(self, s: int, e: int) -> Tensor:
        h = self.hidden[s:e]
        if self.half:
            return torch.mm(h, self.wt, out_dtype=torch.float32)
        return torch.mm(h, self.wt) if self.bias is None else torch.addmm(self.bias, h, self.wt)


def need_readout(what: str, hidden: Tensor, weight: Tensor, bias: Tensor | None):
    """(hidden [N, H], weight, bias) of one type, contiguous; inside autocast in its type, as
    ``F.linear`` casts them."""
    if hidden.dim() < 2 or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"{what}: hidden [..., H] and weight [V, H] do not match: "
                         f"{tuple(hidden.shape)}, {tuple(weight.shape)}")
    if bias is not None and tuple(bias.shape) != (weight.shape[0],):
        raise ValueError(f"{what}: bias {tuple(bias.shape)} does not match {weight.shape[0]} words")
    need_vocab(what, int(weight.shape[0]))
    if weight.shape[1] == 0:
        raise ValueError(f"{what}: hidden rows of width 0")
    if torch.is_autocast_enabled("cuda"):
        dt = torch.get_autocast_dtype("cuda")
        hidden, weight = hidden.to(dt), weight.to(dt)
        bias = None if bias is None else bias.to(dt)
    need_float(what, "hidden", hidden)
    if weight.dtype != hidden.dtype or (bias is not None and bias.dtype != hidden.dtype):
        raise TypeError(f"{what}: hidden, weight and bias must share a type")
    hidden = hidden.reshape(-1, hidden.shape[-1]).contiguous()
    return hidden, weight.contiguous(), None if bias is None else bias.contiguous()


def half_copy(x: Tensor) -> tuple[Tensor, Tensor]:
    """bf16 ``x`` as fp16 times a power of two (see ``dabsn_hip_half_copy``), and its inverse."""
    if x.data_ptr() % 16:
        x = x.clone()
    out = torch.empty(x.shape, device=x.device, dtype=torch.float16)
    aux = torch.empty(2, device=x.device, dtype=torch.float32)
    _lib.check(_lib.load().dabsn_hip_half_copy(x.numel(), x.data_ptr(), aux.data_ptr(),
                                               out.data_ptr(), aux.data_ptr() + 4, stream(x)),
               "half copy")
    return out, aux[1]


class ReadoutGrads:
    """Gradients of a ``Readout`` from gradient rows of its logits, in fp32: the row kernel
    writes rows where ``rows`` says, and ``end`` adds the products of a group of chunks (a product
    of few rows reaches a fifth of the rate: 524 rows x 32000 x 2048 243 TFLOP/s, 8192 rows 1356).

    fp32 readouts: fp32 rows and products, a chunk a group. bf16 ones:
      planes  two bf16 rows that hold 17 bits of each value, stacked as twice the rows of one bf16
              product; as many rows as the hidden width (the planes then take no more than the
              weight's fp32 gradient)
      split   these two bf16 rows for the weight's and the bias's gradients, each a product of its
              own, and one fp16 row, times a power of two by the row's size, for the hidden rows',
              with an fp16 copy of the weight that holds all of its bits, times a power of two; up to
              2**27 values in each, 0.8 GB (8192 x 2048 x 32000: 5.27 ms of kernels, 5.23 with 2**28
              and 6.27 with 2**26)
    """

    def __init__(self, r: Readout, need, chunk: int, split: bool = False):
        self.r, self.need = r, need
        n, V, H, dev = int(r.hidden.shape[0]), r.V, r.H, r.hidden.device
        f32 = torch.float32
        self.kind = "fp32" if not r.half else "split" if split else "planes"
        self.split = (bool(need[1] or need[2]) + 2 * bool(need[0])) if self.kind == "split" else 0
        self.hidden = self.weight = self.bias = None
        self.ldo = -(-V // 8) * 8 if r.half else V
        # A device scalar that the hidden rows' result has to be multiplied by.
        self.scale: Tensor | None = None
        if self.kind == "planes":
            # The products' copies (two fp32 rows and two bf16 rows of H a row) stay within the
            # weight's fp32 gradient or 512 MB.
            fit = max(1, max(4 * V * H, 1 << 29) // (12 * H))
            self.chunk = max(1, min(chunk, n, fit))
            self.group = self.chunk * max(1, min(fit, H) // self.chunk)
        elif self.kind == "split":
            self.chunk = chunk
            self.group = chunk * max(1, _GROUP_LOGITS // (self.ldo * chunk))
            if need[0] and n:
                self.half_weight, self.scale = half_copy(r.weight)
        else:
            self.chunk = self.group = chunk
        self.group = max(1, min(n, self.group))
        if need[0] and (self.kind != "split" or self.group < n or n == 0):
            self.hidden = torch.empty((n, H), device=dev, dtype=f32)
        self.parts = {"fp32": 1, "planes": 2, "split": 3}[self.kind]
        self.buf = torch.empty(self.parts * self.group * self.ldo, device=dev, dtype=r.hidden.dtype)
        self.inverse = torch.empty(self.group, device=dev, dtype=f32) if self.split & 2 else None
        self.first = True

    def groups(self):
        n = int(self.r.hidden.shape[0])
        return [(s, min(n, s + self.group)) for s in range(0, n, self.group)]

    def begin(self, g0: int, g1: int) -> None:
        self.g0, self.g1 = g0, g1

    def rows(self, s: int) -> int:
        """Pointer to the gradient rows from row s on; their stride is ``ldo`` (split rows' three
        times that) and the planes' ``plane()``."""
        step = self.ldo * (3 if self.kind == "split" else 1)
        return self.buf.data_ptr() + (s - self.g0) * step * self.buf.element_size()

    def inverses(self, s: int) -> int | None:
        """Pointer to what undoes the fp16 rows' factors from row s on."""
        return at(self.inverse, s - self.g0)

    def plane(self) -> int:
        return (self.g1 - self.g0) * self.ldo if self.kind == "planes" else 0

    def end(self) -> None:
        r, m, f32 = self.r, self.g1 - self.g0, torch.float32
        rows = r.hidden[self.g0:self.g1]
        if self.kind == "split":
            self._end_split(m, rows)
            return
        high = 2 * m if self.kind == "planes" else m
        d = self.buf[:high * self.ldo].view(high, self.ldo)[:, :r.V]
        if self.need[0]:
            if self.kind == "fp32":
                torch.mm(d, r.weight, out=self.hidden[self.g0:self.g1])
            else:
                p = torch.mm(d, r.weight, out_dtype=f32)
                torch.add(p[:m], p[m:], out=self.hidden[self.g0:self.g1])
                del p
        if self.need[1]:
            if self.kind == "planes":
                rows = torch.cat((rows, rows))
            if self.kind == "fp32":
                self.weight = (torch.mm(d.t(), rows) if self.first
                               else self.weight.addmm_(d.t(), rows))
            elif self.first:
                self.weight = torch.mm(d.t(), rows, out_dtype=f32)
            else:
                torch.addmm(self.weight, d.t(), rows, out_dtype=f32, out=self.weight)
            del rows
        if self.need[2]:
            if self.kind == "fp32":
                self.bias = d.sum(dim=0) if self.first else self.bias.add_(d.sum(dim=0))
            else:
                self._add_bias(high)
        self.first = False

    def _add_bias(self, rows: int) -> None:
        lib, V, dev = _lib.load(), self.r.V, self.buf.device
        if self.first:
            self.bias = torch.empty(V, device=dev, dtype=torch.float32)
        part = torch.empty(lib.dabsn_hip_column_sums_partials(rows, V), device=dev,
                           dtype=torch.float32)
        _lib.check(lib.dabsn_hip_column_sums(
            self.kind == "split", rows, V, self.ldo, self.buf.data_ptr(), not self.first,
            part.data_ptr(), self.bias.data_ptr(), stream(self.buf)), "readout bias gradient")

    def _end_split(self, m: int, rows: Tensor) -> None:
        f32, V = torch.float32, self.r.V
        d = self.buf[:3 * m * self.ldo].view(m, 3, self.ldo)[:, :, :V]
        if self.need[0]:
            p = torch.mm(d[:, 2].view(torch.float16), self.half_weight, out_dtype=f32)
            inverse = self.inverse[:m, None]
            if self.hidden is None:
                self.hidden = p.mul_(inverse)
            else:
                torch.mul(p, inverse, out=self.hidden[self.g0:self.g1])
            del p
        if self.need[1]:
            for i in range(2):
                if self.first and i == 0:
                    self.weight = torch.mm(d[:, 0].t(), rows, out_dtype=f32)
                else:
                    torch.addmm(self.weight, d[:, i].t(), rows, out_dtype=f32, out=self.weight)
        if self.need[2]:
            self._add_bias(m)
        self.first = False

    def results(self):
        """(hidden, weight, bias) gradients in fp32, None where not needed."""
        r = self.r
        if self.first:  # no rows
            zeros = lambda *s: torch.zeros(s, device=r.hidden.device, dtype=torch.float32)  # noqa: E731
            self.weight = zeros(r.V, r.H) if self.need[1] else None
            self.bias = zeros(r.V) if self.need[2] else None
        return self.hidden, self.weight, self.bias


def scaled(x: Tensor | None, like: torch.dtype, *scales: Tensor | None) -> Tensor | None:
    """fp32 ``x`` times up to three device scalars, rounded once to ``like``."""
    if x is None:
        return None
    out = torch.empty(x.shape, device=x.device, dtype=like)
    p = [ops._p(s) for s in scales] + [None] * (3 - len(scales))
    _lib.check(_lib.load().dabsn_hip_scaled(ops._code(like), x.numel(), x.data_ptr(), *p, 1.0,
                                            out.data_ptr(), stream(x)), "scaled gradient")
    return out
