"""Products with their epilogue, and the block's MLP, against 64 bits with the errors carried along.

Every value of the reference comes with a bound of the operator's error in it (``Val``). With
u = 2^-24 and r = eps / 2 of the tensors' type: a sum of n products is off by (n + 8) u of the
terms' magnitudes, in any order and grouping; an activation by its slope times the argument's error
and 8 u of its own terms; a slope by the second derivative (2, 0.8 and 0.5 at most) times the
argument's error; each rounding by r. These worst cases grow as the sums' magnitudes, so results are
also held to 3 r in the mean square relative to the reference's (fp32: and 4 u sqrt(n) for the n products of the sums on the path):
roundings of independent signs stay below the r / sqrt(3) of each of the at most four on a path."""

from __future__ import annotations

import math

import pytest
import torch

import dabsn_amd
from dabsn_amd import fused_linear, fused_mlp
from test_norm import D, U, case as norm_case, half_step, within

BF16, FP32 = torch.bfloat16, torch.float32


def _cpu(*shape, dtype=FP32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("call,error,match", [
    (lambda: fused_linear(_cpu(3, 4).half(), _cpu(5, 4).half()), TypeError, "float32 or bfloat16"),
    (lambda: fused_linear(torch.zeros(()), _cpu(5, 4)), ValueError, "expected x"),
    (lambda: fused_linear(_cpu(3, 4), _cpu(5, 3)), ValueError, "weight"),
    (lambda: fused_linear(_cpu(3, 4), _cpu(4)), ValueError, "weight"),
    (lambda: fused_linear(_cpu(3, 0), _cpu(5, 0)), ValueError, "weight"),
    (lambda: fused_linear(_cpu(3, 4), _cpu(0, 4)), ValueError, "weight"),
    (lambda: fused_linear(_cpu(3, 4), _cpu(5, 4, dtype=BF16)), TypeError, "weight"),
    (lambda: fused_linear(_cpu(3, 4), _cpu(5, 4), _cpu(4)), ValueError, "bias"),
    (lambda: fused_linear(_cpu(3, 4), _cpu(5, 4), _cpu(5, dtype=BF16)), TypeError, "bias"),
    (lambda: fused_linear(_cpu(3, 4), _cpu(5, 4), residual=_cpu(5)), ValueError, "residual"),
    (lambda: fused_linear(_cpu(3, 4), _cpu(5, 4), residual=_cpu(3, 5, dtype=BF16)), TypeError,
     "residual"),
    (lambda: fused_linear(_cpu(3, 4), _cpu(5, 4), activation="relu"), ValueError, "activation"),
    (lambda: fused_linear(_cpu(3, 4), _cpu(5, 4), activation=None), ValueError, "activation"),
    (lambda: fused_linear(_cpu(3, 4), _cpu(5, 4)), RuntimeError, "device"),
    (lambda: fused_mlp(_cpu(3, 4), _cpu(5, 4), _cpu(4, 5), norm="batch"), ValueError, "norm"),
    (lambda: fused_mlp(_cpu(3, 4), _cpu(5, 4), _cpu(4, 5), norm_bias=_cpu(4)), ValueError, "no bias"),
    (lambda: fused_mlp(_cpu(3, 4), _cpu(5, 4), _cpu(3, 5)), ValueError, "w2"),
    (lambda: fused_mlp(_cpu(3, 4), _cpu(5, 4), _cpu(4, 6)), ValueError, "w2"),
    (lambda: fused_mlp(_cpu(3, 4), _cpu(5, 4), _cpu(4, 5), _cpu(4)), ValueError, "b1"),
    (lambda: fused_mlp(_cpu(3, 4), _cpu(5, 4), _cpu(4, 5), eps=-1.0), ValueError, "eps"),
    (lambda: fused_mlp(_cpu(3, 4), _cpu(5, 4), _cpu(4, 5)), RuntimeError, "device"),
    (lambda: dabsn_amd.DABSNBlock(8, 8, 8, mlp_ratio=2.0, mlp_norm="layer"), ValueError,
     "go with mlp_activation"),
    (lambda: dabsn_amd.DABSNBlock(8, 8, 8, mlp_activation="gelu"), ValueError, "mlp_ratio"),
    (lambda: dabsn_amd.DABSNBlock(8, 8, 8, mlp_ratio=2.0, mlp_activation="tanh"), ValueError, "one of"),
    (lambda: dabsn_amd.DABSNSequenceLM(9, 8, mlp_ratio=2.0, mlp_activation="gelu", mlp_norm="x"),
     ValueError, "mlp_norm"),
])
def test_refusals(call, error, match):
    with pytest.raises(error, match=match):
        call()


def test_products_refuse_more_columns_than_they_take():
    w = torch.empty(1 << 21, 1)
    for call in (lambda: fused_linear(torch.empty(2, 1), w), lambda: fused_linear(torch.empty(2, 1 << 21), w.t()),
                 lambda: fused_mlp(torch.empty(2, 1), w, w.t())):
        with pytest.raises(ValueError, match="rows or columns"):
            call()


def test_library_refuses_bad_arguments_before_it_launches():
    from dabsn_amd import _lib

    lib, one = _lib.load(), 1 << 20
    import ctypes

    def call(**change):
        f = dict(dtype=0, transA=0, transB=0, act=0, slope_kind=0, M=4, N=8, K=16, A=one, B=one,
                 lda=16, ldb=16, ldc=8, lds=8, ldr=8, ldk=8, C=one)
        f.update(change)
        return lib.dabsn_hip_linear(ctypes.byref(_lib.LinearCall(**f)), None)

    for bad in (dict(dtype=2), dict(M=-1), dict(N=0), dict(K=-1), dict(M=1 << 31), dict(lda=15),
                dict(ldb=15), dict(transB=1, ldb=7), dict(transA=1, transB=1, lda=3), dict(ldc=7),
                dict(transA=1), dict(act=4), dict(act=-1), dict(slope=one, slope_kind=3),
                dict(slope=one, slope_kind=0), dict(slope=one, slope_kind=1, lds=7),
                dict(residual=one, ldr=7), dict(keep=one, ldk=7, act=2), dict(keep=one),
                dict(lda=1 << 21), dict(ldb=1 << 21), dict(ldc=1 << 21), dict(transB=1, ldb=8, act=1),
                dict(transB=1, ldb=8, bias=one), dict(transB=1, ldb=8, residual=one), dict(A=None), dict(B=None),
                dict(C=None)):
        assert call(**bad) == -2, bad
    assert lib.dabsn_hip_linear(None, None) == -2
    # Parts of a split product, and fp32 operands' planes, lie in the workspace.
    f = dict(dtype=0, M=256, N=2048, K=8192, A=one, B=one, C=one, lda=8192, ldb=8192, ldc=2048)
    need = lib.dabsn_hip_linear_workspace_bytes(ctypes.byref(_lib.LinearCall(**f)))
    assert need > 0 and lib.dabsn_hip_linear_workspace_bytes(None) == 0
    assert lib.dabsn_hip_linear_workspace_bytes(ctypes.byref(_lib.LinearCall(**{**f, "M": 0}))) == 0
    for ws, n in ((one, need - 1), (None, need), (one + 8, need)):
        assert call(**f, workspace=ws, workspace_bytes=n) == -2
    for dtype, rows, n, ldg, ws in ((2, 4, 8, 8, 1 << 30), (0, -1, 8, 8, 1 << 30), (0, 4, 0, 8, 1 << 30),
                                    (0, 4, 8, 7, 1 << 30), (0, 4, 8, 8, 0)):
        assert lib.dabsn_hip_linear_slope(dtype, rows, n, one, ldg, None, 0, 0, one, 8, one, one, ws,
                                          None) == -2


def test_library_refuses_bad_arguments_of_the_mlp_before_it_launches():
    import ctypes

    from dabsn_amd import _lib

    lib, one = _lib.load(), 1 << 20
    good = dict(dtype=1, wdtype=0, act=2, train=1, M=5, H=16, F=24, x=one, w1=one, w2=one, grad=one,
                ldx=16, ldw1=16, ldw2=24, out=one, dx=one, saved=one, workspace=one)

    def status(backward, **change):
        c = _lib.MlpCall(**{**good, **change})
        lib.dabsn_hip_mlp_plan(ctypes.byref(c), backward)
        for name in ("saved_bytes", "workspace_bytes"):
            if name in change:
                setattr(c, name, change[name])
        return (lib.dabsn_hip_mlp_bwd if backward else lib.dabsn_hip_mlp_fwd)(ctypes.byref(c), None)

    for backward in (0, 1):
        for bad in (dict(dtype=2), dict(M=-1), dict(M=1 << 31), dict(H=0), dict(H=16385), dict(F=0),
                    dict(F=1 << 21), dict(act=4), dict(act=-1), dict(ldx=15), dict(ldw1=15),
                    dict(ldw2=23), dict(x=None), dict(w1=None), dict(w2=None), dict(wdtype=3),
                    dict(ldx=1 << 21), dict(ldw1=1 << 21), dict(ldw2=1 << 21), dict(saved=None),
                    dict(saved=one + 8), dict(saved_bytes=8), dict(workspace=None, train=backward),
                    dict(workspace=one + 8, train=backward), dict(workspace_bytes=8, train=backward)):
            assert status(backward, **bad) == -2, (backward, bad)
    assert status(0, out=None) == -2
    for bad in (dict(grad=None), dict(train=0)):
        assert status(1, **bad) == -2, bad
    assert lib.dabsn_hip_mlp_fwd(None, None) == -2 and lib.dabsn_hip_mlp_bwd(None, None) == -2
    assert lib.dabsn_hip_mlp_plan(None, 0) == -2


def test_library_refuses_bad_arguments_of_a_layers_gradients():
    import ctypes

    from dabsn_amd import _lib

    lib, one = _lib.load(), 1 << 20
    good = dict(dtype=1, slope_kind=1, M=40, N=24, K=16, x=one, w=one, grad=one, slope=one, ldx=16,
                ldw=16, ldg=24, lds=24, dx=one, dw=one, db=one, workspace=one)
    need = lib.dabsn_hip_linear_grads_workspace_bytes(ctypes.byref(_lib.LinearGradsCall(**good)))
    assert need > 0 and lib.dabsn_hip_linear_grads_workspace_bytes(None) == 0
    for bad in (dict(dtype=2), dict(M=-1), dict(M=1 << 31), dict(N=0), dict(N=1 << 21), dict(K=0),
                dict(K=1 << 21), dict(ldx=15), dict(ldw=15), dict(ldg=23), dict(lds=23), dict(ldx=1 << 21),
                dict(ldw=1 << 21), dict(ldg=1 << 21), dict(lds=1 << 21), dict(slope_kind=0),
                dict(slope_kind=3), dict(x=None), dict(w=None), dict(grad=None), dict(workspace=None),
                dict(workspace=one + 8), dict(workspace_bytes=need - 1)):
        c = _lib.LinearGradsCall(**{**good, "workspace_bytes": need, **bad})
        assert lib.dabsn_hip_linear_grads(ctypes.byref(c), None) == -2, bad
    assert lib.dabsn_hip_linear_grads(None, None) == -2


class Val:
    """A value in 64 bits and a bound of the error in what the operator holds of it."""

    def __init__(self, v, e=None):
        self.v = v.detach().double()
        self.e = torch.zeros_like(self.v) if e is None else e

    def t(self):
        return Val(self.v.t(), self.e.t())

    def __matmul__(self, o):
        n = self.v.shape[1]
        mag = self.v.abs() @ o.v.abs()
        err = self.e @ o.v.abs() + self.v.abs() @ o.e + self.e @ o.e
        return Val(self.v @ o.v, err + (n + 8) * U * (mag + err))

    def __add__(self, o):
        if o is None:
            return self
        v = self.v + o.v
        return Val(v, self.e + o.e + U * (v.abs() + self.e + o.e))

    def __mul__(self, o):
        v = self.v * o.v
        e = self.v.abs() * o.e + self.e * o.v.abs() + self.e * o.e
        return Val(v, e + U * (v.abs() + e))

    def rounded(self, dtype):
        r = half_step(dtype)
        return Val(self.v, self.e + r * (self.v.abs() + self.e) + 2.0 ** -133)

    def sums(self):
        n = self.v.shape[0]
        return Val(self.v.sum(0), self.e.sum(0) + (n + 40) * U * (self.v.abs() + self.e).sum(0))


def activated(z: Val, act: str):
    """(act(z), act'(z))."""
    v, e = z.v, z.e
    if act == "none":
        return z, Val(torch.ones_like(v))
    if act == "relu2":
        r = v.clamp(min=0)
        return (Val(r * r, (2 * r + e) * e + 2 * U * (r + e) ** 2), Val(2 * r, 2 * e + 2 * U * r))
    if act == "gelu":
        p = 0.5 * torch.special.erfc(-v * math.sqrt(0.5))  # (ndtr is 1 + erf: 2^-53 off in the tail)
        d = torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)
        return (Val(v * p, 1.13 * e + 8 * U * (v * p).abs() + 2 * U * v.abs()),
                Val(p + v * d, 0.8 * e + 16 * U * (p + v.abs() * d) + 4 * U))
    s = torch.sigmoid(v)
    return (Val(v * s, 1.1 * e + 8 * U * (v * s).abs()),
            Val(s * (1 + v * (1 - s)), 0.5 * e + 16 * U * s * (1 + v.abs() * (1 - s))))


def kept(slope: Val, h: Val, act: str, dtype):
    """The slope as the backward has it."""
    if act == "relu2":
        # From the rounded output: the root halves its relative error; small outputs by their own.
        h = h.rounded(dtype)
        low = 2 * (h.v - h.e).clamp(min=0).sqrt()
        high = 2 * (h.v + h.e).sqrt()
        return Val(slope.v, torch.maximum(high - slope.v, slope.v - low) + 4 * U * high)
    if act != "none" and dtype == BF16:
        # In fp16. GELU's distribution function is a fit there, whose tail, at most 1/2, is off by
        # 1.7e-5 of itself: 8.5e-6, which the slope p(z) + z p'(z) has whole where it passes 0.
        fit = 8.5e-6 if act == "gelu" else 0.0
        return Val(slope.v, slope.e + fit + 2.0 ** -11 * (slope.v.abs() + slope.e + fit) + 2.0 ** -25)
    return slope if act == "none" else slope.rounded(dtype)


def check(name, got, want: Val, dtype, terms, spread=True):
    want = want.rounded(dtype)
    within(got, want.v, want.e)
    if spread and want.v.numel() >= 256:
        ratio = float((got.double() - want.v).norm() / want.v.norm())
        most = 3 * half_step(dtype) + (U * math.sqrt(terms) * 4 if dtype == FP32 else 0)
        assert ratio <= most, (name, ratio, most)


def tensors(seed, m, k, n, dtype, bias, residual):
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    t = {"x": rand(m, k), "weight": rand(n, k) / math.sqrt(k), "bias": 0.3 * rand(n) if bias else None,
         "residual": rand(m, n) if residual else None, "grad": rand(m, n)}
    return {name: None if v is None else v.to(dtype).cuda() for name, v in t.items()}


def run(t, act):
    leaves = {k: None if v is None else v.detach().clone().requires_grad_(True)
              for k, v in t.items() if k != "grad"}
    out = fused_linear(leaves["x"], leaves["weight"], leaves["bias"], activation=act,
                       residual=leaves["residual"])
    real = {k: v for k, v in leaves.items() if v is not None}
    grads = torch.autograd.grad(out, list(real.values()), t["grad"])
    return {"out": out.detach(), **dict(zip(real, grads))}


def check_linear(t, act, got):
    dtype = t["x"].dtype
    x, w, g = Val(t["x"]), Val(t["weight"]), Val(t["grad"])
    m, k = t["x"].shape
    n = t["weight"].shape[0]
    z = x @ w.t() + (None if t["bias"] is None else Val(t["bias"]))
    h, slope = activated(z, act)
    res = t["residual"] is not None
    check("out", got["out"], h + (Val(t["residual"]) if res else None), dtype, k)
    if len(got) == 1:
        return
    exact = g * kept(slope, h, act, dtype)
    dz = exact if act == "none" else exact.rounded(dtype)
    check("x", got["x"], dz @ w, dtype, k + n)
    check("weight", got["weight"], dz.t() @ x, dtype, k + m)
    if t["bias"] is not None:
        # Few terms, whose sum cancels as it likes: the worst case alone.
        check("bias", got["bias"], exact.sums(), dtype, 0, spread=False)
    if res:
        assert torch.equal(got["residual"], t["grad"])


SIZES = [(1, 1, 1), (1, 2048, 40), (2, 33, 2050), (3, 7, 5), (15, 520, 96), (16, 64, 48), (17, 64, 33),
         (33, 129, 65), (64, 100, 130), (129, 257, 127), (128, 128, 128), (300, 1001, 77),
         (256, 8192, 64), (1000, 40, 999), (513, 640, 1100), (5000, 24, 17), (2, 9000, 3)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("act,bias,residual", [("none", False, False), ("none", True, True),
                                               ("relu2", True, False), ("relu2", False, True),
                                               ("gelu", True, True), ("silu", True, False)])
@pytest.mark.parametrize("m,k,n", SIZES)
def test_linear(cuda_device, m, k, n, act, bias, residual, dtype):
    t = tensors(m + k + n, m, k, n, dtype, bias, residual)
    got = run(t, act)
    check_linear(t, act, got)
    again = run(t, act)
    assert all(torch.equal(got[k], again[k]) for k in got)
    with torch.no_grad():
        plain = fused_linear(t["x"], t["weight"], t["bias"], activation=act, residual=t["residual"])
    assert torch.equal(plain, got["out"])


# Sizes whose products take the large tiles, with splits and without, in each direction: 256 x 256
# (the first two in all three, of either type; the second split in the forward), 128 x 64 (third and
# fifth, bf16 forward), 128 x 128 (of fp32 planes, the third's weight gradient; of fp32 as it lies,
# the fourth's forward and gradient of the rows and the sixth's weight gradient), and many splits.
LARGE = [(4001, 4010, 3999), (2049, 9001, 2050), (300, 5000, 4100), (5000, 300, 700),
         (515, 6000, 3000), (9000, 200, 2000), (5000, 700, 300), (300, 264, 33000), (20, 50000, 100)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("act,bias,residual", [("relu2", False, False), ("gelu", True, True)])
@pytest.mark.parametrize("m,k,n", LARGE)
def test_linear_large(cuda_device, m, k, n, act, bias, residual, dtype):
    t = tensors(m + k + n, m, k, n, dtype, bias, residual)
    check_linear(t, act, run(t, act))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_linear_large_strides(cuda_device, dtype):
    """256 x 256 tiles whose edges end inside wider arrays of NaN, at odd offsets; the results of
    contiguous operands, bit for bit where the same tiles take them."""
    m, k, n = 4001, 1000, 3999
    t = tensors(1, m, k, n, dtype, True, True)
    wide = {a: torch.full((v.shape[0], v.shape[1] + 5), math.nan, device=v.device, dtype=dtype)
            for a, v in t.items() if v.dim() == 2}
    for a, v in wide.items():
        v[:, 3:-2] = t[a]
    view = {**t, **{a: v[:, 3:-2] for a, v in wide.items()}}
    leaves = {a: view[a].requires_grad_(True) for a in ("x", "weight", "residual")}
    out = fused_linear(leaves["x"], leaves["weight"], t["bias"], activation="silu", residual=leaves["residual"])
    gx, gw, gr = torch.autograd.grad(out, tuple(leaves.values()), view["grad"])
    got = {"out": out.detach(), "x": gx, "weight": gw, "residual": gr}
    check_linear({**t, "bias": t["bias"]}, "silu", {**got, "bias": run(t, "silu")["bias"]})


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("m,k,n", [(1, 8, 300), (5, 1000, 1001), (16, 4104, 16), (9, 33, 5000), (4, 50000, 70)])
def test_linear_few_rows_at_any_offset(cuda_device, m, k, n, dtype):
    """Up to 16 rows, operands and results at every offset modulo eight values."""
    t = tensors(m + n, m, k, n, dtype, True, True)
    want = fused_linear(t["x"], t["weight"], t["bias"], activation="gelu", residual=t["residual"])
    check_linear(t, "gelu", {"out": want})
    for off in (1, 2, 3, 5, 8):
        place = {}
        for a in ("x", "weight", "residual"):
            wide = torch.full((t[a].shape[0], t[a].shape[1] + off + 4), math.nan, device="cuda", dtype=dtype)
            wide[:, off:off + t[a].shape[1]] = t[a]
            place[a] = wide[:, off:off + t[a].shape[1]]
        got = fused_linear(place["x"], place["weight"], t["bias"], activation="gelu", residual=place["residual"])
        check_linear(t, "gelu", {"out": got})


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("m,k,n", [(5, 77, 45), (70, 77, 45), (200, 200, 200), (300, 1000, 264)])
def test_linear_strides_and_edges(cuda_device, m, k, n, dtype):
    """Operands inside wider arrays full of NaN, at odd offsets: nothing beyond an edge is used."""
    t = tensors(4, m, k, n, dtype, True, True)
    want = run(t, "silu")

    def inside(v, left, right):
        wide = torch.full((v.shape[0], v.shape[1] + left + right), math.nan, device=v.device, dtype=dtype)
        wide[:, left:left + v.shape[1]] = v
        return wide.requires_grad_(True), slice(left, left + v.shape[1])

    for left, right in ((1, 2), (8, 8), (3, 0)):
        (x, xs), (w, ws), (r, rs) = (inside(t[a], left, right) for a in ("x", "weight", "residual"))
        grad, gs = inside(t["grad"], left, right)
        b = t["bias"].clone().requires_grad_(True)
        out = fused_linear(x[:, xs], w[:, ws], b, activation="silu", residual=r[:, rs])
        gx, gw, gb, gr = torch.autograd.grad(out, (x, w, b, r), grad.detach()[:, gs])
        got = {"out": out.detach(), "x": gx[:, xs], "weight": gw[:, ws], "bias": gb, "residual": gr[:, rs]}
        check_linear(t, "silu", got)
        assert torch.equal(got["out"], want["out"]) and torch.equal(gb, want["bias"])
    # A weight stored transposed, rows that overlap (stride 0), a gradient from expand.
    turned = t["weight"].t().contiguous().t()
    same = fused_linear(t["x"], turned, t["bias"], activation="silu", residual=t["residual"])
    assert torch.equal(same, want["out"])
    one = {**t, "x": t["x"][:1].expand(m, k), "residual": t["residual"][:1].expand(m, n),
           "grad": t["grad"][:1].expand(m, n)}
    leaf = t["weight"].clone().requires_grad_(True)
    out = fused_linear(one["x"], leaf, t["bias"], activation="silu", residual=one["residual"])
    check_linear(one, "silu", {"out": out})
    (gw,) = torch.autograd.grad(out, leaf, one["grad"])
    full = run({**{a: v.contiguous() for a, v in one.items()}}, "silu")
    assert torch.equal(gw, full["weight"])


@pytest.mark.gpu
def test_linear_shapes_and_needed_gradients(cuda_device):
    t = tensors(5, 60, 50, 40, BF16, True, True)
    want = run(t, "gelu")
    cube = fused_linear(t["x"].view(3, 20, 50), t["weight"], t["bias"], activation="gelu",
                        residual=t["residual"].view(3, 20, 40))
    assert cube.shape == (3, 20, 40) and torch.equal(cube.view(60, 40), want["out"])
    row = fused_linear(t["x"][7], t["weight"], t["bias"], activation="gelu", residual=t["residual"][7])
    assert row.shape == (40,)
    check_linear({**t, "x": t["x"][7:8], "residual": t["residual"][7:8]}, "gelu", {"out": row[None]})
    for name in ("x", "weight", "bias", "residual"):
        leaf = t[name].clone().requires_grad_(True)
        args = {**t, name: leaf}
        out = fused_linear(args["x"], args["weight"], args["bias"], activation="gelu",
                           residual=args["residual"])
        (got,) = torch.autograd.grad(out, leaf, t["grad"])
        assert torch.equal(got, want[name]), name
    # One tensor in two places: a residual that is the input, as in a block.
    sq = tensors(6, 60, 50, 50, FP32, False, False)
    leaf = sq["x"].clone().requires_grad_(True)
    out = fused_linear(leaf, sq["weight"], residual=leaf)
    (got,) = torch.autograd.grad(out, leaf, sq["grad"])
    ref = sq["grad"].double() + sq["grad"].double() @ sq["weight"].double()
    assert float((got.double() - ref).abs().max()) < 1e-4


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_linear_no_rows(cuda_device, dtype):
    t = tensors(7, 0, 41, 13, dtype, True, True)
    got = run(t, "gelu")
    assert got["out"].shape == (0, 13) and got["x"].shape == (0, 41)
    assert float(got["weight"].float().abs().sum() + got["bias"].float().abs().sum()) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("m", [3, 100, 700])
def test_nan_and_infinity_stay_in_their_rows(cuda_device, m, dtype):
    t = tensors(8, m, 90, 70, dtype, True, False)
    want = run(t, "relu2")
    t["x"][1, 89], t["x"][2, 0] = math.nan, math.inf
    got = run(t, "relu2")["out"]
    keep = torch.ones(m, dtype=torch.bool)
    keep[[1, 2]] = False
    assert torch.equal(got[keep], want["out"][keep])
    assert bool(torch.isnan(got[1]).all())
    finite = torch.isfinite(got[2])  # -inf before the activation becomes 0, +inf stays
    assert bool((got[2][finite] == 0).all()) and bool(finite.any()) and not bool(finite.all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("m,k,n", [(40, 64, 40), (1500, 500, 4000), (4001, 1000, 3999), (2049, 9001, 2050)])
def test_infinity_times_round_numbers(cuda_device, m, k, n, dtype):
    """An infinity times weights that bf16 holds whole, or times 0, in products of every kind (the
    third large, the last split): what each sum of products is in 64 bits, infinite or NaN."""
    g = torch.Generator(device=cuda_device).manual_seed(m)
    t = {"x": torch.randn(m, k, device=cuda_device, generator=g), "grad": torch.randn(m, n, device=cuda_device, generator=g),
         "weight": torch.randint(-2, 3, (n, k), device=cuda_device, generator=g).float()}
    t["x"][3, k - 1], t["x"][m - 1, 0], t["x"][7, 1], t["x"][7, 2] = math.inf, -math.inf, math.inf, -math.inf
    t["grad"][5, n - 1], t["grad"][m - 2, 0], t["x"][9, 5] = -math.inf, math.inf, math.nan
    t = {a: v.to(dtype) for a, v in t.items()}
    got = run({**t, "bias": None, "residual": None}, "none")
    x, w, d = (t[a].double() for a in ("x", "weight", "grad"))
    for name, want in (("out", x @ w.t()), ("x", d @ w), ("weight", d.t() @ x)):
        have = got[name].double()
        assert torch.equal(torch.isnan(have), torch.isnan(want)), name
        odd = torch.isinf(want)
        assert torch.equal(have[odd], want[odd]) and torch.equal(torch.isinf(have), odd), name


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["relu2", "gelu", "silu"])
@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_activations_over_their_range(cuda_device, act, dtype):
    """Arguments from -120 to 120 through a product with one term: values relative to themselves
    (their tails too), slopes within their bound."""
    v = torch.cat((torch.linspace(-120, 120, 4001), torch.linspace(-6, 6, 4001), torch.zeros(1)))
    x = v.to(dtype).cuda()[:, None].requires_grad_(True)
    one = torch.ones(1, 1, device=cuda_device, dtype=dtype)
    out = fused_linear(x, one, activation=act)
    (dx,) = torch.autograd.grad(out, x, torch.ones_like(out))
    z = x.detach().double()
    h, slope = activated(Val(z), act)
    r = half_step(dtype)
    # exp's argument is up to 120 (gelu: 7200, but its exp is 0 beyond 104), off by u of itself, which
    # is as much of the value. Factors below fp32's smallest normal number 2^-126 count as 0: that
    # is |z| 2^-126 of a product with z.
    low = (1 + z.abs()) * 2.0 ** -126
    within(out, h.v, (r + 400 * U) * h.v.abs() + low)
    within(dx, slope.v, kept(slope, h, act, dtype).e + (r + 400 * U) * slope.v.abs() + low)


@pytest.mark.gpu
def test_more_rows_than_32_bit_offsets(cuda_device):
    """Results and operands beyond 2^31 elements."""
    m, k, n = 2_200_000, 8, 1000
    g = torch.Generator(device=cuda_device).manual_seed(2)
    x = torch.randn(m, k, device=cuda_device, generator=g).to(BF16)
    w = torch.randn(n, k, device=cuda_device, generator=g).to(BF16)
    out = fused_linear(x, w, activation="relu2")
    for s in (0, 1_000_000, m - 5):
        check_linear({"x": x[s:s + 5], "weight": w, "bias": None, "residual": None, "grad": out[s:s + 5]},
                     "relu2", {"out": out[s:s + 5]})
    leaf = w.clone().requires_grad_(True)
    (gw,) = torch.autograd.grad(fused_linear(x, leaf), leaf, out)
    ref = torch.zeros(n, k, device=cuda_device, dtype=torch.float64)
    mag = torch.zeros_like(ref)
    for s in range(0, m, 200_000):
        a, b = out[s:s + 200_000].double(), x[s:s + 200_000].double()
        ref += a.t() @ b
        mag += a.abs().t() @ b.abs()
    within(gw, ref, m * U * mag + 2.0 ** -8 * ref.abs())
    assert float((gw.double() - ref).norm() / ref.norm()) < 2.0 ** -8


@pytest.mark.gpu
def test_no_second_derivative(cuda_device):
    x = torch.randn(4, 8, device=cuda_device, requires_grad=True)
    w = torch.randn(8, 8, device=cuda_device, requires_grad=True)
    for out in (fused_linear(x, w, activation="silu"), fused_mlp(x, w, w)):
        with pytest.raises(RuntimeError, match="second derivative"):
            torch.autograd.grad(out.sum(), x, create_graph=True)


# ---- the MLP ----------------------------------------------------------------------------------
NAMES = ("x", "norm_weight", "norm_bias", "w1", "b1", "w2", "b2")


def mlp_tensors(seed, m, h, f, dtype, layer, bias):
    x, nw, nb, grad = norm_case(seed, m, h, dtype, dtype, layer)
    g = torch.Generator().manual_seed(seed + 1)
    rand = lambda *s: torch.randn(*s, generator=g).to(dtype).cuda()  # noqa: E731
    return {"x": x, "norm_weight": nw, "norm_bias": nb, "w1": rand(f, h) / math.sqrt(h),
            "w2": rand(h, f) / math.sqrt(f), "b1": 0.3 * rand(f) if bias else None,
            "b2": 0.3 * rand(h) if bias else None, "grad": grad}


def run_mlp(t, act, layer):
    leaves = {a: None if t[a] is None else t[a].detach().clone().requires_grad_(True) for a in NAMES}
    out = fused_mlp(leaves["x"], leaves["w1"], leaves["w2"], leaves["b1"], leaves["b2"],
                    norm="layer" if layer else "rms", norm_weight=leaves["norm_weight"],
                    norm_bias=leaves["norm_bias"], activation=act)
    real = {a: v for a, v in leaves.items() if v is not None}
    return {"out": out.detach(), **dict(zip(real, torch.autograd.grad(out, list(real.values()), t["grad"])))}


def check_mlp(t, act, layer, got):
    dtype = t["x"].dtype
    eps = 1e-5 if layer else 1e-6
    x, w1, w2 = Val(t["x"]), Val(t["w1"]), Val(t["w2"])
    nw = Val(t["norm_weight"])
    mean = x.v.mean(1, keepdim=True) if layer else 0.0
    std = ((x.v - mean).square().mean(1, keepdim=True) + eps).sqrt()
    unit = (x.v - mean) / std
    e = (D / 2 + 9) * U * unit.abs()
    if layer:
        e = e + D * U * x.v.abs().mean(1, keepdim=True) / std
    unit = Val(unit, e)
    some = lambda a: None if t[a] is None else Val(t[a])  # noqa: E731
    normed = (unit * nw + some("norm_bias")).rounded(dtype)
    z = normed @ w1.t() + some("b1")
    h, slope = activated(z, act)
    h16 = h.rounded(dtype)
    out = h16 @ w2.t() + some("b2") + x
    f, width = t["w1"].shape
    check("out", got["out"], out, dtype, f + width)
    g = Val(t["grad"])
    dz = ((g @ w2) * kept(slope, h, act, dtype)).rounded(dtype)
    dn = (dz @ w1).rounded(dtype)
    gw = dn * nw
    level = Val(gw.v.mean(1, keepdim=True), gw.e.mean(1, keepdim=True) + D * U * gw.v.abs().mean(1, keepdim=True))
    both = gw * unit
    along = Val(both.v.mean(1, keepdim=True),
                both.e.mean(1, keepdim=True) + (D + 4) * U * both.v.abs().mean(1, keepdim=True))
    d = Val(gw.v - (level.v if layer else 0) - unit.v * along.v,
            gw.e + (level.e if layer else 0) + (unit * along).e + 4 * U * (
                gw.v.abs() + (unit.v * along.v).abs() + level.v.abs()))
    dx = Val(d.v / std, (d.e + (D / 2 + 12) * U * d.v.abs()) / std)
    rows = t["x"].shape[0]
    check("x", got["x"], dx + g, dtype, 2 * (f + width))
    check("norm_weight", got["norm_weight"], (dn * unit).sums(), dtype, 0, spread=False)
    if layer:
        check("norm_bias", got["norm_bias"], dn.sums(), dtype, 0, spread=False)
    check("w1", got["w1"], dz.t() @ normed, dtype, rows + f + width)
    check("w2", got["w2"], g.t() @ h16, dtype, rows + width)
    if t["b1"] is not None:
        check("b1", got["b1"], dz.sums(), dtype, 0, spread=False)
        check("b2", got["b2"], g.sums(), dtype, 0, spread=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("act,layer,bias", [("relu2", False, False), ("gelu", True, True),
                                            ("silu", False, True), ("relu2", True, True)])
@pytest.mark.parametrize("m,h,f", [(1, 1, 1), (1, 96, 384), (5, 24, 61), (33, 130, 65), (200, 256, 1024),
                                   (300, 77, 308), (1000, 64, 200), (130, 520, 1)])
def test_mlp(cuda_device, m, h, f, act, layer, bias, dtype):
    t = mlp_tensors(m + h + f, m, h, f, dtype, layer, bias)
    got = run_mlp(t, act, layer)
    check_mlp(t, act, layer, got)
    again = run_mlp(t, act, layer)
    assert all(torch.equal(got[a], again[a]) for a in got)
    with torch.no_grad():
        plain = fused_mlp(t["x"], t["w1"], t["w2"], t["b1"], t["b2"], norm="layer" if layer else "rms",
                          norm_weight=t["norm_weight"], norm_bias=t["norm_bias"], activation=act)
    assert torch.equal(plain, got["out"])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("act,layer", [("relu2", False), ("gelu", True)])
@pytest.mark.parametrize("m,h,f", [(4001, 1000, 3999), (300, 2048, 4100), (6000, 256, 1024)])
def test_mlp_large(cuda_device, m, h, f, act, layer, dtype):
    """The slopes in the epilogues of the large tiles."""
    t = mlp_tensors(m, m, h, f, dtype, layer, True)
    check_mlp(t, act, layer, run_mlp(t, act, layer))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("m,h,f", [(5, 24, 61), (33, 130, 65), (130, 77, 331), (700, 1001, 777)])
def test_buffers_start_as_they_like(cuda_device, m, h, f, dtype):
    """Workspaces and results whose memory holds NaN before the call."""
    def poison():
        junk = [torch.full((1 << s,), math.nan, device="cuda") for s in range(8, 24)]
        junk += [torch.full((1 << 23,), math.nan, device="cuda") for _ in range(6)]
        torch.cuda.synchronize()

    t = mlp_tensors(m, m, h, f, dtype, True, True)
    lin = tensors(m, m, h, f, dtype, True, True)
    for act in ("relu2", "gelu"):
        poison()
        check_mlp(t, act, True, run_mlp(t, act, True))
        poison()
        check_linear(lin, act, run(lin, act))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_row_strides_beyond_the_kernels(cuda_device, dtype):
    """Rows further apart than the products take are copied: an operand, a weight and a gradient."""
    t = tensors(3, 20, 40, 24, dtype, True, False)
    want = run(t, "silu")
    wide = {a: torch.empty(t[a].shape[0], (1 << 21) + 8, device="cuda", dtype=dtype) for a in ("x", "weight", "grad")}
    for a, v in wide.items():
        v[:, 8:8 + t[a].shape[1]] = t[a]
        wide[a] = v[:, 8:8 + t[a].shape[1]]
    x, w = wide["x"].requires_grad_(True), wide["weight"].requires_grad_(True)
    out = fused_linear(x, w, t["bias"], activation="silu")
    gx, gw = torch.autograd.grad(out, (x, w), wide["grad"])
    assert torch.equal(out, want["out"]) and torch.equal(gx, want["x"]) and torch.equal(gw, want["weight"])
    one = fused_linear(wide["x"].detach()[:1], t["weight"], t["bias"], activation="silu")
    assert torch.equal(one, fused_linear(t["x"][:1], t["weight"], t["bias"], activation="silu"))


@pytest.mark.gpu
def test_mlp_is_its_parts(cuda_device):
    """The MLP's forward is the norm and two products of the public operators, bit for bit."""
    t = mlp_tensors(3, 90, 72, 200, BF16, True, True)
    normed = dabsn_amd.layer_norm(t["x"], t["norm_weight"], t["norm_bias"])
    h = fused_linear(normed, t["w1"], t["b1"], activation="gelu")
    want = fused_linear(h, t["w2"], t["b2"], residual=t["x"])
    got = fused_mlp(t["x"], t["w1"], t["w2"], t["b1"], t["b2"], norm="layer",
                    norm_weight=t["norm_weight"], norm_bias=t["norm_bias"], activation="gelu")
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_mlp_each_gradient_alone_and_shapes(cuda_device):
    t = mlp_tensors(4, 66, 40, 100, FP32, True, True)
    want = run_mlp(t, "gelu", True)
    for name in NAMES:
        leaf = t[name].clone().requires_grad_(True)
        a = {**t, name: leaf}
        out = fused_mlp(a["x"].view(2, 33, 40), a["w1"], a["w2"], a["b1"], a["b2"], norm="layer",
                        norm_weight=a["norm_weight"], norm_bias=a["norm_bias"], activation="gelu")
        assert out.shape == (2, 33, 40)
        (got,) = torch.autograd.grad(out, leaf, t["grad"].view(2, 33, 40))
        assert torch.equal(got, want[name]), name
    x = t["x"].clone().requires_grad_(True)
    out = fused_mlp(x, t["w1"], t["w2"])  # no weight in the norm
    ref = x.double() / (x.double().square().mean(1, keepdim=True) + 1e-6).sqrt()
    ref = x.double() + (ref @ t["w1"].double().t()).clamp(min=0).square() @ t["w2"].double().t()
    assert float((out.double() - ref).abs().max()) < 1e-4
    (got,) = torch.autograd.grad(out, x, t["grad"])
    (exact,) = torch.autograd.grad(ref, x, t["grad"].double())
    assert float((got.double() - exact).abs().max()) < 1e-4
    none = fused_mlp(t["x"][:0], t["w1"], t["w2"])
    assert none.shape == (0, 40)
    empty = run_mlp({**t, "x": t["x"][:0], "grad": t["grad"][:0]}, "gelu", True)
    assert empty["x"].shape == (0, 40) and all(float(empty[a].abs().sum()) == 0 for a in NAMES)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("m", [3, 130])
def test_mlp_strides(cuda_device, m, dtype):
    """Rows and weights inside wider arrays of NaN, transposed weights, a gradient from expand."""
    t = mlp_tensors(7, m, 40, 84, dtype, True, True)
    want = run_mlp({**t, "grad": t["grad"][:1].expand(m, 40).contiguous()}, "silu", True)
    views = {}
    for a in ("x", "w1", "w2"):
        wide = torch.full((t[a].shape[0], t[a].shape[1] + 7), math.nan, device="cuda", dtype=dtype)
        wide[:, 3:-4] = t[a]
        views[a] = wide[:, 3:-4]
    for w1 in (views["w1"], t["w1"].t().contiguous().t()):
        leaves = {**t, **views, "w1": w1}
        leaves = {a: leaves[a].requires_grad_(True) if a in ("x", "w1", "w2") else t[a] for a in NAMES}
        out = fused_mlp(leaves["x"], leaves["w1"], leaves["w2"], t["b1"], t["b2"], norm="layer",
                        norm_weight=t["norm_weight"], norm_bias=t["norm_bias"], activation="silu")
        assert torch.equal(out, want["out"])
        grads = torch.autograd.grad(out, [leaves[a] for a in ("x", "w1", "w2")], t["grad"][:1].expand(m, 40))
        for a, got in zip(("x", "w1", "w2"), grads):
            assert got.shape == t[a].shape and torch.equal(got, want[a]), a


@pytest.mark.gpu
@pytest.mark.parametrize("act,layer", [("relu2", False), ("gelu", True), ("silu", True)])
def test_mlp_gradients_against_differences(cuda_device, act, layer):
    """Central differences of the fp32 MLP along the gradient's signs. With steps of 1e-2 over
    smooth arguments of order one the third-order term is some 1e-4 of the derivative; the squared
    ReLU's jump of its second derivative adds h times the share of arguments within a step of 0."""
    t = mlp_tensors(6, 40, 48, 96, FP32, layer, True)
    got = run_mlp(t, act, layer)
    for name in NAMES:
        if t[name] is None:
            continue
        way, h = torch.sign(got[name]), 1e-2 / (1 if name not in ("w1", "w2") else 8)

        def f(s):
            a = {**t, name: t[name] + s * way}
            out = fused_mlp(a["x"], a["w1"], a["w2"], a["b1"], a["b2"], norm="layer" if layer else "rms",
                            norm_weight=a["norm_weight"], norm_bias=a["norm_bias"], activation=act)
            return float((out.double() * t["grad"].double()).sum())

        diff, want = (f(h) - f(-h)) / (2 * h), float(got[name].abs().double().sum())
        assert abs(diff - want) <= 1e-2 * want, (name, diff, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("m", [1, 200])
def test_capture_and_replay(cuda_device, m, dtype):
    from test_capture import _capture, _replays

    cases = []
    for s in (1, 2, 3):
        t = mlp_tensors(s, m, 136, 400, dtype, True, True)
        cases.append([t[a] for a in (*NAMES, "grad")])
    static = [v.clone() for v in cases[0]]

    def go(v):
        got = run_mlp(dict(zip((*NAMES, "grad"), v)), "gelu", True)
        return list(got.values())

    graph, outs = _capture(lambda: go(static))
    _replays(graph, outs, static, cases[1:] + cases[:1], go)


@pytest.mark.gpu
def test_two_streams(cuda_device):
    t = mlp_tensors(9, 256, 264, 1000, BF16, False, True)
    want = run_mlp(t, "silu", False)
    torch.cuda.synchronize()
    got = []
    for s in [torch.cuda.Stream() for _ in range(2)] * 3:
        with torch.cuda.stream(s):
            got.append(run_mlp(t, "silu", False))
    torch.cuda.synchronize()
    assert all(torch.equal(g[a], want[a]) for g in got for a in want)


@pytest.mark.gpu
def test_autocast(cuda_device):
    """Products in autocast's type, norm and sum in x's, as the same layers of torch."""
    t = mlp_tensors(10, 50, 64, 128, FP32, True, True)
    leaves = {a: t[a].clone().requires_grad_(True) for a in NAMES}
    with torch.autocast("cuda", dtype=BF16):
        lin = fused_linear(t["x"], t["w1"], t["b1"], activation="gelu")
        out = fused_mlp(leaves["x"], leaves["w1"], leaves["w2"], leaves["b1"], leaves["b2"],
                        norm="layer", norm_weight=leaves["norm_weight"], norm_bias=leaves["norm_bias"],
                        activation="gelu")
    assert lin.dtype == BF16 and out.dtype == FP32
    half = {a: t[a].to(BF16) for a in ("x", "w1", "b1")}
    assert torch.equal(lin, fused_linear(half["x"], half["w1"], half["b1"], activation="gelu"))
    grads = dict(zip(NAMES, torch.autograd.grad(out, list(leaves.values()), t["grad"])))
    want = run_mlp(t, "gelu", True)
    for a in NAMES:
        assert grads[a].dtype == FP32
        # Roundings of 2^-8 each on a path of at most six.
        assert float((grads[a] - want[a]).norm() / want[a].norm()) < 6 * 2.0 ** -8, a
    assert float((out - want["out"]).norm() / want["out"].norm()) < 4 * 2.0 ** -8


# ---- the model --------------------------------------------------------------------------------
@pytest.mark.gpu
def test_a_block_computes_its_reference_mlp(cuda_device):
    """``mlp_activation="relu2"`` is the reference's MLP: same state dict, same function."""
    torch.manual_seed(0)
    plain = dabsn_amd.DABSNBlock(24, 32, 32, residual=True, mlp_ratio=2.0).cuda()
    torch.nn.init.normal_(plain.mlp_fc2.weight, std=0.2)
    fused = dabsn_amd.DABSNBlock(24, 32, 32, residual=True, mlp_ratio=2.0, mlp_activation="relu2").cuda()
    fused.load_state_dict(plain.state_dict())
    h = torch.randn(3, 20, 32, device=cuda_device)
    a, b = h.clone().requires_grad_(True), h.clone().requires_grad_(True)
    up = torch.randn_like(h)
    one, two = plain.forward_mlp(a), fused.forward_mlp(b)
    assert float((one - two).abs().max()) < 1e-5
    one.backward(up)
    two.backward(up)
    assert float((a.grad - b.grad).abs().max()) < 1e-5
    for (name, p), (_, q) in zip(plain.named_parameters(), fused.named_parameters()):
        assert (p.grad is None) == (q.grad is None), name
        if p.grad is not None:
            assert float((p.grad - q.grad).abs().max()) < 1e-4, name


@pytest.mark.gpu
@pytest.mark.parametrize("norm,act,bias", [("rms", "relu2", False), ("layer", "gelu", True)])
def test_a_model_trains_evaluates_and_remembers_with_it(cuda_device, norm, act, bias):
    torch.manual_seed(1)
    m = dabsn_amd.DABSNSequenceLM(50, 32, depth=2, residual=True, mlp_ratio=4.0, mlp_activation=act,
                                  mlp_norm=norm, mlp_bias=bias).cuda()
    for block in m.blocks:
        torch.nn.init.normal_(block.mlp_fc2.weight, std=0.1)
    ids = torch.randint(0, 50, (2, 24), device=cuda_device)
    loss = dabsn_amd.chunked_linear_cross_entropy(m.forward_hidden(ids)[:, :-1], m.readout.weight,
                                                  m.readout.bias, ids[:, 1:])
    loss.backward()
    for block in m.blocks:
        for p in (block.mlp_norm.weight, block.mlp_fc1.weight, block.mlp_fc2.weight):
            assert bool(torch.isfinite(p.grad).all()) and float(p.grad.abs().max()) > 0
        if bias:
            assert float(block.mlp_fc1.bias.grad.abs().max()) > 0
    m.eval()
    with torch.no_grad():
        full = m(ids)
        _, mem = dabsn_amd.forward_with_memory(m, ids[:, :23], extend=True)
        last, mem = dabsn_amd.forward_with_memory(m, ids[:, 23:], mem, extend=True)
    assert float((last[:, -1] - full[:, -1]).abs().max()) < 1e-3
    other = dabsn_amd.DABSNSequenceLM(50, 32, depth=2, residual=True, mlp_ratio=4.0).cuda()
    with pytest.raises(ValueError, match="mlp"):
        dabsn_amd.forward_with_memory(other, ids, mem)
