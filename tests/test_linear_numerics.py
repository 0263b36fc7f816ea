"""Accuracy of the linear layer and the MLP where bounds by magnitudes or norms would not see a loss."""

from __future__ import annotations

import math

import pytest
import torch

from dabsn_amd import fused_linear, fused_mlp
from test_linear import Val, activated, check_linear, run, tensors
from test_norm import U, within

BF16, FP32 = torch.bfloat16, torch.float32

# ---- slopes far from zero ---------------------------------------------------------------------
# GELU's slope is 2^-25 at -5.5 and 2^-39 at -7.7, SiLU's at -20.5 and -30.7.
TAILS = {"gelu": (-7.5, -4.5), "silu": (-30.0, -14.0)}


def _tail(act):
    z = torch.linspace(*TAILS[act], 4096).to(BF16)
    _, slope = activated(Val(z.cuda()), act)
    # Kept with 2^-11 of itself or 2^-39; GELU's fit 1.7e-5 of a term below half the slope there;
    # exp's argument (up to 30) u of itself off, some more operations.
    tol = (2.0 ** -11 + 2e-5 + 64 * U) * slope.v.abs() + 2.0 ** -39
    return z, slope.v, tol


@pytest.mark.gpu
@pytest.mark.parametrize("act", TAILS)
def test_gradients_of_tails(cuda_device, act):
    """Small slopes relative to themselves: through a product with one term, in the gradient's pass."""
    z, slope, tol = _tail(act)
    x = z.cuda()[:, None].requires_grad_(True)
    one = torch.ones(1, 1, device=cuda_device, dtype=BF16)
    (dx,) = torch.autograd.grad(fused_linear(x, one, activation=act), x, torch.ones_like(x))
    within(dx[:, 0], slope, tol + 2.0 ** -8 * (slope.abs() + tol))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 256])
@pytest.mark.parametrize("act", TAILS)
def test_gradients_of_tails_of_the_mlp(cuda_device, act, m):
    """The same in the products' epilogues: a first layer without weights, whose arguments are its bias."""
    z, slope, tol = _tail(act)
    f, h = z.numel(), 8
    x = torch.randn(m, h, device=cuda_device).to(BF16)
    b1 = z.cuda().requires_grad_(True)
    w1 = torch.zeros(f, h, device=cuda_device, dtype=BF16)
    w2 = torch.zeros(h, f, device=cuda_device, dtype=BF16)
    w2[0] = 1
    up = torch.zeros(m, h, device=cuda_device, dtype=BF16)
    up[:, 0] = 1
    (db,) = torch.autograd.grad(fused_mlp(x, w1, w2, b1, activation=act), b1, up)
    # All rows have the same dz, rounded to bf16; their number is a power of two.
    within(db / m, slope, tol + 2.0 ** -8 * (slope.abs() + tol))


# ---- GELU beside bf16 where its value or its slope cancels ------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 40, 300])
def test_a_residual_that_cancels_gelu(cuda_device, m):
    """The value is not rounded before the residual is added: what is left of it is right to fp32's
    bounds (an argument of one term, 8 u of the value and 2 u of the argument) and one rounding."""
    z = torch.linspace(-6, 6, 4096).to(BF16).cuda()
    h = activated(Val(z), "gelu")[0]
    res = (-h.v).to(BF16)
    x = torch.ones(m, 1, device=cuda_device, dtype=BF16)
    out = fused_linear(x, z[:, None], activation="gelu", residual=res.expand(m, -1))
    want = h.v + res.double()
    tol = h.e + U * want.abs() + 48 * U * h.v.abs()  # exp's argument, up to 18, u of itself off
    for row in out:
        within(row, want, tol + 2.0 ** -8 * (want.abs() + tol))


@pytest.mark.gpu
def test_gelus_slope_where_it_passes_zero(cuda_device):
    """-0.75 and a small bias: the slope's bound is of fp32, and 2^-11 and 2^-8 of its own small value."""
    b = torch.linspace(-0.01, 0.01, 2001).to(BF16).cuda().requires_grad_(True)
    x = torch.full((1, 1), -0.75, device=cuda_device, dtype=BF16)
    one = torch.ones(2001, 1, device=cuda_device, dtype=BF16)
    (db,) = torch.autograd.grad(fused_linear(x, one, b, activation="gelu"), b, torch.ones_like(b)[None])
    slope = activated(Val(b.detach().double() - 0.75), "gelu")[1]
    tol = slope.e + 2.0 ** -11 * slope.v.abs() + 2.0 ** -39
    within(db, slope.v, tol + 2.0 ** -8 * (slope.v.abs() + tol))


# ---- infinities and NaN -----------------------------------------------------------------------
def _same_kind(name, got, want):
    """NaN where NaN, infinite where infinite, and finite elsewhere."""
    got, want = got.double(), want.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), name
    odd = torch.isinf(want)
    assert torch.equal(torch.isinf(got), odd) and torch.equal(got[odd], want[odd]), name


def _mixed(g, *shape):
    """Values that one bf16 holds whole, zeros among them, and values that take three."""
    v = torch.randn(*shape, device="cuda", generator=g)
    v[::2] = torch.randint(-2, 3, v[::2].shape, device="cuda", generator=g).float()
    return v


# Products of planes in tiles of 256 x 256 (the last in splits) and of fp32 as it lies.
KINDS = [(40, 64, 40), (4001, 1000, 3999), (2049, 9001, 2050)]


@pytest.mark.gpu
@pytest.mark.parametrize("act,residual", [("relu2", False), ("relu2", True), ("gelu", True), ("silu", False)])
@pytest.mark.parametrize("m,k,n", KINDS)
def test_infinities_through_activations(cuda_device, m, k, n, act, residual):
    g = torch.Generator(device=cuda_device).manual_seed(m)
    x, w, grad = torch.randn(m, k, device=cuda_device, generator=g), _mixed(g, n, k) / 8, _mixed(g, m, n)
    x[3, k - 1], x[m - 1, 0], x[7, 1], x[7, 2], x[9, 5] = math.inf, -math.inf, math.inf, -math.inf, math.nan
    b, res = 0.1 * torch.randn(n, device=cuda_device, generator=g), None
    if residual:
        res = torch.randn(m, n, device=cuda_device, generator=g)
        res[3, ::3], res[5, 5] = -math.inf, math.inf
    leaves = [t.requires_grad_(True) for t in (x, w, b, *((res,) if residual else ()))]
    out = fused_linear(x, w, b, activation=act, residual=res)
    dx, dw, db = torch.autograd.grad(out, leaves, grad)[:3]
    z = Val(x).v @ Val(w).v.t() + b.detach().double()
    h, slope = activated(Val(z), act)
    _same_kind("out", out.detach(), h.v if res is None else h.v + res.detach().double())
    dz = grad.double() * slope.v
    _same_kind("x", dx, dz @ w.detach().double())
    _same_kind("weight", dw, dz.t() @ x.detach().double())
    _same_kind("bias", db, dz.sum(0))


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["relu2", "gelu"])
@pytest.mark.parametrize("m,h,f", [(40, 24, 61), (4001, 1000, 3999), (300, 2048, 4100), (6000, 256, 1024)])
def test_infinite_gradients_through_the_mlps_slopes(cuda_device, m, h, f, act):
    """An infinite gradient times the second layer times the slope, seen in the first layer's bias; an
    infinite inner value through the second product and the residual."""
    g = torch.Generator(device=cuda_device).manual_seed(m)
    x, w1 = torch.randn(m, h, device=cuda_device, generator=g), torch.randn(f, h, device=cuda_device, generator=g)
    w1, w2, up = w1 / math.sqrt(h), _mixed(g, h, f) / 8, torch.randn(m, h, device=cuda_device, generator=g)
    up[2, 4], up[m - 1, h - 1], up[5, 3], up[5, 6] = math.inf, -math.inf, math.inf, math.inf
    b1 = (0.1 * torch.randn(f, device=cuda_device, generator=g)).requires_grad_(True)
    (db,) = torch.autograd.grad(fused_mlp(x, w1, w2, b1, activation=act), b1, up)
    X, W1, W2 = x.double(), w1.double(), w2.double()
    z = (X / (X.square().mean(1, keepdim=True) + 1e-6).sqrt()) @ W1.t()
    _, slope = activated(Val(z + b1.detach().double()), act)
    _same_kind("b1", db, ((up.double() @ W2) * slope.v).sum(0))
    with torch.no_grad():
        b1[f // 2], x[4, 1] = 1e30, math.inf  # one column of infinities where squared, and a row of NaN
        out = fused_mlp(x, w1, w2, b1, activation=act)
        X = x.double()
        z = (X / (X.square().mean(1, keepdim=True) + 1e-6).sqrt()) @ W1.t() + b1.double()
        hidden = activated(Val(z), act)[0].v.float().double()  # 1e60 is infinite in fp32
        _same_kind("out", out, X + hidden @ W2.t())


@pytest.mark.gpu
@pytest.mark.parametrize("value", [math.inf, math.nan])
@pytest.mark.parametrize("m,k,n", [(2048, 1024, 2048), (4096, 2048, 4096)])
def test_results_without_a_finite_one_take_no_age(cuda_device, m, k, n, value):
    """All results infinite or NaN (a training step that has run off): forming them anew by fp32 matrix
    instructions takes 1.5 times the planes' time again by their rates, and what the loads' latency adds
    (measured 2.4 and 4.2 times in all); elements one by one, as it was, took 67 and 180 times."""
    x = torch.randn(m, k, device=cuda_device)
    w = torch.randn(n, k, device=cuda_device)

    def fastest():
        times = []
        for _ in range(4):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            fused_linear(x, w)
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)

    finite = fastest()
    x[:, k // 3] = value
    assert fastest() < 15 * finite
    _same_kind("out", fused_linear(x, w), x.double() @ w.double().t())


# ---- fp32 as planes ---------------------------------------------------------------------------
# Six products of bf16 planes (hi, mid, lo) make an fp32 one. Bounds by the terms' magnitudes grow with
# their number n beyond what a missing product would change (2.4e-6 of the result in the norm for lo hi
# and hi lo, 2.8e-6 for mid mid, at any n). In the norm, sums of n products in at most n / 8
# additions, whose partial sums grow as the root of their number and whose roundings of at most u = 2^-24
# have independent signs, are off by u sqrt(n / 8 / 6) or less, and their last rounding by u / sqrt(3);
# what the planes leave out is 6e-9.
def _norm_bound(n):
    return U * (1 + 2 * math.sqrt(n / 48))


def _off(got, want):
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.parametrize("n", [300, 4001])
def test_the_bound_sees_a_missing_product_of_planes(n):
    g = torch.Generator().manual_seed(n)
    a, b = torch.randn(150, n, generator=g), torch.randn(130, n, generator=g)

    def planes(rest):
        for _ in range(3):
            part = rest.to(BF16).float()
            yield part.double()
            rest = rest - part

    pa, pb = list(planes(a)), list(planes(b))
    want = a.double() @ b.double().t()
    pairs = [(2, 0), (0, 2), (1, 1), (1, 0), (0, 1), (0, 0)]
    products = {p: pa[p[0]] @ pb[p[1]].t() for p in pairs}
    whole = sum(products.values())
    assert _off(whole, want) < 1e-8
    for p in pairs:
        assert _off(whole - products[p], want) > _norm_bound(n), p


# Between them these take 256 x 256 and 128 x 128 tiles of planes, split and whole, in all three
# directions.
PLANES = [(515, 1500, 4001), (4001, 777, 1001), (1001, 2050, 2050), (300, 2050, 4001), (2050, 300, 4001),
          (2050, 4001, 300)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", PLANES)
def test_fp32_products_hold_24_bits(cuda_device, m, k, n):
    t = tensors(m + k + n, m, k, n, FP32, False, False)
    got = run(t, "none")
    x, w, g = (t[a].double() for a in ("x", "weight", "grad"))
    for name, want, terms in (("out", x @ w.t(), k), ("x", g @ w, n), ("weight", g.t() @ x, m)):
        assert _off(got[name], want) <= _norm_bound(terms), name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_all_gradients_of_strided_operands(cuda_device, dtype):
    """256 x 256 tiles on rows inside wider arrays of NaN at odd offsets. fp32 operands are packed into
    planes wherever they lie: the contiguous ones' results, bit for bit."""
    m, k, n = 4001, 1000, 3999
    t = tensors(1, m, k, n, dtype, True, True)
    view = {}
    for a in ("x", "weight", "residual", "grad"):
        wide = torch.full((t[a].shape[0], t[a].shape[1] + 5), math.nan, device=cuda_device, dtype=dtype)
        wide[:, 3:-2] = t[a]
        view[a] = wide[:, 3:-2]
    leaves = {a: v.requires_grad_(True) for a, v in view.items() if a != "grad"}
    leaves["bias"] = t["bias"].clone().requires_grad_(True)
    out = fused_linear(leaves["x"], leaves["weight"], leaves["bias"], activation="silu",
                       residual=leaves["residual"])
    grads = torch.autograd.grad(out, tuple(leaves.values()), view["grad"])
    got = {"out": out.detach(), **dict(zip(leaves, grads))}
    check_linear(t, "silu", got)
    want = run(t, "silu")
    same = want if dtype == FP32 else ("bias", "residual")
    assert all(torch.equal(got[a], want[a]) for a in same)


# ---- what the branch's backward hands on ------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("m,h,f", [(1, 8, 300), (40, 24, 61), (300, 77, 5000), (300, 512, 8192), (4001, 1000, 3999)])
def test_the_normed_rows_gradient_is_not_rounded(cuda_device, m, h, f):
    """Whole numbers throughout: dz = g W2 (|dz| < 256) is exact in bf16, its product with W1 in fp32, and
    so are that one's sums over the rows, the norm's bias in fp32. A rounding of the product to 8 bits
    would show."""
    g = torch.Generator(device=cuda_device).manual_seed(m + f)

    def whole(most, *shape):
        return torch.randint(-most, most + 1, shape, device=cuda_device, generator=g).to(BF16)

    x, up, w1, w2 = torch.randn(m, h, device=cuda_device).to(BF16), whole(1, m, h), whole(2, f, h), whole(1, h, f)
    nb = torch.zeros(h, device=cuda_device, requires_grad=True)
    nw = torch.ones(h, device=cuda_device)
    out = fused_mlp(x, w1, w2, norm="layer", norm_weight=nw, norm_bias=nb, activation="none")
    (db,) = torch.autograd.grad(out, nb, up)
    dz = up.double() @ w2.double()
    assert float(dz.abs().max()) <= 256
    dn = dz @ w1.double()
    assert float(dn.abs().sum(0).max()) < 2 ** 24
    assert f < 1000 or bool((dn.to(BF16).double() != dn).any())  # sums of a few hundred terms have 8 bits
    assert torch.equal(db.double(), dn.sum(0))
