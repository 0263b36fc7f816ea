"""Layer norm and RMS norm against the definition in 64 bits, values and gradients.

u = 2^-24, D = 96 bounds the additions on any path of a row's sum (64 values a thread at most, 6
steps of a wave, 16 waves, and a few operations around them). A mean is off by D u mean|x|; the
deviations x - mean by that and u of themselves; 1 / std by (D / 2 + 8) u of itself (the mean's
error enters the variance squared). So with v = (x - mean) / std

  |error of v| <= (D u mean|x| / std) + (D / 2 + 9) u |v|                                   = e
  |error of y| <= |w| e + 3 u (|v w| + |b|) + rounding |y|
  |error of dx| <= (u (D + 6) (|gw| + mean|gw| + |v| mean|gw v|) + |v| mean(|gw| e) + e |mean(gw v)|)
                   / std + (D / 2 + 12) u |dx| + rounding |dx|
  |error of dw| <= sum |g| e + rows u sum |g v| + rounding |dw|,  db without e

(the sums over the rows have fewer than ``rows`` + 40 additions on a path). Roundings are at most
half a step, eps / 2 of the type: 2^-24 in fp32, 2^-8 in bf16."""

from __future__ import annotations

import math

import pytest
import torch

import dabsn_amd
from dabsn_amd import layer_norm, rms_norm

U, D = 2.0 ** -24, 96


def _cpu(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("call,error,match", [
    (lambda: layer_norm(_cpu(3, 4, dtype=torch.float16)), TypeError, "float32 or bfloat16"),
    (lambda: layer_norm(torch.zeros(3, 4).double()), TypeError, "float32 or bfloat16"),
    (lambda: layer_norm(torch.zeros(())), ValueError, "expected x"),
    (lambda: layer_norm(_cpu(3, 0)), ValueError, "expected x"),
    (lambda: rms_norm(_cpu(1, 16385)), ValueError, "expected x"),
    (lambda: layer_norm(_cpu(3, 4), _cpu(5)), ValueError, "weight"),
    (lambda: layer_norm(_cpu(3, 4), _cpu(4), _cpu(3)), ValueError, "bias"),
    (lambda: layer_norm(_cpu(3, 4), _cpu(4, dtype=torch.bfloat16)), TypeError, "weight"),
    (lambda: layer_norm(_cpu(3, 4, dtype=torch.bfloat16), _cpu(4), _cpu(4, dtype=torch.bfloat16)),
     TypeError, "bias"),
    (lambda: layer_norm(_cpu(3, 4), eps=-1.0), ValueError, "eps"),
    (lambda: rms_norm(_cpu(3, 4), eps=math.nan), ValueError, "eps"),
    (lambda: rms_norm(_cpu(3, 4), _cpu(4)), RuntimeError, "device"),
])
def test_refusals(call, error, match):
    with pytest.raises(error, match=match):
        call()


def test_library_refuses_bad_arguments_before_it_launches():
    from dabsn_amd import _lib

    lib, one = _lib.load(), 1 << 20
    for dtype, wdtype, rows, h, ld in ((2, 2, 1, 4, 4), (0, 1, 1, 4, 4), (0, 0, -1, 4, 4),
                                       (0, 0, 1, 0, 4), (0, 0, 1, 16385, 16385), (0, 0, 1, 4, 3),
                                       (0, 0, 1 << 31, 4, 4)):
        assert lib.dabsn_hip_norm_fwd(dtype, wdtype, 1, rows, h, one, ld, one, one, 1e-5, one, one, None) == -2
        assert lib.dabsn_hip_norm_bwd(dtype, wdtype, 1, rows, h, one, ld, one, one, one, ld, None, one,
                                      one, one, one, 1 << 40, None) == -2
    assert lib.dabsn_hip_norm_fwd(0, 0, 1, 1, 4, None, 4, one, one, 1e-5, one, one, None) == -2
    assert lib.dabsn_hip_norm_fwd(0, 0, 1, 1, 4, one, 4, one, one, -1.0, one, one, None) == -2
    need = lib.dabsn_hip_norm_workspace_bytes(0, 100, 64)
    assert need > 0 and lib.dabsn_hip_norm_workspace_bytes(0, -1, 64) == 0
    assert lib.dabsn_hip_norm_bwd(0, 0, 1, 100, 64, one, 64, one, one, one, 64, None, one, one, one, one,
                                  need - 1, None) == -2


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def case(seed, rows, h, dtype, wdtype, layer, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, h, generator=g) * (0.5 + torch.rand(rows, 1, generator=g)) + shift
    w = 1 + 0.3 * torch.randn(h, generator=g)
    b = 0.3 * torch.randn(h, generator=g) if layer else None
    grad = torch.randn(rows, h, generator=g)
    move = lambda t, d: None if t is None else t.to(d).cuda()  # noqa: E731
    return move(x, dtype), move(w, wdtype), move(b, wdtype), move(grad, dtype)


def check(x, w, b, grad, eps, layer, out, dx, dw, db, add=None):
    """Results against the definition in 64 bits, within the module's bounds."""
    rnd = half_step(x.dtype)
    X, G = x.detach().double(), grad.double()
    W = torch.ones_like(X[0]) if w is None else w.detach().double()
    mean = X.mean(1, keepdim=True) if layer else 0.0
    std = ((X - mean).square().mean(1, keepdim=True) + eps).sqrt()
    v = (X - mean) / std
    e = (D / 2 + 9) * U * v.abs()
    if layer:
        e = e + D * U * X.abs().mean(1, keepdim=True) / std
    y = v * W if b is None else v * W + b.detach().double()
    tol = W.abs() * e + 3 * U * ((v * W).abs() + (0 if b is None else b.detach().double().abs()))
    within(out, y, tol + rnd * (y.abs() + tol))
    if dx is None:
        return
    gw = G * W
    s1 = gw.mean(1, keepdim=True) if layer else torch.zeros_like(std)
    s2 = (gw * v).mean(1, keepdim=True)
    want = (gw - s1 - v * s2) / std
    m1 = gw.abs().mean(1, keepdim=True) if layer else 0.0
    tol = (U * (D + 6) * (gw.abs() + m1 + v.abs() * (gw * v).abs().mean(1, keepdim=True))
           + v.abs() * (gw.abs() * e).mean(1, keepdim=True) + e * s2.abs()) / std
    tol = tol + (D / 2 + 12) * U * want.abs()
    if add is not None:
        want = want + add.double()
        tol = tol + U * want.abs()
    within(dx, want, tol + rnd * (want.abs() + tol))
    n = X.shape[0] + 40
    for got, terms, more in ((dw, G * v, (G.abs() * e).sum(0)), (db, G, 0.0)):
        if got is not None:
            ref = terms.sum(0)
            tol = more + n * U * terms.abs().sum(0)
            within(got, ref, tol + half_step(got.dtype) * (ref.abs() + tol))  # its own type's step


def within(got, want, tol):
    bad = (got.detach().double() - want).abs() - (tol + 2.0 ** -126)
    assert not bool(torch.isnan(got).any()) and float(bad.max() if bad.numel() else 0) <= 0, float(bad.max())


def run(x, w, b, grad, layer, eps):
    leaves = [t.detach().clone().requires_grad_(True) if t is not None else None for t in (x, w, b)]
    out = layer_norm(*leaves, eps=eps) if layer else rms_norm(leaves[0], leaves[1], eps=eps)
    real = [t for t in leaves if t is not None]
    grads = iter(torch.autograd.grad(out, real, grad))
    return [out.detach()] + [None if t is None else next(grads) for t in leaves]


# Every width class of the kernels (lanes by vectors), both sides of its border, odd widths.
SIZES = [(1, 1), (1, 2048), (2, 7), (5, 63), (4, 64), (9, 256), (130, 257), (33, 512), (2000, 511),
         (1030, 1001), (1024, 1024), (1025, 1024), (17, 2047), (1100, 2048), (3, 2049), (6, 4096),
         (40, 4097), (5, 8192), (3, 8193), (2, 16384), (4099, 40), (5000, 3)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,wdtype", [(torch.float32, torch.float32),
                                          (torch.bfloat16, torch.bfloat16),
                                          (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("layer", [True, False])
@pytest.mark.parametrize("rows,h", SIZES)
def test_values_and_gradients(cuda_device, rows, h, layer, dtype, wdtype):
    eps = 1e-5 if layer else 1e-6
    x, w, b, grad = case(rows + h, rows, h, dtype, wdtype, layer)
    got = run(x, w, b, grad, layer, eps)
    check(x, w, b, grad, eps, layer, *got)
    assert got[1].dtype == dtype and got[2].dtype == wdtype
    again = run(x, w, b, grad, layer, eps)
    assert all(a is None or torch.equal(a, c) for a, c in zip(got, again))
    with torch.no_grad():
        plain = layer_norm(x, w, b, eps=eps) if layer else rms_norm(x, w, eps=eps)
    assert torch.equal(plain, got[0])


@pytest.mark.gpu
@pytest.mark.parametrize("layer", [True, False])
def test_difficult_rows(cuda_device, layer):
    """A mean far above the spread, rows of one value, rows of zeros, tiny and large rows."""
    x, w, b, grad = case(5, 64, 300, torch.float32, torch.float32, layer, shift=200.0)
    check(x, w, b, grad, 1e-5, layer, *run(x, w, b, grad, layer, 1e-5))
    x[3], x[4], x[5], x[6] = 0.0, 7.5, x[5] * 1e-12, x[6] * 1e12
    check(x, w, b, grad, 1e-5, layer, *run(x, w, b, grad, layer, 1e-5))


@pytest.mark.gpu
def test_a_row_of_nan_or_infinity_stays_alone(cuda_device):
    x, w, b, grad = case(6, 40, 700, torch.float32, torch.float32, True)
    want = run(x, w, b, grad, True, 1e-5)
    x[7, 3], x[11, 699], x[39, 0] = math.nan, math.inf, -math.inf
    got = run(x, w, b, grad, True, 1e-5)
    keep = torch.ones(40, dtype=torch.bool)
    keep[[7, 11, 39]] = False
    for a, c in ((got[0], want[0]), (got[1], want[1])):
        assert torch.equal(a[keep], c[keep]) and bool(torch.isnan(a[~keep]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_shapes_strides_and_absent_tensors(cuda_device, dtype):
    x, w, b, grad = case(7, 60, 203, dtype, dtype, True)
    want = run(x, w, b, grad, True, 1e-5)
    wide = torch.full((60, 211), math.nan, device=cuda_device, dtype=dtype)
    wide[:, 5:208] = x
    wide_grad = torch.full((60, 219), math.nan, device=cuda_device, dtype=dtype)
    wide_grad[:, 3:206] = grad
    leaf = wide.requires_grad_(True)
    out = layer_norm(leaf[:, 5:208], w, b)
    (g,) = torch.autograd.grad(out, leaf, wide_grad[:, 3:206])
    assert torch.equal(out.detach(), want[0]) and torch.equal(g[:, 5:208], want[1])
    tall = x.t().contiguous().t()
    assert torch.equal(layer_norm(tall, w, b), want[0])
    cube = layer_norm(x.view(3, 20, 203), w, b)
    assert cube.shape == (3, 20, 203) and torch.equal(cube.view(60, 203), want[0])
    assert torch.equal(layer_norm(x[9], w, b), want[0][9])
    # An expanded upstream gradient, and one that is not contiguous.
    leaf = x.clone().requires_grad_(True)
    up = grad[:1].expand(60, 203)
    (g,) = torch.autograd.grad(layer_norm(leaf, w, b), leaf, up)
    check(x, w, b, up, 1e-5, True, want[0], g, None, None)
    for weight, bias in ((None, None), (w, None), (None, b)):
        leaves = [t.clone().requires_grad_(True) for t in (x, weight, bias) if t is not None]
        at = iter(leaves)
        args = [next(at) if t is not None else None for t in (x, weight, bias)]
        out = layer_norm(*args)
        grads = dict(zip(map(id, leaves), torch.autograd.grad(out, leaves, grad)))
        check(x, weight, bias, grad, 1e-5, True, out, *(grads.get(id(a)) for a in args))
    # Only one gradient wanted; the weight shared by two calls.
    leaf = w.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(layer_norm(x, leaf, b), leaf, grad)
    assert torch.equal(g, want[2])
    leaf = w.clone().requires_grad_(True)
    both = rms_norm(x[:30], leaf) + rms_norm(x[30:], leaf)
    assert torch.autograd.grad(both, leaf, grad[:30])[0].shape == (203,)


@pytest.mark.gpu
def test_no_rows(cuda_device):
    for dtype in (torch.float32, torch.bfloat16):
        x, w, b, grad = case(8, 0, 41, dtype, dtype, True)
        out, dx, dw, db = run(x, w, b, grad, True, 1e-5)
        assert out.shape == dx.shape == (0, 41)
        assert float(dw.float().abs().sum() + db.float().abs().sum()) == 0


@pytest.mark.gpu
def test_long_inputs(cuda_device):
    """More than 2^31 elements: rows past 32-bit offsets."""
    rows, h = 530_000, 4096
    x = torch.empty(rows, h, device=cuda_device, dtype=torch.bfloat16)
    x.normal_(generator=torch.Generator(device=cuda_device).manual_seed(1))
    w = torch.ones(h, device=cuda_device, dtype=torch.bfloat16, requires_grad=True)
    leaf = x.requires_grad_(True)
    out = rms_norm(leaf, w)
    dx, dw = torch.autograd.grad(out, (leaf, w), x.detach())
    for s in (0, rows - 3):
        part = x.detach()[s:s + 3]
        check(part, w, None, part, 1e-6, False, out[s:s + 3], dx[s:s + 3], None, None)
    ref = torch.zeros(h, device=cuda_device, dtype=torch.float64)
    for s in range(0, rows, 53_000):
        part = x.detach()[s:s + 53_000].double()
        term = part * part / (part.square().mean(1, keepdim=True) + 1e-6).sqrt()
        ref += term.sum(0)
    # At most 691 rows a partial sum, 64 partial sums a slot and 16 slots, each addition u of the sum.
    within(dw, ref, (2 ** -8 + (D + 780) * U) * ref)  # the terms are positive


@pytest.mark.gpu
def test_gradients_against_differences(cuda_device):
    """Directional derivatives of the operators by central differences, in steps that keep the
    third-order term h^2 / 6 f''' and the rounding u |f| / h both below 2e-3 of the derivative."""
    x, w, b, grad = case(9, 12, 96, torch.float32, torch.float32, True)
    for layer in (True, False):
        _, dx, dw, db = run(x, w, b if layer else None, grad, layer, 1e-5)
        for at, d in (("x", dx), ("w", dw), ("b", db)):
            if d is None:
                continue
            way = torch.sign(d)  # the derivative along it is sum|d|: nothing cancels
            h = 1e-2

            def f(s):
                args = {"x": x, "w": w, "b": b}
                args[at] = args[at] + s * way
                out = layer_norm(args["x"], args["w"], args["b"], eps=1e-5) if layer else \
                    rms_norm(args["x"], args["w"], eps=1e-5)
                return float((out.double() * grad.double()).sum())

            got, want = (f(h) - f(-h)) / (2 * h), float(d.abs().double().sum())
            assert abs(got - want) <= 4e-3 * want, (at, got, want)


@pytest.mark.gpu
def test_no_second_derivative(cuda_device):
    x = torch.randn(4, 8, device=cuda_device, requires_grad=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(layer_norm(x).sum(), x, create_graph=True)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,h", [(1, 2048), (700, 333), (64, 5000)])
def test_capture_and_replay(cuda_device, rows, h):
    from test_capture import _capture, _replays

    cases = [case(s, rows, h, torch.bfloat16, torch.bfloat16, True) for s in (1, 2, 3)]
    static = [v.clone() for v in cases[0]]

    def go(v):
        leaves = [t.detach().requires_grad_(True) for t in v[:3]]
        out = layer_norm(*leaves)
        return [out.detach(), *torch.autograd.grad(out, leaves, v[3])]

    graph, outs = _capture(lambda: go(static))
    _replays(graph, outs, static, cases[1:] + cases[:1], go)


@pytest.mark.gpu
def test_two_streams(cuda_device):
    x, w, b, grad = case(11, 20000, 300, torch.float32, torch.float32, True)
    want = run(x, w, b, grad, True, 1e-5)
    torch.cuda.synchronize()
    got = []
    for s in [torch.cuda.Stream() for _ in range(2)] * 2:
        with torch.cuda.stream(s):
            got.append(run(x, w, b, grad, True, 1e-5))
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for g in got for a, c in zip(g, want))


@pytest.mark.gpu
def test_against_the_blocks_norm(cuda_device):
    """The module's norm rounds before the weight; the operator once: within two roundings."""
    from dabsn_amd.model import MLPRMSNorm

    x, w, _, _ = case(12, 50, 96, torch.bfloat16, torch.bfloat16, False)
    m = MLPRMSNorm(96).cuda().to(torch.bfloat16)
    m.weight.data.copy_(w)
    want = m(x).double()
    assert bool(((rms_norm(x, w).double() - want).abs() <= 3 * 2.0 ** -8 * want.abs() + 1e-30).all())
    assert dabsn_amd.rms_norm is rms_norm
