"""Token log probabilities, entropy and top alternatives against the definition in 64 bits.

Tolerances, u = 2^-24 (half a step of fp32): a row's exp-sum takes at most V / 64 additions a
thread and some 20 to join them, each an error of u; the exponent's argument carries three
roundings of itself, so a term e^-a an error of 3 a u, and these weighted by the terms are at
most 3 ln V u for terms that matter; the exponential and the logarithm an ulp (2 u) each. With
S = V / 64 + 64 + 3 ln V the sum's relative error is at most S u. A log probability is
(x - m) / T - ln s: 3 u of its first part, 2 u of its second, S u and its own rounding:
u (4 |z - max z| + 4 ln V + S). The entropy is ln s - U / s with U the sum of e (x - m): the same
errors once more on U / s, at most ln V: u (S (1 + 2 ln V) + 8 ln V). A gradient's dense part is
p times a factor of magnitude F = sum |g| + |g_H| (|logp| + H + 1) (1: logp and H hold ln s, and
a relative error S u of s is an absolute one of its logarithm, also where both are 0 as for one
word): u p F (2 S + 3 |arg| + 16), |arg| <= 104 where p is not 0; at a target or an alternative 4 u |g| more, all over T; then one
rounding to the logits' type (u, or 2^-8 for bf16).
"""

from __future__ import annotations

import math

import pytest
import torch

import dabsn_amd
from dabsn_amd import chunked_linear_token_logprobs, token_logprobs
from dabsn_amd.kernels import check_errors

U = 2.0 ** -24
INF = math.inf


# ---- refusals (no GPU) -----------------------------------------------------------------------
@pytest.mark.parametrize("call,error,match", [
    (lambda: token_logprobs(torch.zeros(2, 5).half(), torch.zeros(2).long()), TypeError, "float32 or"),
    (lambda: token_logprobs(torch.zeros(2, 5), torch.zeros(3).long()), ValueError, "does not match"),
    (lambda: token_logprobs(torch.zeros(2, 5), torch.zeros(2)), TypeError, "int64 or int32"),
    (lambda: token_logprobs(torch.zeros(2, 5), top=6), ValueError, "top must lie"),
    (lambda: token_logprobs(torch.zeros(2, 500), top=129), ValueError, "top must lie"),
    (lambda: token_logprobs(torch.zeros(2, 5), top=-1), ValueError, "top must lie"),
    (lambda: token_logprobs(torch.zeros(2, 0)), ValueError, "vocabulary"),
    (lambda: token_logprobs(torch.tensor(1.0)), ValueError, "logits"),
    (lambda: token_logprobs(torch.zeros(2, 5), temperature=0.0), ValueError, "temperature"),
    (lambda: token_logprobs(torch.zeros(2, 5), temperature=-1.0), ValueError, "temperature"),
    (lambda: token_logprobs(torch.zeros(2, 5), temperature=math.nan), ValueError, "temperature"),
    (lambda: token_logprobs(torch.zeros(2, 5)), RuntimeError, "device tensors"),
    (lambda: chunked_linear_token_logprobs(torch.zeros(2, 3), torch.zeros(5, 4), None), ValueError,
     "do not match"),
    (lambda: chunked_linear_token_logprobs(torch.zeros(2, 3), torch.zeros(5, 3), torch.zeros(4)),
     ValueError, "bias"),
    (lambda: chunked_linear_token_logprobs(torch.zeros(2, 3), torch.zeros(5, 3).bfloat16(), None),
     TypeError, "share a type"),
    (lambda: chunked_linear_token_logprobs(torch.zeros(2, 3), torch.zeros(5, 3), None),
     RuntimeError, "device tensors"),
])
def test_refusals(call, error, match):
    with pytest.raises(error, match=match):
        call()


def test_library_refuses_bad_arguments_before_it_launches():
    from dabsn_amd import _lib

    lib = _lib.load()
    one = 1 << 20  # never read: every call is refused by its sizes
    fwd = lambda dtype=0, rows=2, V=5, ld=5, bias=None, t=1.0, top=0: (  # noqa: E731
        lib.dabsn_hip_token_logprobs(dtype, rows, V, one, ld, bias, one, -100, t, top, one, one, one,
                                     one, one, one, None))
    for kw in (dict(dtype=2), dict(rows=-1), dict(V=0), dict(ld=4), dict(t=0.0), dict(top=6),
               dict(top=129, V=500, ld=500), dict(dtype=1, bias=one), dict(V=(1 << 31), ld=1 << 31)):
        assert fwd(**kw) == -2, kw
    assert lib.dabsn_hip_token_logprobs(0, 2, 5, None, 5, None, one, -100, 1.0, 0, one, one, one, one,
                                        one, one, None) == -2
    bwd = lambda dtype=0, ldo=5, plane=0, top=0: lib.dabsn_hip_token_logprobs_bwd(  # noqa: E731
        dtype, 2, 5, one, 5, None, one, -100, 1.0, top, one, one, one, one, one, one, one, ldo, plane,
        None)
    for kw in (dict(ldo=4), dict(plane=9), dict(dtype=1, plane=16), dict(top=6)):
        assert bwd(**kw) == -2, kw
    assert lib.dabsn_hip_column_sums(0, 4, 10, 12, one, 0, one, one, None) == -2  # stride not of 8
    assert lib.dabsn_hip_scaled(3, 4, one, one, None, None, 1.0, one, None) == -2
    assert lib.dabsn_hip_half_copy(4, one + 2, one, one, one, None) == -2  # not aligned


# ---- the definition in 64 bits ---------------------------------------------------------------
def reference(x, targets, top, T, ignore=-100):
    """(logprobs, entropy, top log probabilities, top indices, z, p, logp) of x [rows, V]."""
    x = x.detach().double().cpu()
    z = x / T
    m = z.amax(1, keepdim=True)
    empty = m == -INF
    m = torch.where(empty, 0.0, m)
    s = torch.exp(z - m).sum(1, keepdim=True)
    logp = torch.where(empty, -INF, z - m - torch.log(torch.where(empty, 1.0, s)))
    logp = torch.where(torch.isnan(s), math.nan, logp)
    p = logp.exp()
    ent = -torch.where(p > 0, p * logp, 0.0 * p).sum(1)
    ent = torch.where(empty[:, 0], 0.0, ent)
    lp = None
    if targets is not None:
        t = targets.cpu().long()
        ok = t != ignore
        lp = torch.where(ok, logp.gather(1, t.clamp(min=0)[:, None])[:, 0], 0.0)
    tl = ti = None
    if top:
        order = torch.where(torch.isnan(x), -INF, x) + 0.0  # NaN with -inf; -0 is 0
        ti = order.sort(dim=1, descending=True, stable=True).indices[:, :top]
        tl = logp.gather(1, ti)
    return lp, ent, tl, ti, z, p, logp


def sum_error(V):
    return V / 64 + 64 + 3 * math.log(V)


def check_forward(got, x, targets, top, T):
    lp, ent, tl, ti, _, _, _ = reference(x, targets, top, T)
    V, S = x.shape[1], sum_error(x.shape[1])
    ln = math.log(V)

    def close(a, b, tol):
        a, b = a.double().cpu().reshape(b.shape), b.float().double()  # beyond fp32's range: inf
        same = (a == b) | (torch.isnan(a) & torch.isnan(b))
        bad = ~same & ~((a - b).abs() <= tol)
        assert not bool(bad.any()), (float((a - b).abs()[bad].max()), V)

    # |z - max z| <= |log p| + ln V, and the result's own rounding
    spread = lambda b: U * (5 * b.abs().nan_to_num(0, 0, 0) + 8 * ln + S)  # noqa: E731
    if lp is not None:
        assert got.logprobs.dtype == torch.float32
        close(got.logprobs, lp, spread(lp))
    close(got.entropy, ent, U * (S * (1 + 2 * ln) + 8 * ln))
    if top:
        assert torch.equal(got.top_indices.cpu().reshape(ti.shape), ti)
        close(got.top_logprobs, tl, spread(tl))


def logits_of(seed, rows, V, dtype, spread=3.0, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, V, generator=g) * spread).to(dtype)
    t = torch.randint(0, V, (rows,), generator=g)
    t[::5] = -100
    return x.to(device), t.to(device)


SIZES = [(1, 1, 1), (3, 2, 2), (5, 7, 3), (4, 8, 8), (17, 16, 16), (33, 60, 5), (18, 64, 64), (700, 65, 20),
         (19, 128, 128), (19, 129, 100), (9, 1024, 128), (9, 1025, 128),
         (3, 1023, 127), (5, 2049, 5), (3, 4099, 33), (2, 8192, 1), (600, 9001, 7), (1, 32000, 5),
         (2, 50021, 128), (1, 150001, 20)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,V,top", SIZES)
def test_forward_matches_the_definition(cuda_device, rows, V, top, dtype):
    for T, k in ((1.0, top), (0.7, 0), (3.0, min(top, 2))):
        x, t = logits_of(rows * 7 + V, rows, V, dtype)
        check_forward(token_logprobs(x, t, top=k, temperature=T), x, t, k, T)
    check_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [61, 127, 300, 1031, 9001])
def test_masks_infinities_and_equal_logits(cuda_device, V, dtype):
    """Rows: most words ruled out by -inf, by the type's lowest value; only one word left; none
    left; all at the lowest; all equal; two levels (more equal logits than candidates fit);
    rising and falling; zeros of both signs; NaN; +inf; values at the type's ends."""
    low = torch.finfo(dtype).min
    g = torch.Generator().manual_seed(V)
    base = (torch.randn(14, V, generator=g) * 3).to(dtype)
    drop = torch.rand(V, generator=g) < 0.9
    drop[3] = False
    base[0, drop] = -INF
    base[1, drop] = low
    base[2], base[2, V - 1] = -INF, 2.0
    base[3] = -INF
    base[4] = low
    base[5] = 1.5
    base[6] = torch.where(torch.rand(V, generator=g) < 0.6, 4.0, 1.0).to(dtype)
    base[7] = torch.arange(V).float().to(dtype)
    base[8] = -torch.arange(V).float().to(dtype)
    base[9] = torch.where(torch.rand(V, generator=g) < 0.5, 0.0, -0.0).to(dtype)
    base[10, V // 2] = math.nan
    base[11, V // 3] = INF
    base[12, 0], base[12, 1] = torch.finfo(dtype).max, low
    base[13], base[13, 5] = low, -INF
    t = torch.randint(0, V, (14,), generator=g)
    t[0], t[1], t[6] = 3, 3, -100
    x, t = base.cuda(), t.cuda()
    for T, top in ((1.0, 20), (0.5, min(V, 128)), (1.0, 1)):
        check_forward(token_logprobs(x, t, top=top, temperature=T), x, t, top, T)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_shapes_and_index_types(cuda_device, dtype):
    """Rows of a wider tensor from an odd column, every alignment of a row's start, transposed
    and expanded logits, leading dimensions, int32 targets, no targets, no rows."""
    big, _ = logits_of(3, 6, 1300, dtype)
    for off in range(8):
        x = big[:, off:off + 1217]
        t = torch.arange(6, device=x.device)
        check_forward(token_logprobs(x, t, top=9), x, t, 9, 1.0)
    x = big.t()[:700].t().contiguous().t().t()[:, ::2]
    t32 = torch.arange(6, device=x.device, dtype=torch.int32)
    check_forward(token_logprobs(x, t32, top=4), x, t32, 4, 1.0)
    wide = big[:1].expand(5, 1300)
    check_forward(token_logprobs(wide, t32[:5], top=2), wide, t32[:5], 2, 1.0)
    cube = big[:, :1200].reshape(2, 3, 1200)
    r = token_logprobs(cube, t32.view(2, 3), top=3)
    assert r.logprobs.shape == r.entropy.shape == (2, 3) and r.top_indices.shape == (2, 3, 3)
    check_forward(r, cube.reshape(6, 1200), t32, 3, 1.0)
    one = token_logprobs(big[0], t32[0], top=3)
    assert one.entropy.shape == () and one.top_logprobs.shape == (3,)
    none = token_logprobs(big, top=2)
    assert none.logprobs is None and none.top_indices.shape == (6, 2)
    empty = token_logprobs(big[:0], t32[:0], top=2)
    assert empty.logprobs.shape == (0,) and empty.top_indices.shape == (0, 2)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1e-6, 0.013, 37.0, 1e6])
def test_temperatures_from_end_to_end(cuda_device, T):
    """Forward and gradients; at 1e-6 a row is its largest logit (two equal ones share it)."""
    x, t = logits_of(4, 6, 2050, torch.float32)
    x[0, 7] = x[0, 1900] = 20.0
    t[1] = 7
    check_forward(token_logprobs(x, t, top=5, temperature=T), x, t, 5, T)
    leaf = x.clone().requires_grad_(True)
    r = token_logprobs(leaf, t, top=5, temperature=T)
    g = torch.rand(6, generator=torch.Generator().manual_seed(1)).cuda()
    (got,) = torch.autograd.grad((r.logprobs, r.entropy), leaf, (g, g))
    want, F, points = reference_grad(x, t, 0, T, g, g, None)
    check_grad(got, want, F, points, 2050, torch.float32)


@pytest.mark.gpu
def test_gradient_of_the_gradient_is_refused(cuda_device):
    x, t = logits_of(4, 3, 50, torch.float32)
    leaf = x.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(token_logprobs(leaf, t).logprobs.sum(), leaf, create_graph=True)


@pytest.mark.gpu
def test_rows_past_32_bit_offsets(cuda_device):
    """2,200 rows of a million bf16 words: 4.4 GB, so element offsets pass 2^31 and byte offsets
    2^32; the last rows against the definition."""
    rows, V = 2200, 1_000_003
    x = torch.empty(rows, V, device=cuda_device, dtype=torch.bfloat16)
    g = torch.Generator(device=cuda_device).manual_seed(0)
    for r in range(0, rows, 200):
        x[r:r + 200] = torch.randn(200, V, generator=g, device=cuda_device) * 3
    t = torch.full((rows,), V - 1, device=cuda_device)
    got = token_logprobs(x, t, top=3)
    tail = dabsn_amd.TokenLogprobs(*(f[-2:] for f in got))
    check_forward(tail, x[-2:], t[-2:], 3, 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("V,top", [(3, 2), (130, 0)])
def test_rows_of_several_launches(cuda_device, V, top):
    """More rows than one launch takes give the bits of their two parts."""
    rows, cut = (1 << 21) + 21, 1 << 21
    g = torch.Generator(device=cuda_device).manual_seed(V)
    x = torch.randn(rows, V, generator=g, device=cuda_device).to(torch.bfloat16).requires_grad_(True)
    t = torch.randint(0, V, (rows,), generator=g, device=cuda_device)
    up = torch.randn(rows, generator=g, device=cuda_device)

    def call(s, e):
        r = token_logprobs(x[s:e], t[s:e], top=top)
        total = (r.logprobs * up[s:e]).sum() + (r.entropy * up[s:e]).sum()
        if top:
            total = total + (r.top_logprobs * up[s:e, None]).sum()
        return [f.detach() for f in r if f is not None], torch.autograd.grad(total, x)[0][s:e]

    whole, grad = call(0, rows)
    for s, e in ((0, cut), (cut, rows)):
        part, g = call(s, e)
        assert all(torch.equal(a[s:e], b) for a, b in zip(whole, part))
        assert torch.equal(grad[s:e], g)


@pytest.mark.gpu
def test_the_first_call_is_not_captured(cuda_device, monkeypatch):
    """Its error word would be made, and cleared on every replay, by the graph. A call before it
    makes the word, also one that reads its own."""
    x, t = logits_of(2, 4, 30, torch.float32)
    monkeypatch.setattr(dabsn_amd.kernels.ops, "_STICKY", {})
    with monkeypatch.context() as m:
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        with pytest.raises(RuntimeError, match="once before the capture"):
            token_logprobs(x, t)
    monkeypatch.setenv("DABSN_HIP_ERROR_CHECK", "sync")
    eager = token_logprobs(x, t).logprobs
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    assert torch.equal(token_logprobs(x, t).logprobs, eager)


@pytest.mark.gpu
def test_bad_targets_are_reported(cuda_device, monkeypatch):
    x, t = logits_of(1, 4, 30, torch.float32)
    t[1], t[2] = 30, -1
    r = token_logprobs(x, t)
    assert torch.isnan(r.logprobs).tolist() == [False, True, True, False]
    with pytest.raises(RuntimeError, match="error word"):
        check_errors()
    check_errors()
    monkeypatch.setenv("DABSN_HIP_ERROR_CHECK", "sync")
    with pytest.raises(RuntimeError, match="outside"):
        token_logprobs(x, t)
    monkeypatch.delenv("DABSN_HIP_ERROR_CHECK")
    check_errors()


# ---- gradients -------------------------------------------------------------------------------
def reference_grad(x, targets, top, T, gl, ge, gt, ignore=-100):
    """(gradient, magnitude F p / T + at-point terms) in 64 bits."""
    _, ent, _, ti, _, p, logp = reference(x, targets, top, T)
    rows = torch.arange(x.shape[0])
    d = lambda v: v.double().cpu()  # noqa: E731
    lq = torch.where(p > 0, logp, 0.0)
    total = torch.zeros(x.shape[0], dtype=torch.float64)
    points = torch.zeros_like(p)
    if gl is not None:
        ok = targets.cpu() != ignore
        g = torch.where(ok, d(gl), 0.0)
        total = total + g
        points[rows, targets.cpu().long().clamp(min=0)] += g
    if gt is not None:
        total = total + d(gt).sum(1)
        points.scatter_add_(1, ti, d(gt))
    h = d(ge)[:, None] if ge is not None else torch.zeros(x.shape[0], 1, dtype=torch.float64)
    dense = -p * (total[:, None] + h * (lq + ent[:, None]))
    size = total.abs()
    if gt is not None:
        size = size + d(gt).abs().sum(1)
    if gl is not None:
        size = size + d(gl).abs()
    # Exponentials below 2^-126 are 0, so p may lack that much: it enters F by as much as check_grad
    # multiplies F by at least, u 328, leaves of it; |logp| <= 104 there.
    factor = size[:, None] + h.abs() * (lq.abs().clamp(max=104) + ent[:, None] + 1)
    F = (p + 2.0 ** -126 / (328 * U)) * factor / T
    live = (p.sum(1) > 0)[:, None]
    return torch.where(live, (dense + points) / T, 0.0), F, points.abs() / T


def check_grad(got, want, F, points, V, dtype):
    S = sum_error(V)
    rnd = U if dtype == torch.float32 else 2.0 ** -8
    tol = U * (F * (2 * S + 3 * 104 + 16) + 4 * points) + rnd * want.abs() * (1 + 1e-3)
    # values below the type's normal range round absolutely
    err = (got.double().cpu() - want).abs()
    assert bool((err <= tol + 2.0 ** -126).all()), float((err - tol).max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,V,top,T", [(1, 1, 1, 1.0), (5, 7, 3, 0.7), (33, 60, 5, 1.0), (600, 65, 20, 1.0), (20, 128, 128, 3.0),
                                          (20, 200, 9, 1.0),
                                          (4, 1031, 128, 2.0), (3, 4099, 33, 1.0), (2, 9001, 5, 0.5),
                                          (1, 50021, 2, 1.0)])
def test_gradients_match_the_formula(cuda_device, rows, V, top, T, dtype):
    x, t = logits_of(rows + V, rows, V, dtype)
    if V > 20:
        x[:, ::3] = -INF  # ruled-out words, targets among them
        t[t % 3 == 0] = 1
    g = torch.Generator().manual_seed(V)
    gl, ge = torch.randn(rows, generator=g).cuda(), torch.randn(rows, generator=g).cuda()
    gt = torch.randn(rows, top, generator=g).cuda()
    if V > 20:
        with torch.no_grad():  # a target that is an alternative too
            t[-1] = token_logprobs(x, top=top).top_indices[-1, 0]
    finite = torch.isfinite(x).sum(1).min() >= top
    for use in ("l", "e", "t", "le", "let"):
        if "t" in use and not finite:
            continue
        leaf = x.detach().clone().requires_grad_(True)
        r = token_logprobs(leaf, t, top=top, temperature=T)
        outs = [o for k, o in (("l", r.logprobs), ("e", r.entropy), ("t", r.top_logprobs)) if k in use]
        ups = [u for k, u in (("l", gl), ("e", ge), ("t", gt)) if k in use]
        (got,) = torch.autograd.grad(outs, leaf, ups)
        want, F, points = reference_grad(x, t, top, T, gl if "l" in use else None,
                                         ge if "e" in use else None, gt if "t" in use else None)
        assert got.dtype == dtype
        check_grad(got, want, F, points, V, dtype)


@pytest.mark.gpu
def test_gradients_match_differences(cuda_device):
    """A direction's derivative against central differences of the definition in 64 bits at steps
    of 1e-6: an error of the square of the step and of 2^-53 / step, far below the 1e-5 asked."""
    x, t = logits_of(8, 6, 257, torch.float32)
    d = torch.randn(6, 257, generator=torch.Generator().manual_seed(2), dtype=torch.float64)
    g = torch.rand(6, dtype=torch.float64, generator=torch.Generator().manual_seed(3)) + 0.5
    leaf = x.clone().requires_grad_(True)
    r = token_logprobs(leaf, t, top=4, temperature=0.8)
    total = (r.logprobs * g.cuda().float()).sum() + (r.entropy * g.cuda().float()).sum() + (
        r.top_logprobs * g.cuda().float()[:, None]).sum()
    (got,) = torch.autograd.grad(total, leaf)

    def value(v):
        lp, ent, tl, *_ = reference(v, t, 4, 0.8)
        return float((g * lp).sum() + (g * ent).sum() + (g[:, None] * tl).sum())

    step = 1e-6
    want = (value(x.double().cpu() + step * d) - value(x.double().cpu() - step * d)) / (2 * step)
    assert abs(float((got.double().cpu() * d).sum()) - want) <= 1e-5 * float(d.abs().sum())


@pytest.mark.gpu
def test_gradients_of_strided_expanded_and_emptied_rows(cuda_device):
    big, _ = logits_of(5, 6, 1300, torch.bfloat16)
    t = torch.arange(6, device=cuda_device)
    base = big.clone().requires_grad_(True)
    r = token_logprobs(base[:, 3:1220], t)
    (got,) = torch.autograd.grad(r.logprobs.sum(), base)  # an expanded upstream gradient
    want, F, pts = reference_grad(big[:, 3:1220], t, 0, 1.0, torch.ones(6), None, None)
    check_grad(got[:, 3:1220], want, F, pts, 1217, torch.bfloat16)
    assert float(got[:, :3].float().abs().max()) == 0 == float(got[:, 1220:].float().abs().max())
    row = big[:1, :500].float().requires_grad_(True)
    r = token_logprobs(row.expand(6, 500), t)
    (got,) = torch.autograd.grad(r.logprobs.sum(), row)
    want, F, pts = reference_grad(row.expand(6, 500), t, 0, 1.0, torch.ones(6), None, None)
    check_grad(got, want.sum(0, keepdim=True), F.sum(0) * 2, pts.sum(0) * 2, 500, torch.float32)
    dead = torch.full((3, 40), -INF, device=cuda_device).requires_grad_(True)
    r = token_logprobs(dead, t[:3], top=2)
    assert r.entropy.tolist() == [0.0] * 3 and r.top_indices.tolist() == [[0, 1]] * 3
    (got,) = torch.autograd.grad((r.logprobs, r.entropy, r.top_logprobs), dead,
                                 (torch.ones(3).cuda(), torch.ones(3).cuda(), torch.ones(3, 2).cuda()))
    assert float(got.abs().max()) == 0


# ---- from hidden rows ------------------------------------------------------------------------
def readout_case(seed, n, H, V, dtype, bias=True):
    g = torch.Generator().manual_seed(seed)
    h = torch.randn(n, H, generator=g).to(dtype)
    w = (torch.randn(V, H, generator=g) * 2 / H ** 0.5).to(dtype)
    b = torch.randn(V, generator=g).to(dtype) if bias else None
    t = torch.randint(0, V, (n,), generator=g)
    t[::7] = -100
    return [x if x is None else x.cuda() for x in (h, w, b, t)]


def logit_error(h, w, b):
    """The fp32 products' error: H + 2 additions, u each, of the terms' magnitudes."""
    mag = h.double().cpu().abs() @ w.double().cpu().abs().t()
    if b is not None:
        mag = mag + b.double().cpu().abs()
    return U * (h.shape[1] + 2) * mag.amax(1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,H,V,budget,bias", [(1, 3, 5, None, True), (70, 48, 33, 16 * 33, True),
                                               (90, 24, 128, None, False), (50, 24, 200, None, True),
                                               (300, 200, 1001, 40 * 1001, False),
                                               (130, 72, 4099, 1 << 18, True)])
def test_linear_form_matches_the_definition(cuda_device, n, H, V, budget, bias, dtype):
    """The logits' error (``logit_error``, e a row) shifts a log probability by 2 e and the entropy
    by 2 e (1 + ln V), beside the row kernel's own; gradients in the norm: the softmax's relative
    error 2 e + the rows', and for bf16 one rounding, 2^-8."""
    h, w, b, t = readout_case(n + V, n, H, V, dtype, bias)
    leaves = [x if x is None else x.clone().requires_grad_(True) for x in (h, w, b)]
    r = chunked_linear_token_logprobs(*leaves, t, temperature=0.9, chunk_budget=budget)
    ref = [x if x is None else x.double().cpu().requires_grad_(True) for x in (h, w, b)]
    x = torch.nn.functional.linear(*ref)
    logp = torch.log_softmax(x / 0.9, dim=1)
    ok = (t != -100).cpu()
    want_lp = torch.where(ok, logp.gather(1, t.cpu().clamp(min=0)[:, None])[:, 0], 0.0)
    want_ent = -(logp.exp() * logp).sum(1)
    e = logit_error(h, w, b) / 0.9
    S, ln = sum_error(V), math.log(V)
    spread = (x.amax(1) - x.amin(1)).detach() / 0.9
    assert bool(((r.logprobs.double().cpu() - want_lp).abs() <= 2 * e + U * (8 * spread + 8 * ln + S)).all())
    assert bool(((r.entropy.double().cpu() - want_ent).abs()
                 <= 2 * e * (1 + ln) + U * (S * (1 + 2 * ln) + 8 * ln)).all())
    g = torch.Generator().manual_seed(1)
    gl, ge = torch.randn(n, generator=g), torch.randn(n, generator=g) * 0.1
    got = torch.autograd.grad((r.logprobs, r.entropy), [v for v in leaves if v is not None],
                              (gl.cuda(), ge.cuda()))
    want = torch.autograd.grad((want_lp, want_ent), [v for v in ref if v is not None],
                               (gl.double(), ge.double()))
    tol = 4 * float(e.max()) * (1 + ln) + U * (4 * S + 400 + n + V + H) + (
        2.0 ** -8 if dtype == torch.bfloat16 else 0.0)
    for a, c in zip(got, want):
        assert a.dtype == dtype and float((a.double().cpu() - c).norm()) <= tol * float(c.norm())


@pytest.mark.gpu
def test_linear_form_alternatives_frozen_readout_and_leading_dimensions(cuda_device):
    h, w, b, t = readout_case(4, 24, 64, 700, torch.bfloat16)
    r = chunked_linear_token_logprobs(h.view(2, 12, 64), w, b, t.view(2, 12), top=6, chunk_budget=5 * 700)
    assert r.top_indices.shape == (2, 12, 6)
    x = torch.nn.functional.linear(h.float(), w.float(), b.float())
    flat = token_logprobs(x, t, top=6)
    # the alternatives' logits agree to the products' error
    got = x.gather(1, r.top_indices.view(24, 6))
    assert float((got - x.gather(1, flat.top_indices)).abs().max()) <= 2 * float(logit_error(h, w, b).max())
    hidden = h.clone().requires_grad_(True)
    r = chunked_linear_token_logprobs(hidden, w, b, t, chunk_budget=5 * 700)
    (one,) = torch.autograd.grad(r.logprobs.sum(), hidden)
    leaves = [v.clone().requires_grad_(True) for v in (h, w, b)]
    r = chunked_linear_token_logprobs(*leaves, t, chunk_budget=5 * 700)
    assert torch.equal(one, torch.autograd.grad(r.logprobs.sum(), leaves)[0])
    with torch.autocast("cuda", torch.bfloat16):
        a = chunked_linear_token_logprobs(h.float(), w.float(), b.float(), t)
    assert torch.equal(a.logprobs, chunked_linear_token_logprobs(h, w, b, t).logprobs)


# ---- as a user's program runs them -----------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("train", [False, True])
def test_capture_and_replay(cuda_device, train):
    from test_capture import _capture, _replays

    token_logprobs(torch.zeros(1, 4, device=cuda_device))  # the error word exists before
    cases = [logits_of(s, 40, 2050, torch.bfloat16) for s in (1, 2, 3)]
    static = [v.clone() for v in cases[0]]
    ups = torch.randn(2, 40, device=cuda_device)

    def run(v):
        x, t = v
        if not train:
            return list(token_logprobs(x, t, top=5))
        leaf = x.detach().requires_grad_(True)
        r = token_logprobs(leaf, t, top=5)
        return [*r, *torch.autograd.grad((r.logprobs, r.entropy), leaf, tuple(ups))]

    graph, outs = _capture(lambda: [o.detach() for o in run(static)])
    _replays(graph, outs, static, cases[1:] + cases[:1], lambda v: [o.detach() for o in run(v)])


@pytest.mark.gpu
def test_calls_on_two_streams_do_not_disturb_each_other(cuda_device):
    x, t = logits_of(1, 512, 9001, torch.bfloat16)
    want = token_logprobs(x, t, top=20)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(token_logprobs(x, t, top=20))
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(a, b) for a, b in zip(o, want))


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [None, 5.0])
def test_a_model_scores_its_tokens(cuda_device, scale):
    """``DABSNSequenceLM.token_logprobs`` against its own forward."""
    torch.manual_seed(0)
    m = dabsn_amd.DABSNSequenceLM(61, 32, depth=1, embed_scale=scale).cuda()
    ids = torch.randint(0, 61, (3, 20), device=cuda_device)
    with torch.no_grad():
        r = m.token_logprobs(ids, top=4)
        logp = torch.log_softmax(m(ids).double(), dim=-1)
    want = logp[:, :-1].gather(2, ids[:, 1:, None])[..., 0]
    assert float((r.logprobs[:, :-1].double() - want).abs().max()) <= 1e-5
    assert float(r.logprobs[:, -1].abs().max()) == 0
    assert float((r.top_logprobs.double() - logp.topk(4).values).abs().max()) <= 1e-5
