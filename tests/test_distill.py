"""Distillation from a teacher's top logits against the definition in 64 bits.

Tolerances, u = 2^-24, S = V / 64 + 64 + 3 ln V (the exp-sum's relative error in u, derived in
test_scoring.py): the teacher's weights are 64-bit values of its fp32 inputs, with 1 / T in fp32:
an exponent off by 2 u |t| / T. A log probability of the student is off by
e = u (4 (spread + ln V) + S), the rest's log sum by 2 S u, so a row's loss by e + 2 S u + 4 u M
with M the largest |t| / T, each at most times sum q + q_r = 1, and its rounding. A gradient is
T / n (p b - q): p and b off by S u + 312 u each (an exponent argument of at most 104, 3 u), q by
4 u M + u; p a at other tokens, a = b - q_r / r a difference: 2 S u (b + q_r / r) p; then one
rounding to the logits' type (u, or 2^-8 for bf16)."""

from __future__ import annotations

import math

import pytest
import torch

import dabsn_amd
from dabsn_amd import chunked_linear_distillation, distillation_from_logits, token_logprobs
from dabsn_amd.kernels import check_errors
from test_scoring import logit_error, sum_error

U = 2.0 ** -24
INF = math.inf
I64 = torch.int64


# ---- refusals (no GPU) -----------------------------------------------------------------------
def _z(*s, dtype=torch.float32):
    return torch.zeros(s, dtype=dtype)


@pytest.mark.parametrize("call,error,match", [
    (lambda: distillation_from_logits(_z(2, 5).half(), _z(2, 3), _z(2, 3, dtype=I64)), TypeError, "logits must"),
    (lambda: distillation_from_logits(_z(5), _z(3), _z(3, dtype=I64)), ValueError, "expected logits"),
    (lambda: distillation_from_logits(_z(2, 5), _z(2, 3).double(), _z(2, 3, dtype=I64)), TypeError,
     "top_logits must"),
    (lambda: distillation_from_logits(_z(2, 5), _z(2, 3), _z(2, 4, dtype=I64)), ValueError, "do not match"),
    (lambda: distillation_from_logits(_z(2, 5), _z(3, 3), _z(3, 3, dtype=I64)), ValueError, "does not match"),
    (lambda: distillation_from_logits(_z(2, 5), _z(2, 0), _z(2, 0, dtype=I64)), ValueError, "1 to 128"),
    (lambda: distillation_from_logits(_z(2, 500), _z(2, 129), _z(2, 129, dtype=I64)), ValueError, "1 to 128"),
    (lambda: distillation_from_logits(_z(2, 5), _z(2, 3), _z(2, 3)), TypeError, "int64 or int32"),
    (lambda: distillation_from_logits(_z(2, 5), _z(2, 3), _z(2, 3, dtype=I64), temperature=0), ValueError,
     "temperature"),
    (lambda: distillation_from_logits(_z(2, 5), _z(2, 3), _z(2, 3, dtype=I64), teacher_lse=_z(3)),
     ValueError, "teacher_lse"),
    (lambda: distillation_from_logits(_z(2, 5), _z(2, 3), _z(2, 3, dtype=I64),
                                      teacher_lse=_z(2, dtype=I64)), TypeError, "teacher_lse"),
    (lambda: distillation_from_logits(_z(1, 480_001), _z(1, 3), _z(1, 3, dtype=I64), teacher_lse=_z(1)),
     ValueError, "480000"),
    (lambda: distillation_from_logits(_z(2, 5), _z(2, 3), _z(2, 3, dtype=I64)), RuntimeError, "device"),
    (lambda: chunked_linear_distillation(_z(2, 3), _z(5, 4), None, _z(2, 3), _z(2, 3, dtype=I64)),
     ValueError, "do not match"),
    (lambda: chunked_linear_distillation(_z(2, 3), _z(5, 3), None, _z(2, 3), _z(2, 3, dtype=I64)),
     RuntimeError, "device"),
])
def test_refusals(call, error, match):
    with pytest.raises(error, match=match):
        call()


def test_library_refuses_bad_arguments_before_it_launches():
    from dabsn_amd import _lib

    lib, one = _lib.load(), 1 << 20
    f = lambda dtype=0, rows=2, V=5, ld=5, bias=None, top=3, vt=0, t=1.0, lse=None, out=None, ldo=0, half=0, scale=one: (  # noqa: E731,E501
        lib.dabsn_hip_distill(dtype, rows, V, one, ld, bias, top, vt, one, one, -100, t, lse, one, one,
                              one, scale, half, out, ldo, one, None))
    for kw in (dict(dtype=3), dict(V=0), dict(ld=4), dict(top=0), dict(top=129), dict(vt=2), dict(t=0.0),
               dict(V=480_001, ld=480_001, lse=one), dict(dtype=1, bias=one), dict(out=one, ldo=4),
               dict(out=one, ldo=8, bias=one), dict(out=one, ldo=8, scale=None),
               dict(dtype=1, out=one, ldo=8, half=1)):
        assert f(**kw) == -2, kw
    assert lib.dabsn_hip_distill_bwd(0, 2, 5, one, 5, 0, one, 1.0, one, one, one, one, 0, one, None) == -2
    assert lib.dabsn_hip_distill_rows(2, 5, 0, 0, one, one, -100, one, None) == -2
    assert lib.dabsn_hip_distill_mean(2, None, 1.0, 1.0, one, one, None) == -2


# ---- the definition in 64 bits ---------------------------------------------------------------
def reference(x, values, tokens, T, lse=None, ignore=-100):
    """(loss, gradient, loss tolerance, gradient tolerance without its rounding), x [rows, V]."""
    x, v, k = x.detach().double().cpu(), values.double().cpu(), tokens.cpu().long()
    V = x.shape[1]
    z = x / T
    m = z.amax(1, keepdim=True)
    empty = m == -INF
    m = torch.where(empty, 0.0, m)
    s = torch.exp(z - m).sum(1, keepdim=True)
    logp = torch.where(empty, -INF, z - m - torch.log(torch.where(empty, 1.0, s)))
    p = logp.exp()
    here = (k != ignore) & (v != -INF)
    some = here.any(1)
    at = torch.where(here, k, 0)
    u = torch.where(here, v / T, -INF)
    if lse is None:
        n = torch.logsumexp(u, 1)
    else:
        n = lse.double().cpu()
    logq = u - n[:, None]
    q = torch.where(here & some[:, None], torch.exp(logq), 0.0)
    lp = logp.gather(1, at)
    rows = torch.where(q > 0, q * (logq - lp), 0.0).sum(1)
    spread = torch.zeros_like(p).scatter_add_(1, at, q)
    hit = torch.zeros_like(p).scatter_add_(1, at, here.double()) > 0
    total, back, rest = q.sum(1), torch.zeros_like(q.sum(1)), torch.zeros_like(q.sum(1))
    left = torch.where(hit, 0.0, p).sum(1)
    if lse is not None:
        rest = torch.where(left > 0, (1 - total).clamp(min=0), 0.0)
        rows = rows + torch.where(rest > 0, rest * (torch.log(rest) - torch.log(left)), 0.0)
        total = total + rest
        back = torch.where(left > 0, rest / left, 0.0)
    grad = p * total[:, None] - spread - torch.where(hit, 0.0, p * back[:, None])
    count = max(1, int(some.sum()))
    f = torch.where(some & ~empty[:, 0], T / count, 0.0)[:, None]
    loss = float(T * T * torch.where(some, rows, 0.0).sum() / count)
    # tolerances
    S, ln = sum_error(V), math.log(V)
    M = float(torch.where(here, v, 0.0).abs().amax()) / T + float(n[some].abs().amax() if some.any() else 0)
    far = float(torch.where(here & torch.isfinite(lp), (lp - m * 0).abs(), 0.0).amax())
    weight = (q.sum(1) + rest).amax().item() if some.any() else 0.0
    logs = float(torch.where(rest > 0, torch.log(rest.clamp(min=1e-300)).abs(), 0.0).amax())
    e = U * (4 * (far + ln) + 3 * S + 4 * M * (1 + far + M + logs) + 8) + 2 * U * abs(loss) / T ** 2
    tol_loss = T * T * weight * e
    tol = U * ((S + 4 * 104 + 8) * p * (total + back)[:, None] * 2
               + (8 * M + 8) * (spread + p * torch.where(left > 0, 4 * M * 1.0 / left, 0.0)[:, None]
                                * (0.0 if lse is None else 1.0)))
    return loss, grad * f, tol_loss, tol * f.abs()


def check(loss, grad, want, dtype):
    ref, g, tol_loss, tol = want
    assert loss.dtype == torch.float32 and loss.shape == ()
    if math.isfinite(ref):
        assert abs(float(loss.detach()) - ref) <= tol_loss, (float(loss.detach()), ref, tol_loss)
    else:
        assert float(loss.detach()) == ref
    rnd = U if dtype == torch.float32 else 2.0 ** -8
    err = (grad.double().cpu() - g).abs()
    bound = tol + rnd * (g.abs() + tol) + 2.0 ** -126
    assert grad.dtype == dtype and bool((err <= bound).all()), float((err - bound).max())


def case(seed, rows, V, K, dtype, rest=False, T=1.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, V, generator=g) * 2.5).to(dtype)
    teacher = x.float() + torch.randn(rows, V, generator=g) * 1.5
    values, tokens = teacher.topk(K, dim=1)
    lse = torch.logsumexp(teacher.double() / T, 1).float() if rest else None
    if rows > 3:
        tokens[rows // 2, K // 2:] = -100  # a shorter list
        tokens[1] = -100  # a padding row
    return [v if v is None else v.cuda() for v in (x, values, tokens, lse)]


def run(x, values, tokens, lse, T=1.0, up=1.0):
    leaf = x.detach().clone().requires_grad_(True)
    loss = distillation_from_logits(leaf, values, tokens, temperature=T, teacher_lse=lse)
    (g,) = torch.autograd.grad(loss * up, leaf)
    return loss, g / up if up != 1.0 else g


SIZES = [(1, 1, 1), (3, 2, 2), (5, 7, 3), (33, 60, 8), (18, 64, 64), (600, 65, 8), (19, 128, 128), (19, 129, 20),
         (9, 300, 17), (9, 1024, 128), (9, 1025, 128), (4, 1031, 1),
         (5, 2049, 64), (3, 4099, 33), (2, 9001, 65), (1, 32000, 64), (2, 50021, 37)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("rows,V,K", SIZES)
def test_loss_and_gradient_match_the_definition(cuda_device, rows, V, K, rest, dtype):
    for T in (1.0, 2.0, 0.7):
        x, values, tokens, lse = case(rows + V, rows, V, K, dtype, rest, T)
        check(*run(x, values, tokens, lse, T), reference(x, values, tokens, T, lse), dtype)
    check_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("V,K", [(50, 20), (128, 128), (200, 100), (1031, 128), (9001, 40)])
def test_tokens_listed_twice_and_absent_entries(cuda_device, V, K, rest):
    """The same token at several places of a row (its weights add), in neighbouring and far
    places; entries with the value -inf; a row with one entry; rows with none."""
    x, values, tokens, lse = case(7, 8, V, K, torch.float32, rest)
    if rest:
        lse += 2.0  # weights that leave a rest though tokens repeat
    tokens[0, 1] = tokens[0, 0]
    tokens[2, K - 1] = tokens[2, 0]
    tokens[3, :] = tokens[3, 0]
    values[5, ::2] = -INF
    values[6] = -INF
    tokens[7, 1:] = -100
    check(*run(x, values, tokens, lse), reference(x, values, tokens, 1.0, lse), torch.float32)


@pytest.mark.gpu
def test_far_tokens_that_share_a_mark_are_not_taken_for_one(cuda_device):
    """Words 2^15 apart share a bit of the mark that finds tokens listed twice."""
    x, values, tokens, _ = case(9, 4, 70000, 4, torch.float32)
    tokens[0] = torch.tensor([5, 5 + 32768, 5 + 65536, 6])
    tokens[2] = torch.tensor([9, 9 + 32768, 9, 9 + 32768])
    check(*run(x, values, tokens, None), reference(x, values, tokens, 1.0), torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masked_students(cuda_device, dtype):
    """Unlisted words ruled out by -inf or the lowest value (the rest is left out, or its mass is
    0), every word listed, a student sure of a listed word (a rest of 1e-12), a listed word ruled
    out (loss inf)."""
    low = torch.finfo(dtype).min
    x, values, tokens, lse = case(11, 6, 300, 12, dtype, True)
    keep = torch.zeros(6, 300, dtype=torch.bool, device="cuda").scatter_(1, tokens.clamp(min=0), True)
    x[0] = torch.where(keep[0], x[0], -INF)
    x[2] = torch.where(keep[2], x[2], low)
    x[4, tokens[4, 0]] = 40.0
    x[5, tokens[5, 0]] = 30.0
    check(*run(x, values, tokens, lse), reference(x, values, tokens, 1.0, lse), dtype)
    x, values, tokens, lse = case(12, 3, 100, 100, dtype, True)
    check(*run(x, values, tokens, lse), reference(x, values, tokens, 1.0, lse), dtype)
    x, values, tokens, lse = case(13, 3, 100, 10, dtype, False)
    x[0, tokens[0, 3]] = -INF
    loss, g = run(x, values, tokens, lse)
    assert float(loss.detach()) == INF and bool(torch.isfinite(g).all())
    x[2] = -INF
    loss, g = run(x, values, tokens, lse)
    assert float(loss.detach()) == INF and float(g[2].float().abs().max()) == 0


@pytest.mark.gpu
def test_the_rest_of_the_largest_vocabulary(cuda_device):
    x, values, tokens, lse = case(2, 2, 480_000, 30, torch.bfloat16, True)
    tokens[0, 0], tokens[1, 0] = 479_999, 0
    check(*run(x, values, tokens, lse), reference(x, values, tokens, 1.0, lse), torch.bfloat16)


@pytest.mark.gpu
def test_gradients_formed_with_the_loss_of_strided_rows(cuda_device):
    """Rows of a wider tensor, whose gradient rows lie at other addresses modulo a line."""
    wide = torch.randn(2100, 8200, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    base = (wide * 2.5).requires_grad_(True)
    values, tokens = base.detach()[:, 5:8196].topk(9, dim=1)
    loss = distillation_from_logits(base[:, 5:8196], values, tokens)
    (g,) = torch.autograd.grad(loss, base)
    dense = base.detach()[:, 5:8196].contiguous().requires_grad_(True)
    (want,) = torch.autograd.grad(distillation_from_logits(dense, values, tokens), dense)
    # the same terms in other groups: the softmax's sums differ by their roundings
    assert float((g[:, 5:8196] - want).abs().max()) <= 4 * sum_error(8191) * U * float(want.abs().max())
    assert float(g[:, :5].abs().max()) == 0 == float(g[:, 8196:].abs().max())


@pytest.mark.gpu
def test_only_padding_and_no_rows(cuda_device):
    x, values, tokens, lse = case(3, 5, 40, 6, torch.float32, True)
    tokens.fill_(-100)
    loss, g = run(x, values, tokens, lse)
    assert float(loss.detach()) == 0 and float(g.abs().max()) == 0
    loss, g = run(x[:0], values[:0], tokens[:0], lse[:0])
    assert float(loss.detach()) == 0 and g.shape == (0, 40)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_shapes_and_types(cuda_device, dtype):
    x, values, tokens, lse = case(5, 6, 1300, 16, dtype, True)
    for off in (1, 2, 3, 5, 7):  # rows at every alignment; the gradient's rows are dense
        part = x[:, off:off + 1217]
        tk = tokens.clamp(max=1216)
        check(*run_view(x, off, values, tk, lse), reference(part, values, tk, 1.0, lse), dtype)
    cube = x.view(2, 3, 1300)
    loss = distillation_from_logits(cube, values.view(2, 3, 16), tokens.view(2, 3, 16).int(),
                                    teacher_lse=lse.view(2, 3))
    assert torch.equal(loss, distillation_from_logits(x, values, tokens, teacher_lse=lse))
    half = values.bfloat16()
    a = distillation_from_logits(x, half, tokens, teacher_lse=lse)
    assert torch.equal(a, distillation_from_logits(x, half.float(), tokens, teacher_lse=lse.double()))
    b = distillation_from_logits(x, values.t().contiguous().t(), tokens.t().contiguous().t())
    assert torch.equal(b, distillation_from_logits(x, values, tokens))


def run_view(x, off, values, tokens, lse):
    base = x.clone().requires_grad_(True)
    loss = distillation_from_logits(base[:, off:off + 1217], values, tokens, teacher_lse=lse)
    (g,) = torch.autograd.grad(loss, base)
    assert float(g[:, :off].float().abs().max()) == 0
    return loss, g[:, off:off + 1217]


@pytest.mark.gpu
def test_upstream_factor_scales_the_gradient(cuda_device):
    """A factor of 4 and one of 1/8 are exact; twice through a kept graph gives the same bits."""
    x, values, tokens, lse = case(5, 6, 1300, 16, torch.bfloat16, True)
    leaf = x.clone().requires_grad_(True)
    loss = distillation_from_logits(leaf, values, tokens, teacher_lse=lse)
    (g1,) = torch.autograd.grad(loss, leaf, retain_graph=True)
    (g2,) = torch.autograd.grad(loss, leaf, retain_graph=True)
    (g4,) = torch.autograd.grad(loss * 4, leaf, retain_graph=True)
    (g8,) = torch.autograd.grad(loss / 8, leaf)
    assert torch.equal(g1, g2) and torch.equal(g1 * 4, g4) and torch.equal(g1 / 8, g8)


FUSED = [(8300, 2050, 16), (4096, 4096, 5), (1030, 16385, 64), (520, 32777, 40), (400, 65000, 20),
         (150, 131080, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,V,K", FUSED)
def test_gradients_formed_with_the_loss(cuda_device, n, V, K, dtype):
    """Many logits: rows of every way to hold them, and of sizes that take two passes. The gradient equals the one that a factor of 2
    forms again, halved (exact), bit for bit, its first rows the definition's, and a second
    backward gives it again though the first one's result was changed."""
    assert n * V >= 1 << 24
    x = (torch.randn(n, V, generator=torch.Generator(device="cuda").manual_seed(V), device="cuda")
         * 2.5).to(dtype)
    values, tokens = (x.float() + torch.randn(n, V, device="cuda")).topk(K, dim=1)
    tokens[8:] = torch.where(torch.arange(n - 8, device="cuda")[:, None] % 7 == 0, -100, tokens[8:])
    tokens[0, 0] = tokens[0, -1]
    x[1, tokens[1, 0]] = 30.0
    lse = torch.logsumexp(x.float(), 1) + 1
    leaf = x.requires_grad_(True)
    for rest in (None, lse):
        loss = distillation_from_logits(leaf, values, tokens, temperature=1.0, teacher_lse=rest)
        (g2,) = torch.autograd.grad(loss * 2, leaf, retain_graph=True)
        (g1,) = torch.autograd.grad(loss, leaf, retain_graph=True)
        assert torch.equal(g2 / 2, g1)
        loss = distillation_from_logits(leaf, values, tokens, temperature=1.0, teacher_lse=rest)
        (ga,) = torch.autograd.grad(loss, leaf, retain_graph=True)
        assert torch.equal(ga, g1)
        ga.zero_()
        (gb,) = torch.autograd.grad(loss, leaf)
        assert torch.equal(gb, g1)
        with torch.no_grad():
            plain = distillation_from_logits(leaf, values, tokens, teacher_lse=rest)
        # Without a gradient the rows' sums are of other groups: ln s and the rest's logarithm
        # differ by at most 2 S U each, both times weights of at most 1 in sum; rows and mean are
        # rounded once in each.
        off = abs(float(plain) - float(loss.detach()))
        assert off <= U * (4 * sum_error(V) + 8 * (1 + abs(float(loss.detach()))))
        part = None if rest is None else rest[:8]
        _, grad, _, tol = reference(x[:8], values[:8], tokens[:8], 1.0, part)
        counted = int((tokens != -100).any(1).sum())
        small = int((tokens[:8] != -100).any(1).sum())
        rnd = U if dtype == torch.float32 else 2.0 ** -8
        want, tol = grad * small / counted, tol * small / counted
        err = (g1[:8].double().cpu() - want).abs()
        assert bool((err <= tol + (rnd + 2 * U) * (want.abs() + tol) + 2.0 ** -126).all())


@pytest.mark.gpu
def test_gradients_formed_with_the_loss_in_a_graph(cuda_device):
    """Loss and backward captured together replay with new inputs."""
    from test_capture import _capture, _replays

    token_logprobs(torch.zeros(1, 4, device=cuda_device))
    cases = [case(s, 4100, 4104, 16, torch.bfloat16, True) for s in (1, 2, 3)]
    static = [v.clone() for v in cases[0]]

    def go(v):
        leaf = v[0].detach().requires_grad_(True)
        loss = distillation_from_logits(leaf, v[1], v[2], teacher_lse=v[3])
        return [loss.detach(), *torch.autograd.grad(loss, leaf)]

    graph, outs = _capture(lambda: go(static))
    _replays(graph, outs, static, cases[1:] + cases[:1], go)


@pytest.mark.gpu
def test_loss_weight(cuda_device):
    """A weight of 1/4 is exact in the loss and the gradients of both forms."""
    x, values, tokens, lse = case(5, 6, 4101, 16, torch.bfloat16, True)
    for big in (False, True):
        rep = 700 if big else 1
        xs, vs, ts = x.repeat(rep, 1).requires_grad_(True), values.repeat(rep, 1), tokens.repeat(rep, 1)
        a = distillation_from_logits(xs, vs, ts)
        b = distillation_from_logits(xs, vs, ts, loss_weight=0.25)
        assert torch.equal(a / 4, b)
        assert torch.equal(torch.autograd.grad(a, xs)[0] / 4, torch.autograd.grad(b, xs)[0])
    h, w, b, values, tokens, lse = linear_case(1, 96, 64, 1000, 16, torch.bfloat16)
    h.requires_grad_(True)
    one = chunked_linear_distillation(h, w, b, values, tokens, teacher_lse=lse)
    part = chunked_linear_distillation(h, w, b, values, tokens, teacher_lse=lse, loss_weight=0.25)
    assert torch.equal(one / 4, part)
    assert torch.equal(torch.autograd.grad(one, h)[0] / 4, torch.autograd.grad(part, h)[0])


@pytest.mark.gpu
@pytest.mark.parametrize("rest", [False, True])
def test_many_rows(cuda_device, rest):
    """Rows whose losses are summed by many workgroups, the last of them one row long."""
    rows = 5 * 4096 + 1
    x, values, tokens, lse = case(3, rows, 9, 3, torch.float32, rest)
    check(*run(x, values, tokens, lse), reference(x, values, tokens, 1.0, lse), torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [3, 130])
def test_rows_of_several_launches(cuda_device, V):
    """More rows than one launch takes: the gradient rows are those of its two parts (times their
    counts), and the mean that of their means. Each part's mean is off by U of itself (its last
    rounding) and U (those of its partial sums, all of one sign), the whole's as well."""
    rows, cut, K = (1 << 21) + 21, 1 << 21, 2
    g = torch.Generator(device=cuda_device).manual_seed(V)
    x = torch.randn(rows, V, generator=g, device=cuda_device).to(torch.bfloat16)
    values = torch.randn(rows, K, generator=g, device=cuda_device)
    tokens = torch.randint(0, V, (rows, K), generator=g, device=cuda_device)
    loss, grad = run(x, values, tokens, None)
    head, gh = run(x[:cut], values[:cut], tokens[:cut], None)
    tail, gt = run(x[cut:], values[cut:], tokens[cut:], None)
    want = (float(head.detach()) * cut + float(tail.detach()) * (rows - cut)) / rows
    assert abs(float(loss.detach()) - want) <= 4 * U * want
    # Each side times its count: a half step of bf16 each (and of the factor's and the value's fp32,
    # within 1 + 2^-7), and at listed words, where the value is the difference p f - q f of terms of
    # at most 1, U for each of the products and the difference whose factors f differ: 4 U a side.
    for s, e, part, n in ((0, cut, gh, cut), (cut, rows, gt, rows - cut)):
        for a in range(s, e, 1 << 18):
            got = grad[a:min(e, a + (1 << 18))].double() * rows
            ref = part[a - s:min(e, a + (1 << 18)) - s].double() * n
            err = (got - ref).abs() - 2.0 ** -8 * (got.abs() + ref.abs()) * (1 + 2.0 ** -7)
            assert float(err.max()) <= 8 * U


@pytest.mark.gpu
def test_no_gradient_is_formed_where_none_is_recorded(cuda_device):
    """An evaluation of a model's parameters under no_grad: no room for the weight's gradient
    (32 MB in fp32) is taken, the logits' chunk and small arrays apart."""
    h, w, b, values, tokens, lse = linear_case(2, 32, 512, 16384, 4, torch.bfloat16)
    w, b = torch.nn.Parameter(w), torch.nn.Parameter(b)
    with torch.no_grad():
        chunked_linear_distillation(h, w, b, values, tokens, teacher_lse=lse)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        chunked_linear_distillation(h, w, b, values, tokens, teacher_lse=lse)
        assert torch.cuda.max_memory_allocated() - before < 32 * 16384 * 4 + (1 << 20)
        x = torch.nn.Parameter(torch.randn(4096, 5000, device=cuda_device))  # formed ahead otherwise
        k = torch.zeros(4096, 1, device=cuda_device, dtype=torch.int64)
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        distillation_from_logits(x, torch.zeros(4096, 1, device=cuda_device), k)
        assert torch.cuda.max_memory_allocated() - before < 1 << 20


@pytest.mark.gpu
def test_gradient_matches_differences(cuda_device):
    """Central differences of the definition in 64 bits, steps of 1e-6 (errors near 1e-9)."""
    x, values, tokens, lse = case(21, 6, 257, 9, torch.float32, True, 1.5)
    d = torch.randn(6, 257, generator=torch.Generator().manual_seed(2), dtype=torch.float64)
    _, g = run(x, values, tokens, lse, 1.5)
    f = lambda v: reference(v, values, tokens, 1.5, lse)[0]  # noqa: E731
    xd, step = x.double().cpu(), 1e-6
    want = (f(xd + step * d) - f(xd - step * d)) / (2 * step)
    assert abs(float((g.double().cpu() * d).sum()) - want) <= 1e-5


@pytest.mark.gpu
def test_bad_tokens_are_reported(cuda_device, monkeypatch):
    x, values, tokens, _ = case(5, 6, 40, 4, torch.float32)
    tokens[3, 2] = 40
    loss, g = run(x, values, tokens, None)
    assert math.isnan(float(loss.detach())) and torch.isnan(g).all(1).tolist() == [False] * 3 + [True] + [False] * 2
    with pytest.raises(RuntimeError, match="error word"):
        check_errors()
    monkeypatch.setenv("DABSN_HIP_ERROR_CHECK", "sync")
    with pytest.raises(RuntimeError, match="outside"):
        run(x, values, tokens, None)
    monkeypatch.delenv("DABSN_HIP_ERROR_CHECK")
    check_errors()


# ---- from hidden rows ------------------------------------------------------------------------
def linear_case(seed, n, H, V, K, dtype, bias=True, rest=True):
    g = torch.Generator().manual_seed(seed)
    h = torch.randn(n, H, generator=g).to(dtype)
    w = (torch.randn(V, H, generator=g) * 2 / H ** 0.5).to(dtype)
    b = torch.randn(V, generator=g).to(dtype) if bias else None
    teacher = torch.nn.functional.linear(h.float(), w.float()) + torch.randn(n, V, generator=g)
    values, tokens = teacher.topk(K, dim=1)
    lse = torch.logsumexp(teacher, 1) if rest else None
    tokens[n // 2] = -100
    return [v if v is None else v.cuda() for v in (h, w, b, values, tokens, lse)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,H,V,K,budget,bias,rest", [
    (2, 3, 5, 2, None, True, True), (70, 48, 33, 5, 16 * 33, True, False),
    (300, 200, 1001, 20, 40 * 1001, False, True), (513, 73, 4099, 64, 1 << 18, True, True),
    (130, 8, 700, 128, None, True, False)])
def test_linear_form_matches_the_definition(cuda_device, n, H, V, K, budget, bias, rest, dtype):
    """One chunk, chunks in a group, groups with a shorter last one, odd sizes. The logits' error
    e (``logit_error``) shifts the loss by at most 2 e; a gradient's terms p and q relative to p
    by 2 e, a random sum over rows or words, so in the norm 4 e and the row kernel's error, the
    products' own n + V + H additions of u, for bf16 the fp16 rows' 2^-11 and one rounding, 2^-8.
    The gradient is the difference p - q: its norm against the one of p and q together, which the
    errors go by, enters as their quotient."""
    h, w, b, values, tokens, lse = linear_case(n + V, n, H, V, K, dtype, bias, rest)
    leaves = [x if x is None else x.clone().requires_grad_(True) for x in (h, w, b)]
    loss = chunked_linear_distillation(*leaves, values, tokens, teacher_lse=lse, chunk_budget=budget)
    x = h.double().cpu() @ w.double().cpu().t() + (0.0 if b is None else b.double().cpu())
    ref, d, tol_loss, _ = reference(x, values, tokens, 1.0, lse)
    e = float(logit_error(h, w, b).max())
    assert abs(float(loss.detach()) - ref) <= tol_loss + 2 * e
    got = torch.autograd.grad(loss * 2.0, [v for v in leaves if v is not None])
    want = [d @ w.double().cpu(), d.t() @ h.double().cpu()] + ([] if b is None else [d.sum(0)])
    p = torch.softmax(x, 1) / n
    both = max(1.0, float((p + (p - d * 1.0).abs()).norm() / d.norm()))
    tol = both * (4 * e + U * (4 * sum_error(V) + 900 + n + V + H)
                  + (2.0 ** -11 if dtype == torch.bfloat16 else 0))
    for a, c in zip(got, want):
        # a product's sum may cancel: against the norm of its terms' magnitudes
        err = float((a.double().cpu() / 2 - c).norm())
        assert a.dtype == dtype
        assert err <= (tol * 4 + (2.0 ** -8 if dtype == torch.bfloat16 else 0)) * float(c.norm()), (err, float(c.norm()))


@pytest.mark.gpu
@pytest.mark.parametrize("hs,ws", [(1e-30, 1.0), (1.0, 1e-30), (1e25, 1e-25), (1e-38, 1e38), (0.0, 1.0)])
def test_linear_form_of_large_and_small_values(cuda_device, hs, ws):
    """Hidden rows and weights far outside fp16's range (powers of two aside the copies hold their
    bits), bf16 subnormals, and zeros: gradients within 1e-2 of the definition in the norm (2^-8 and
    some of the products' rounding), those below fp32's normal range apart."""
    h, w, b, values, tokens, lse = linear_case(9, 60, 32, 200, 8, torch.bfloat16)
    h, w = (h.double() * hs).to(torch.bfloat16), (w.double() * ws).to(torch.bfloat16)
    leaves = [x.requires_grad_(True) for x in (h, w, b)]
    loss = chunked_linear_distillation(*leaves, values, tokens, teacher_lse=lse)
    x = h.double().cpu() @ w.double().cpu().t() + b.double().cpu()
    ref, d, _, _ = reference(x.detach(), values, tokens, 1.0, lse)
    assert abs(float(loss.detach()) - ref) <= 1e-5 * abs(ref)
    got = torch.autograd.grad(loss, leaves)
    want = [d @ w.detach().double().cpu(), d.t() @ h.detach().double().cpu(), d.sum(0)]
    for a, c in zip(got, want):
        assert bool(torch.isfinite(a).all())
        assert float((a.double().cpu() - c).norm()) <= 1e-2 * float(c.norm()) + 1e-36


@pytest.mark.gpu
def test_weights_that_are_not_the_rows(cuda_device):
    """A teacher_lse far below its row's makes the loss NaN and is reported."""
    x, values, tokens, lse = case(5, 6, 40, 4, torch.float32, True)
    lse[2] -= 8
    loss, _ = run(x, values, tokens, lse)
    assert math.isnan(float(loss.detach()))
    with pytest.raises(RuntimeError, match="error word"):
        check_errors()


@pytest.mark.gpu
def test_linear_form_parts_modes_and_memory(cuda_device):
    h, w, b, values, tokens, lse = linear_case(1, 96, 64, 1000, 16, torch.bfloat16)
    kw = dict(teacher_lse=lse, chunk_budget=7 * 1000)
    leaves = [v.clone().requires_grad_(True) for v in (h, w, b)]
    loss = chunked_linear_distillation(*leaves, values, tokens, **kw)
    full = torch.autograd.grad(loss, leaves, retain_graph=True)
    again = torch.autograd.grad(loss, leaves)
    assert all(torch.equal(x, y) for x, y in zip(full, again))
    for i in range(3):  # each alone: a frozen body, a frozen readout, only a bias
        some = [v.clone().requires_grad_(k == i) for k, v in enumerate((h, w, b))]
        one = chunked_linear_distillation(*some, values, tokens, **kw)
        assert torch.equal(one, loss)
        assert torch.equal(torch.autograd.grad(one, some[i])[0], full[i])
    with torch.no_grad():
        assert torch.equal(chunked_linear_distillation(h, w, b, values, tokens, **kw), loss)
    cube = chunked_linear_distillation(h.view(4, 24, 64), w, b, values.view(4, 24, 16),
                                       tokens.view(4, 24, 16), teacher_lse=lse.view(4, 24),
                                       chunk_budget=7 * 1000)
    assert torch.equal(cube, loss)
    with torch.autocast("cuda", torch.bfloat16):
        cast = chunked_linear_distillation(h.float(), w.float(), b.float(), values, tokens, **kw)
    assert torch.equal(cast, loss)
    empty = chunked_linear_distillation(h[:0].requires_grad_(True), leaves[1], leaves[2], values[:0],
                                        tokens[:0])
    ge = torch.autograd.grad(empty, leaves[1:])
    assert float(empty.detach()) == 0 and all(float(g.float().abs().max()) == 0 for g in ge)


# ---- as a user's program runs them -----------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("linear", [False, True])
def test_capture_and_replay(cuda_device, linear):
    from test_capture import _capture, _replays

    token_logprobs(torch.zeros(1, 4, device=cuda_device))  # the error word exists before
    if linear:
        cases = [linear_case(s, 90, 64, 1000, 16, torch.bfloat16) for s in (1, 2, 3)]
    else:
        cases = [case(s, 40, 2050, 16, torch.bfloat16, True) for s in (1, 2, 3)]
    static = [v.clone() for v in cases[0]]

    def go(v):
        if linear:
            leaves = [x.detach().requires_grad_(True) for x in v[:3]]
            loss = chunked_linear_distillation(*leaves, v[3], v[4], teacher_lse=v[5],
                                               chunk_budget=20 * 1000)
        else:
            leaves = [v[0].detach().requires_grad_(True)]
            loss = distillation_from_logits(leaves[0], v[1], v[2], teacher_lse=v[3], temperature=2.0)
        return [loss.detach(), *torch.autograd.grad(loss, leaves)]

    graph, outs = _capture(lambda: go(static))
    _replays(graph, outs, static, cases[1:] + cases[:1], go)


@pytest.mark.gpu
def test_a_student_learns_from_a_teachers_scores(cuda_device):
    """The run of all operators together: a teacher model scores a text, its alternatives' log
    probabilities (normalised, so their log-sum-exp is 0) are the student's targets, and the
    student's gradients, the scaled embedding's and the tied readout's among them, equal those of
    the definition written with torch's own operations on the same student: fp32 throughout,
    sums of some thousand terms, so 1e-4 in the norm."""
    torch.manual_seed(0)
    ids = torch.randint(0, 61, (2, 24), device=cuda_device)
    teacher = dabsn_amd.DABSNSequenceLM(61, 48, depth=1).cuda()
    with torch.no_grad():
        teacher.readout.weight.mul_(4.0)
        scores = teacher.token_logprobs(ids, top=10)
    student = dabsn_amd.DABSNSequenceLM(61, 32, depth=1, embed_scale=32 ** 0.5, tie_embeddings=True).cuda()
    lse = torch.zeros(2, 24, device=cuda_device)
    loss = student.distillation_loss(ids, scores.top_logprobs, scores.top_indices, teacher_lse=lse)
    loss.backward()
    got = {n: p.grad.clone() for n, p in student.named_parameters() if p.grad is not None}
    student.zero_grad()
    h = student.backbone(torch.nn.functional.embedding(ids, student.embed.weight) * 32 ** 0.5)
    logp = torch.log_softmax(student.readout(h).double(), dim=-1)
    q = scores.top_logprobs.double().exp()
    p = logp.gather(2, scores.top_indices)
    rest = 1 - q.sum(-1)
    hit = torch.zeros_like(logp).scatter_(2, scores.top_indices, 1.0)
    left = (logp.exp() * (1 - hit)).sum(-1)
    want = ((q * (scores.top_logprobs - p)).sum(-1) + rest * (rest.log() - left.log())).mean()
    want.backward()
    assert abs(float(loss.detach()) - float(want.detach())) <= 1e-5 * max(1.0, float(want.detach()))
    scale = max(float(p.grad.norm()) for p in student.parameters() if p.grad is not None)
    for n, prm in student.named_parameters():
        if prm.grad is not None:
            err = float((got[n] - prm.grad).norm())
            assert err <= 1e-4 * max(float(prm.grad.norm()), 1e-3 * scale), n
