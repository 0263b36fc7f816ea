"""Rows of a vocabulary where 32 bits are short: masks of large finite numbers, students far from
their teacher, tokens that are nearly certain, against the definitions in 64 bits of test_scoring.py
and test_distill.py, with the tolerances derived there.

Where a token is nearly certain the tolerance is relative (``sure``), u = 2^-24: with R = the other
words' mass over its own, log p = -ln(1 + R). A term of R carries the rounding of its exponent's
argument, u |z - max z| of itself, the same again from the steps of the running reference, 3 u of
exponential and product, and the sum S u (``sum_error``); the rounding of 1 / T is taken out of R, and
stays in the entropy's -sum p log p once more, u |z - max z|. So log p and 1 - p are off by at most
u (3 spread + S + 32) of themselves, and so is the entropy, a sum of terms of one sign.
"""

from __future__ import annotations

import math

import pytest
import torch

from dabsn_amd import (chunked_linear_distillation, chunked_linear_token_logprobs,
                       distillation_from_logits, token_logprobs)
from test_distill import check, reference as distill_reference
from test_scoring import (U, check_forward, check_grad, logit_error, logits_of, reference,
                          reference_grad, sum_error)

INF = math.inf
FILLS = [-1e9, -1e10, -1e20, -1e30, "lowest", -6e7, -4e7]
TEMPERATURES = [0.5, 1.0, 1.5, 2.0, 2.5, 3.0, 5.0, 8.0]


def masked_rows(V, dtype, fill, seed):
    """Rows: nine words of ten at the fill; all but the last; all; the fill beside -inf; all but
    word 3 of those before the row's second half; an unmasked one."""
    fill = torch.finfo(dtype).min if fill == "lowest" else fill
    x, _ = logits_of(seed, 6, V, dtype, device="cpu")
    drop = torch.rand(V, generator=torch.Generator().manual_seed(seed)) < 0.9
    drop[5] = False
    x[0, drop] = fill
    x[1, :-1] = fill
    x[2] = fill
    x[3, drop] = fill
    x[3, ::3] = -INF
    x[4, :V // 2] = fill
    x[4, 3] = 1.0
    return x.cuda(), torch.tensor([5, V - 1, 2, 5, 3, 7]).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("fill", FILLS)
@pytest.mark.parametrize("V", [61, 300, 9001])
def test_scores_of_rows_masked_by_large_numbers(cuda_device, V, fill, dtype):
    x, t = masked_rows(V, dtype, fill, V)
    g = torch.Generator().manual_seed(1)
    gl, ge = torch.randn(6, generator=g).cuda(), torch.randn(6, generator=g).cuda()
    for T in TEMPERATURES:
        check_forward(token_logprobs(x, t, top=9, temperature=T), x, t, 9, T)
        leaf = x.clone().requires_grad_(True)
        r = token_logprobs(leaf, t, top=9, temperature=T)
        (got,) = torch.autograd.grad((r.logprobs, r.entropy), leaf, (gl, ge))
        check_grad(got, *reference_grad(x, t, 0, T, gl, ge, None), V, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [61, 300, 9001])
def test_scores_of_large_positive_logits(cuda_device, V, dtype):
    """Logits around 1e8, 1e10 and 1e30, all of a row or one word in seven."""
    for k, big in enumerate((1e8, 1e10, 1e30)):
        x, t = logits_of(k, 5, V, dtype)
        x[0] = (x[0].float() * big / 100 + big).to(dtype)
        x[1, ::7] = (x[1, ::7].float() * big / 100 + big).to(dtype)
        x[2, 4] = big
        x[3] = big
        t[:] = torch.tensor([1, 7, 4, 0, 3])
        for T in (0.5, 1.0, 2.5):
            check_forward(token_logprobs(x, t, top=3, temperature=T), x, t, 3, T)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("fill", FILLS)
@pytest.mark.parametrize("V", [61, 300, 9001])
def test_distillation_of_rows_masked_by_large_numbers(cuda_device, V, fill, rest, dtype):
    """A listed word is ruled out in no row (its loss would be the fill itself); row 4 has no list."""
    x, _ = masked_rows(V, dtype, fill, V)
    x = x[[0, 1, 3, 4, 2, 5]]
    words = [(x[r].float() > -1e4).nonzero()[:, 0] for r in range(6)]
    words[4] = torch.arange(3, device=x.device)
    K = 4
    tokens = torch.full((6, K), -100, device=x.device)
    for r, w in enumerate(words):
        if r != 4:
            tokens[r, :min(K, len(w))] = w[:K]
    values = torch.randn(6, K, generator=torch.Generator().manual_seed(3)).cuda()
    for T in TEMPERATURES:
        lse = (torch.logsumexp(values.double() / T, 1) + 0.4).float() if rest else None
        leaf = x.clone().requires_grad_(True)
        loss = distillation_from_logits(leaf, values, tokens, temperature=T, teacher_lse=lse)
        (got,) = torch.autograd.grad(loss, leaf)
        check(loss, got, distill_reference(x, values, tokens, T, lse), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("fill", [-1e10, -1e30])
def test_many_masked_rows_with_the_gradient_formed_ahead(cuda_device, fill):
    """Enough logits that loss and gradient are formed together (2100 x 8200): bit for bit what a
    factor of 2 forms again, its first rows the definition's."""
    x, t = logits_of(5, 2100, 8200, torch.bfloat16)
    keep = torch.rand(2100, 8200, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda") < 0.1
    x = torch.where(keep, x, fill).to(torch.bfloat16)
    values, tokens = x.float().topk(6, dim=1)
    leaf = x.requires_grad_(True)
    loss = distillation_from_logits(leaf, values, tokens, temperature=2.0)
    (g1,) = torch.autograd.grad(loss, leaf, retain_graph=True)
    (g2,) = torch.autograd.grad(loss * 2, leaf)
    assert math.isfinite(float(loss.detach())) and torch.equal(g2 / 2, g1)
    _, grad, _, tol = distill_reference(x[:6], values[:6], tokens[:6], 2.0)
    grad, tol = grad * 6 / 2100, tol * 6 / 2100
    err = (g1[:6].double().cpu() - grad).abs()
    assert bool((err <= tol + 2.0 ** -8 * (grad.abs() + tol) * (1 + 2.0 ** -10) + 2.0 ** -126).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [60, 128, 300, 9001])
@pytest.mark.parametrize("margin,T", [(80.0, 1.0), (100.0, 1.0), (200.0, 1.0), (600.0, 1.0), (10.0, 0.05),
                                      (150.0, 0.7)])
def test_a_student_far_from_the_rest(cuda_device, V, margin, T, dtype):
    """The words off the list lie ``margin`` logits below the listed ones, where fp32 holds no mass
    of theirs beside the listed words': the loss still grows with the distance, and their gradient
    is theirs. Nothing is left out until 64 bits hold the mass as 0 (row 3, 2000 below)."""
    g = torch.Generator().manual_seed(V)
    x = torch.randn(5, V, generator=g)
    tokens = torch.stack([torch.randperm(V, generator=g)[:7] for _ in range(5)])
    x.scatter_(1, tokens, x.gather(1, tokens) + margin)
    x[3].scatter_(0, tokens[3], 2000.0 * T)
    x[4, tokens[4, 0]] = 3 * margin
    tokens[1, 3] = tokens[1, 2]
    tokens[2, 4:] = -100
    x = x.to(dtype).cuda()
    values = torch.randn(5, 7, generator=g)
    lse = (torch.logsumexp(values.double() / T, 1) + 0.5).float().cuda()
    values, tokens = values.cuda(), tokens.cuda()
    leaf = x.clone().requires_grad_(True)
    loss = distillation_from_logits(leaf, values, tokens, temperature=T, teacher_lse=lse)
    (got,) = torch.autograd.grad(loss, leaf)
    check(loss, got, distill_reference(x, values, tokens, T, lse), dtype)


def far_case(V, T, rest):
    """Logits around 3000 and a teacher near them."""
    g = torch.Generator().manual_seed(V)
    x = 3000 + torch.randn(4, V, generator=g)
    teacher = x + 0.5 * torch.randn(4, V, generator=g)
    values, tokens = teacher.topk(8, dim=1)
    lse = (torch.logsumexp(teacher.double() / T, 1).float() + 0.01).cuda() if rest else None
    return x.cuda(), values.cuda(), tokens.cuda(), lse


@pytest.mark.gpu
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("T", [1.0, 2.0])
@pytest.mark.parametrize("V", [50, 300, 9001])
def test_gradients_of_logits_far_from_zero(cuda_device, V, T, rest):
    """Off the list p_j a, p off by u (3 spread + S + 32) of itself (S = ``sum_error``) wherever the
    logits lie: log2 e / T is rounded by 1e-8 of itself, which at 3000 alone would be 4e-5."""
    x, values, tokens, lse = far_case(V, T, rest)
    leaf = x.clone().requires_grad_(True)
    loss = distillation_from_logits(leaf, values, tokens, temperature=T, teacher_lse=lse)
    (got,) = torch.autograd.grad(loss, leaf)
    _, grad, _, _ = distill_reference(x, values, tokens, T, lse)
    z = x.double().cpu() / T
    tol = U * (3 * float(z.amax() - z.amin()) + sum_error(V) + 32)
    err = (got.double().cpu() - grad).abs() / (T / 4)
    p = torch.softmax(z, 1)
    scale = grad.abs() / (T / 4)
    listed = torch.zeros_like(p, dtype=torch.bool).scatter_(1, tokens.cpu(), True)
    if rest:  # a = Q - q_r / p_r, a difference
        left = torch.where(listed, 0.0, p).sum(1, keepdim=True)
        scale = scale + 2 * p / left
    assert bool((err <= tol * scale + 2 * U * scale)[~listed].all())


@pytest.mark.gpu
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("T", [0.7, 1.1, 3.3])
@pytest.mark.parametrize("V", [50, 300, 9001])
def test_the_temperature_has_64_bits(cuda_device, V, T, rest):
    """Logits around 3000: a temperature rounded to 32 bits (0.7 by 1.7e-8 of itself) would take the
    teacher's weights off by 1e-5 to 7e-5 of themselves against its normaliser. They are 64-bit values
    here; the student's log probabilities are off by u (3 spread + S + 32) (S = ``sum_error``)."""
    x, values, tokens, lse = far_case(V, T, rest)
    leaf = x.clone().requires_grad_(True)
    loss = distillation_from_logits(leaf, values, tokens, temperature=T, teacher_lse=lse)
    (got,) = torch.autograd.grad(loss, leaf)
    ref, grad, _, _ = distill_reference(x, values, tokens, T, lse)
    z = x.double().cpu() / T
    tol = U * (3 * float(z.amax() - z.amin()) + sum_error(V) + 32)
    assert abs(float(loss.detach()) - ref) <= T * T * tol + 2 * U * ref
    p = torch.softmax(z, 1)
    bound = T / 4 * tol * (p + (p - grad * 4 / T).abs()) + 2 * U * grad.abs()
    assert bool(((got.double().cpu() - grad).abs() <= bound).all())


GAPS = [3.0, 5.0, 7.0, 9.0, 11.0, 13.0, 15.0, 17.0]  # log p from -5e-2 to -4e-8


def sure_rows(V, dtype, seed):
    """Rows whose token t lies a gap above the others' log-sum-exp."""
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(8, V, generator=g) * 1.5).to(dtype).float()
    t = torch.randint(0, V, (8,), generator=g)
    t[0], t[1] = 0, V - 1
    x.scatter_(1, t[:, None], -INF)
    x.scatter_(1, t[:, None], (torch.logsumexp(x, 1) + torch.tensor(GAPS))[:, None])
    return x.to(dtype).cuda(), t.cuda()


def sure(x, T):
    z = x.double().cpu() / T
    return U * (3 * (z.amax(1) - z.amin(1)) + sum_error(x.shape[1]) + 32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [1.0, 0.7])
@pytest.mark.parametrize("V", [50, 128, 300, 2050, 9001, 40000])
def test_scores_of_nearly_certain_tokens(cuda_device, V, T, dtype):
    x, t = sure_rows(V, dtype, V)
    lp, ent, _, _, _, p, logp = reference(x, t, 0, T)
    exact = -torch.log1p(torch.exp((x.double().cpu() - x.double().cpu().amax(1, keepdim=True)) / T)
                         .scatter(1, t.cpu()[:, None], 0.0).sum(1))  # the same, without cancellation
    tol = sure(x, T)
    leaf = x.clone().requires_grad_(True)
    r = token_logprobs(leaf, t, top=1, temperature=T)
    for got in (r.logprobs, r.top_logprobs[:, 0]):
        assert bool(((got.detach().double().cpu() - exact).abs() <= tol * exact.abs()).all())
    assert bool(((r.entropy.detach().double().cpu() - ent).abs() <= tol * ent + 1e-15).all())
    # The gradient at the token: (1 - p) / T of its log probability's, p (-log p - H) / T of the entropy's.
    rows = torch.arange(8)
    (g,) = torch.autograd.grad(r.logprobs.sum(), leaf, retain_graph=True)
    rnd = U if dtype == torch.float32 else 2.0 ** -8
    want = -torch.expm1(exact) / T
    assert bool(((g.double().cpu()[rows, t.cpu()] - want).abs() <= (tol + rnd * (1 + tol)) * want).all())
    (g,) = torch.autograd.grad(r.top_logprobs.sum(), leaf, retain_graph=True)
    assert bool(((g.double().cpu()[rows, t.cpu()] - want).abs() <= (tol + rnd * (1 + tol)) * want).all())
    (g,) = torch.autograd.grad(r.entropy.sum(), leaf)
    want = -exact.exp() * (exact + ent) / T
    size = exact.abs() + ent
    # (the factor's own rounding goes by the place of the largest logit, 2^-20 of 1, in fp32)
    assert bool(((g.double().cpu()[rows, t.cpu()] - want).abs()
                 <= (tol * size + 2.0 ** -43) / T + rnd * want.abs() * (1 + tol)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("T", [1.0, 0.7])
@pytest.mark.parametrize("V", [50, 128, 300, 2050, 9001, 40000])
def test_distillation_of_nearly_certain_tokens(cuda_device, V, T, rest):
    """A student near its teacher, both sure of a token: the gradient there is p - q, a difference of
    numbers near 1 that each hold an error of ``sure`` times 1 - p (q of the fp32 values' own)."""
    x, t = sure_rows(V, torch.float32, V)
    g = torch.Generator().manual_seed(V + 1)
    teacher = x.cpu() + 0.3 * torch.randn(8, V, generator=g)
    values, tokens = teacher.topk(6, dim=1)
    lse = torch.logsumexp(teacher.double() / T, 1).float().cuda() if rest else None
    values, tokens = values.cuda(), tokens.cuda()
    tol = sure(x, T)
    for r in range(8):  # a row each, so that each has its loss
        row = slice(r, r + 1)
        part = None if lse is None else lse[row]
        leaf = x[row].clone().requires_grad_(True)
        loss = distillation_from_logits(leaf, values[row], tokens[row], temperature=T, teacher_lse=part)
        (got,) = torch.autograd.grad(loss, leaf)
        ref, grad, _, _ = distill_reference(x[row], values[row], tokens[row], T, part)
        u = values[row].double().cpu() / T
        q = torch.exp(u - (torch.logsumexp(u, 1) if part is None else part.double().cpu())[:, None])
        z = x[row].double().cpu() / T
        p = torch.softmax(z, 1)
        w = p.gather(1, tokens[row].cpu())  # listed
        other = 1 - p.amax().item()  # 64 bits: to 1e-16
        # Loss: sum q (ln q - ln p): each ln p off by tol (1 - p) for the sure one, tol (|ln p| + 1) others.
        off = (q * torch.where(w > 0.5, other, w.log().abs() + 1)).sum() + max(0.0, 1 - float(q.sum())) * (
            1 + (w.log().abs().max() if rest else 0.0))
        assert abs(float(loss.detach()) - ref) <= T * T * (float(tol[r]) * float(off) + 1e-12) + U * ref * 2
        at = tokens[row].cpu()
        err = (got.double().cpu() - grad).abs().gather(1, at)
        bound = T * (float(tol[r]) * torch.where(w > 0.5, other, w) + 1e-15) + 2 * U * grad.abs().gather(1, at)
        assert bool((err <= bound).all()), (r, err, bound)


# ---- gradients of a bf16 readout ---------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("budget", [None, 64 * 1003])
def test_readout_gradients_of_words_that_are_never_likely(cuda_device, budget, rest):
    """Words whose probability is 1e-9 to 1e-15 in every row, word by word: a gradient's terms are off
    by the logits' error 2 e (``logit_error``), the softmax's, 2^-17 of the planes and n additions of
    u, each of the term itself, and the result by its rounding to bf16."""
    from test_distill import linear_case

    n, H, V = 300, 64, 1003
    h, w, b, values, tokens, lse = linear_case(3, n, H, V, 16, torch.bfloat16, rest=rest)
    b[:40] = -torch.linspace(14, 26, 40).to(torch.bfloat16)
    tokens[tokens < 40] = -100
    leaves = [v.clone().requires_grad_(True) for v in (h, w, b)]
    loss = chunked_linear_distillation(*leaves, values, tokens, teacher_lse=lse, chunk_budget=budget)
    _, gw, gb = torch.autograd.grad(loss, leaves)
    x = h.double().cpu() @ w.double().cpu().t() + b.double().cpu()
    _, d, _, _ = distill_reference(x, values, tokens, 1.0, lse)
    p = torch.softmax(x, 1)
    # The terms' magnitudes: p Q + p q_r / p_r + q.
    size = 2 * p / n + d.abs()
    tol = 4 * float(logit_error(h, w, b).max()) + U * (4 * sum_error(V) + 900 + n) + 2.0 ** -17
    hd = h.double().cpu()
    for got, want, terms in ((gw, d.t() @ hd, size.t() @ hd.abs()),
                             (gb[:, None], d.sum(0)[:, None], size.sum(0)[:, None])):
        err = (got.double().cpu() - want).norm(dim=1)
        bound = tol * terms.norm(dim=1) + 2.0 ** -8 * want.norm(dim=1) * (1 + 2.0 ** -8)
        assert bool((err <= bound)[:40].all()), (err / want.norm(dim=1))[:40]
        assert bool((err <= bound).all())


@pytest.mark.gpu
def test_readout_gradients_of_rows_that_are_nearly_certain(cuda_device):
    """Student and teacher sure of a token to 1e-10 and less: hidden gradients that small, row by row.
    Terms as above; an fp16 row holds them to 2^-11 of the row's size."""
    n, H, V = 24, 64, 1003
    g = torch.Generator().manual_seed(5)
    w = (torch.randn(V, H, generator=g) * 2 / H ** 0.5).to(torch.bfloat16).cuda()
    t = torch.randint(0, V, (n,), generator=g).cuda()
    wt = w[t].float()
    scale = torch.linspace(36, 52, n)[:, None].cuda()
    h = (wt * scale / wt.square().sum(1, keepdim=True)).to(torch.bfloat16)
    x = h.double().cpu() @ w.double().cpu().t()
    values, tokens = (x + 0.1 * torch.randn(n, V, generator=g).double()).float().topk(8, dim=1)
    leaf = h.clone().requires_grad_(True)
    loss = chunked_linear_distillation(leaf, w, None, values.cuda(), tokens.cuda())
    (got,) = torch.autograd.grad(loss, leaf)
    _, d, _, _ = distill_reference(x, values, tokens, 1.0, None)
    # p - q at the token itself, 2^-53 of 1 in 64 bits, is the others' sum: a row's gradient sums to 0.
    at = t.cpu()[:, None]
    d.scatter_(1, at, 0.0)
    d.scatter_(1, at, -d.sum(1, keepdim=True))
    q = torch.zeros_like(x).scatter_(1, tokens, torch.softmax(values.double(), 1))
    small = lambda v: torch.minimum(v, 1 - v)  # noqa: E731
    size = (small(torch.softmax(x, 1)) + small(q)) / n
    want = d @ w.double().cpu()
    assert float(want.norm(dim=1).max()) < 1e-6 and float(want.norm(dim=1).min()) < 1e-11
    norms = w.double().cpu().norm(dim=1)
    tol = 4 * float(logit_error(h, w, None).max()) + U * (4 * sum_error(V) + 900 + V) + 2.0 ** -10
    err = (got.double().cpu() - want).norm(dim=1)
    # The operator forms exp(log p) Q - q at the token in 64 bits: an exponential (an ulp, 2^-52), the
    # sum Q, a product and a difference, each of 2^-53 of numbers at most 1.
    own = 5 * 2.0 ** -53 / n * norms[t.cpu()]
    assert bool((err <= tol * (size @ norms) + own + 2.0 ** -8 * want.norm(dim=1)).all()), err / want.norm(dim=1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("fill", [-INF, -1e9, -1e30, "lowest"])
@pytest.mark.parametrize("V", [90, 1003])
def test_a_readout_whose_bias_rules_words_out(cuda_device, V, fill, dtype):
    """Scores and distillation from hidden rows with a third of the words ruled out by the bias: the
    definition's values (errors as in test_scoring.py and test_distill.py, logits off by e), and
    exact zeros in those words' gradients."""
    from test_distill import linear_case

    n, H = 70, 48
    fill = torch.finfo(dtype).min if fill == "lowest" else fill
    h, w, b, values, tokens, _ = linear_case(7, n, H, V, 8, dtype, rest=False)
    out = torch.arange(V, device="cuda") % 3 == 1
    b[out] = fill
    tokens[out[tokens.clamp(min=0)] & (tokens >= 0)] = -100
    t = torch.arange(n, device="cuda") % (V // 3) * 3
    x = h.double().cpu() @ w.double().cpu().t() + b.double().cpu()
    e = float(logit_error(h, w, torch.where(out, 0.0, b.float())).max())
    lp, ent, _, _, _, p, _ = reference(x, t, 0, 0.9)
    leaves = [v.clone().requires_grad_(True) for v in (h, w, b)]
    r = chunked_linear_token_logprobs(*leaves, t, temperature=0.9, chunk_budget=30 * V)
    z = x[:, ~out.cpu()] / 0.9
    spread, ln, S = float(z.amax() - z.amin()), math.log(V), sum_error(V)
    close = lambda a, c, tol: float((a.detach().double().cpu() - c).abs().max()) <= tol  # noqa: E731
    assert close(r.logprobs, lp, 2 * e / 0.9 + U * (8 * spread + 8 * ln + S))
    assert close(r.entropy, ent, 2 * e / 0.9 * (1 + ln) + U * (S * (1 + 2 * ln) + 8 * ln))
    loss = chunked_linear_distillation(*leaves, values, tokens, chunk_budget=30 * V)
    ref, d, tol, _ = distill_reference(x, values, tokens, 1.0)
    assert abs(float(loss.detach()) - ref) <= tol + 2 * e
    hd, wd = h.double().cpu(), w.double().cpu()
    _, F, _ = reference_grad(x, t, 0, 0.9, torch.ones(n), torch.ones(n), None)
    dense = reference_grad(x, t, 0, 0.9, torch.ones(n), torch.ones(n), None)[0]
    rnd = U if dtype == torch.float32 else 2.0 ** -8
    for total, g, size in ((r.logprobs.sum() + r.entropy.sum(), dense, F + dense.abs()),
                           (loss, d, 2 * p / n + d.abs())):
        got = torch.autograd.grad(total, leaves)
        rel = 8 * e * (1 + ln) + U * (4 * S + 900 + n + V + H) + (2.0 ** -10 if dtype != torch.float32 else 0)
        for a, want, terms in ((got[0], g @ wd, size @ wd.abs()), (got[1], g.t() @ hd, size.t() @ hd.abs()),
                               (got[2], g.sum(0), size.sum(0))):
            err = (a.double().cpu() - want).abs()
            assert bool((err <= rel * terms + rnd * want.abs() * (1 + rel) + 2.0 ** -126).all())
        assert float(got[1][out].float().abs().max()) == 0 == float(got[2][out].float().abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("gap", [20.0, 40.0, 60.0, 80.0])
def test_hidden_gradients_where_the_list_holds_nearly_all(cuda_device, gap):
    """A sure token and a list that leaves 1e-7 to 1e-5 of what it leaves: the fp16 rows' factor goes
    by a difference of nearly equal numbers and must not take an unlisted word out of range."""
    n, H, V = 64, 32, 600
    g = torch.Generator().manual_seed(int(gap))
    w = torch.zeros(V, H)
    w[:8] = torch.eye(8, H)
    w[8:] = torch.randn(V - 8, H, generator=g) * 0.02
    h = torch.zeros(n, H)
    h[:, 0] = gap
    h[:, 1:8] = -3.0 * torch.rand(n, 7, generator=g)  # listed, far above the rest
    b = torch.zeros(V)
    b[8:] = -torch.linspace(19, 23, V - 8)
    h, w, b = (v.to(torch.bfloat16).cuda() for v in (h, w, b))
    tokens = torch.arange(8).expand(n, 8).contiguous().cuda()
    values = (h.float() @ w.float().t())[:, :8] + 0.5 * torch.randn(n, 8, generator=g).cuda()
    leaf = h.clone().requires_grad_(True)
    loss = chunked_linear_distillation(leaf, w, b, values, tokens)
    (got,) = torch.autograd.grad(loss, leaf)
    x = h.double().cpu() @ w.double().cpu().t() + b.double().cpu()
    _, d, _, _ = distill_reference(x, values, tokens, 1.0, None)
    d[:, 0] = -d[:, 1:].sum(1)  # a row sums to 0; the difference p - q near 1 would not be exact here
    want = d @ w.double().cpu()
    q = torch.zeros_like(x).scatter_(1, tokens.cpu(), torch.softmax(values.double().cpu(), 1))
    small = lambda v: torch.minimum(v, 1 - v)  # noqa: E731
    size = (small(torch.softmax(x, 1)) + small(q)) / n
    norms = w.double().cpu().norm(dim=1)
    tol = 4 * float(logit_error(h, w, b).max()) + U * (4 * sum_error(V) + 900 + V) + 2.0 ** -10
    err = (got.double().cpu() - want).norm(dim=1)
    own = 5 * 2.0 ** -53 / n * norms[0]
    assert bool(torch.isfinite(got).all())
    assert bool((err <= tol * (size @ norms) + own + 2.0 ** -8 * want.norm(dim=1)).all()), err / want.norm(dim=1)
