"""The scaled token embedding and its table's gradient.

The forward is one fp32 product and one rounding, so it equals torch's expression bit for bit.
The gradient of a word is a sum of c fp32 terms in some fixed grouping, c - 1 additions of
u = 2^-24 each relative to the terms' magnitudes, a product and one rounding (u, or 2^-8 for
bf16): |error| <= scale * u (c + 1) * sum |g| + rounding * |value|."""

from __future__ import annotations

import math

import pytest
import torch

import dabsn_amd
from dabsn_amd import scaled_embedding
from dabsn_amd.kernels import check_errors

U = 2.0 ** -24


@pytest.mark.parametrize("call,error,match", [
    (lambda: scaled_embedding(torch.zeros(3).long(), torch.zeros(5, 4).half()), TypeError, "float32"),
    (lambda: scaled_embedding(torch.zeros(3), torch.zeros(5, 4)), TypeError, "int64 or int32"),
    (lambda: scaled_embedding(torch.zeros(3).long(), torch.zeros(5)), ValueError, "expected weight"),
    (lambda: scaled_embedding(torch.zeros(3).long(), torch.zeros(0, 4)), ValueError, "vocabulary"),
    (lambda: scaled_embedding(torch.zeros(3).long(), torch.zeros(5, 0)), ValueError, "expected weight"),
    (lambda: scaled_embedding(torch.zeros(3).long(), torch.zeros(5, 4), scale=math.inf), ValueError,
     "scale"),
    (lambda: scaled_embedding(torch.zeros(3).long(), torch.zeros(5, 4), padding_idx=5), ValueError,
     "padding_idx"),
    (lambda: scaled_embedding(torch.zeros(3).long(), torch.zeros(5, 4)), RuntimeError, "device"),
])
def test_refusals(call, error, match):
    with pytest.raises(error, match=match):
        call()


def test_library_refuses_bad_arguments_before_it_launches():
    from dabsn_amd import _lib

    lib, one = _lib.load(), 1 << 20
    for dtype, n, V, H, ld in ((2, 1, 5, 4, 4), (0, -1, 5, 4, 4), (0, 1, 0, 4, 4), (0, 1, 5, 0, 4),
                               (0, 1, 5, 4, 3), (0, 1 << 31, 5, 4, 4), (0, 1, 5, 1 << 24, 1 << 24)):
        assert lib.dabsn_hip_embedding_fwd(dtype, n, V, H, one, one, ld, 1.0, one, one, None) == -2
    assert lib.dabsn_hip_embedding_workspace_bytes(-1, 5, 4) == 0
    need = lib.dabsn_hip_embedding_workspace_bytes(5000, 60, 64)
    assert need > 0
    assert lib.dabsn_hip_embedding_bwd(0, 5000, 60, 64, one, -1, one, 1.0, one, one, need - 1, None) == -2
    assert lib.dabsn_hip_embedding_bwd(0, 5000, 60, 64, None, -1, one, 1.0, one, one, need, None) == -2


def case(seed, n, V, H, dtype, skew):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(V, H, generator=g).to(dtype)
    if skew == "one":
        ids = torch.full((n,), V // 2)
    elif skew == "zipf":
        share = 1.0 / (torch.arange(V) + 2.7)
        ids = torch.multinomial(share, n, replacement=True, generator=g) if n else torch.zeros(0).long()
    elif skew == "sorted":
        ids = torch.randint(0, V, (n,), generator=g).sort().values
    else:
        ids = torch.randint(0, V, (n,), generator=g)
    grad = torch.randn(n, H, generator=g).to(dtype)
    return ids.cuda(), w.cuda(), grad.cuda()


def check_grad(got, ids, grad, V, scale, padding=None):
    keep = (ids >= 0) & (ids < V)
    if padding is not None:
        keep &= ids != padding
    i, g = ids[keep], grad[keep].double()
    want = torch.zeros(V, grad.shape[1], dtype=torch.float64, device=g.device).index_add_(0, i, g)
    mag = torch.zeros_like(want).index_add_(0, i, g.abs())
    count = torch.bincount(i, minlength=V).double()[:, None]
    rnd = U if grad.dtype == torch.float32 else 2.0 ** -8
    s32 = float(torch.tensor(scale, dtype=torch.float32))
    err = (got.double() - s32 * want).abs()
    bound = abs(s32) * U * (count + 1) * mag + rnd * (abs(s32) * want.abs() * (1 + 2 ** -10)) + 2.0 ** -126
    assert got.dtype == grad.dtype
    assert bool((err <= bound).all()), float((err - bound).max())
    assert float(got[count[:, 0] == 0].float().abs().sum()) == 0


SIZES = [(1, 1, 1), (2, 5, 3), (63, 60, 8), (64, 60, 24), (65, 1000, 40), (256, 32000, 64),
         (4096, 60, 33), (4097, 60, 33), (4097, 1023, 8), (5000, 1024, 16), (10000, 70000, 40),
         (9000, 2000000, 2), (70001, 65, 513), (40000, 1100, 8)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("skew", ["even", "zipf", "one", "sorted"])
@pytest.mark.parametrize("n,V,H", SIZES)
def test_lookup_and_gradient(cuda_device, n, V, H, skew, dtype):
    ids, w, grad = case(n + V + H, n, V, H, dtype, skew)
    scale = 1.0 if skew == "one" else math.sqrt(H) * 0.7
    leaf = w.clone().requires_grad_(True)
    out = scaled_embedding(ids, leaf, scale=scale)
    s32 = torch.tensor(scale, dtype=torch.float32, device=ids.device)
    assert torch.equal(out.detach(), (w.float()[ids] * s32).to(dtype))
    (got,) = torch.autograd.grad(out, leaf, grad, retain_graph=True)
    check_grad(got, ids, grad, V, scale)
    (again,) = torch.autograd.grad(out, leaf, grad)
    assert torch.equal(got, again)
    check_errors()


@pytest.mark.gpu
def test_sum_keeps_token_order(cuda_device):
    """A word's terms 2^24, 1, -2^24 in fp32 give 0 in token order (2^24 + 1 rounds to even) and 1
    in others; tokens of other words between them. Few and many tokens (both sorts)."""
    for n in (300, 9000):
        ids = torch.randint(1, 50, (n,), generator=torch.Generator().manual_seed(n))
        at = torch.tensor([7, n // 2, n - 3])
        ids[at] = 0
        grad = torch.zeros(n, 16)
        grad[at] = torch.tensor([2.0 ** 24, 1.0, -2.0 ** 24])[:, None]
        w = torch.zeros(50, 16, device=cuda_device, requires_grad=True)
        (got,) = torch.autograd.grad(scaled_embedding(ids.cuda(), w), w, grad.cuda())
        assert float(got.abs().max()) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_padding_shapes_strides_and_index_types(cuda_device, dtype):
    ids, w, grad = case(3, 5000, 700, 40, dtype, "zipf")
    for pad in (0, -700, 699):
        leaf = w.clone().requires_grad_(True)
        out = scaled_embedding(ids, leaf, padding_idx=pad)
        assert torch.equal(out.detach(), w[ids])  # the padding row is looked up as it is
        (got,) = torch.autograd.grad(out, leaf, grad)
        check_grad(got, ids, grad, 700, 1.0, pad % 700)
    cube = scaled_embedding(ids.view(50, 100).int(), w, scale=2.0)
    assert cube.shape == (50, 100, 40) and torch.equal(cube.view(-1, 40), w[ids] * 2)
    assert scaled_embedding(ids[3], w).shape == (40,)
    turned = scaled_embedding(ids.view(50, 100).t(), w)
    assert torch.equal(turned, w[ids.view(50, 100).t()])
    wide = torch.zeros(700, 91, device=cuda_device, dtype=dtype)
    wide[:, 3:43] = w
    leaf = wide.requires_grad_(True)
    out = scaled_embedding(ids, leaf[:, 3:43], scale=0.5)
    assert torch.equal(out.detach(), w[ids] * 0.5)
    (got,) = torch.autograd.grad(out, leaf, grad)
    check_grad(got[:, 3:43], ids, grad, 700, 0.5)
    tall = w.t().contiguous().t()  # columns first
    assert torch.equal(scaled_embedding(ids, tall), w[ids])
    up = torch.randn(40, device=cuda_device).to(dtype).expand(5000, 40)  # an expanded gradient
    leaf = w.clone().requires_grad_(True)
    (got,) = torch.autograd.grad(scaled_embedding(ids, leaf), leaf, up)
    check_grad(got, ids, up, 700, 1.0)
    leaf = w.clone().requires_grad_(True)
    none = scaled_embedding(ids[:0], leaf)
    (got,) = torch.autograd.grad(none, leaf, none.detach())
    assert none.shape == (0, 40) and float(got.float().abs().sum()) == 0


@pytest.mark.gpu
def test_bad_ids_are_reported(cuda_device, monkeypatch):
    ids, w, grad = case(3, 300, 70, 24, torch.float32, "even")
    ids[5], ids[9] = 70, -1
    leaf = w.clone().requires_grad_(True)
    out = scaled_embedding(ids, leaf)
    rows = torch.isnan(out).all(1)
    assert rows.nonzero()[:, 0].tolist() == [5, 9]
    (got,) = torch.autograd.grad(out, leaf, grad)
    check_grad(got, ids, grad, 70, 1.0)
    with pytest.raises(RuntimeError, match="error word"):
        check_errors()
    monkeypatch.setenv("DABSN_HIP_ERROR_CHECK", "sync")
    with pytest.raises(RuntimeError, match="outside"):
        scaled_embedding(ids, w)
    monkeypatch.delenv("DABSN_HIP_ERROR_CHECK")
    check_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("n,V", [(200, 60), (3000, 5000), (9000, 60), (9000, 5000)])
def test_capture_and_replay(cuda_device, n, V):
    from test_capture import _capture, _replays

    scaled_embedding(torch.zeros(1, device=cuda_device).long(), torch.zeros(2, 8, device=cuda_device))
    cases = [case(s, n, V, 72, torch.bfloat16, "zipf") for s in (1, 2, 3)]
    static = [v.clone() for v in cases[0]]

    def go(v):
        leaf = v[1].detach().requires_grad_(True)
        out = scaled_embedding(v[0], leaf, scale=3.0)
        return [out.detach(), *torch.autograd.grad(out, leaf, v[2])]

    graph, outs = _capture(lambda: go(static))
    _replays(graph, outs, static, cases[1:] + cases[:1], go)


@pytest.mark.gpu
def test_two_streams(cuda_device):
    ids, w, grad = case(5, 20000, 3000, 64, torch.float32, "zipf")
    leaf = w.clone().requires_grad_(True)
    (want,) = torch.autograd.grad(scaled_embedding(ids, leaf), leaf, grad)
    torch.cuda.synchronize()
    got = []
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(2):
        for s in streams:
            with torch.cuda.stream(s):
                got += torch.autograd.grad(scaled_embedding(ids, leaf), leaf, grad)
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


@pytest.mark.gpu
def test_a_model_with_a_scaled_embedding(cuda_device):
    """``embed_scale`` multiplies what the blocks see, in training, evaluation and with a carried
    memory, whose file remembers it; without it the plain embedding runs."""
    torch.manual_seed(0)
    m = dabsn_amd.DABSNSequenceLM(50, 32, depth=1, embed_scale=3.0).cuda()
    plain = dabsn_amd.DABSNSequenceLM(50, 32, depth=1).cuda()
    plain.load_state_dict(m.state_dict())
    with torch.no_grad():
        plain.embed.weight.mul_(3.0)
        ids = torch.randint(0, 50, (2, 20), device=cuda_device)
        assert torch.equal(m(ids), plain(ids))
        a, mem = dabsn_amd.forward_with_memory(m, ids, extend=True)
        b, _ = dabsn_amd.forward_with_memory(plain, ids, extend=True)
        assert torch.equal(a, b)
    assert mem.fingerprint["embed_scale"] == 3.0
    with pytest.raises(ValueError, match="embed_scale"):
        dabsn_amd.forward_with_memory(plain, ids, mem)
