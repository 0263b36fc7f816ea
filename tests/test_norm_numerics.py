"""The norms' backward with rows to add, as the MLP calls it, at every width, and of a shared weight."""

from __future__ import annotations

import pytest
import torch

from dabsn_amd import _lib, rms_norm
from dabsn_amd.kernels import dense, ops
from test_norm import SIZES, case, check


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,wdtype", [(torch.float32, torch.float32),
                                          (torch.bfloat16, torch.bfloat16),
                                          (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("layer", [True, False])
@pytest.mark.parametrize("rows,h", SIZES)
def test_backward_with_rows_to_add(cuda_device, rows, h, layer, dtype, wdtype):
    eps = 1e-5 if layer else 1e-6
    x, w, b, grad = case(rows + h, rows, h, dtype, wdtype, layer)
    add = torch.randn(rows, h, generator=torch.Generator().manual_seed(h)).to(dtype).cuda()
    out, stats = dense.norm(x, w, b, eps, layer, True)
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    db = torch.empty_like(w) if layer else None
    lib, p = _lib.load(), ops._p
    code = ops._code(dtype)
    nbytes = lib.dabsn_hip_norm_workspace_bytes(code, rows, h)
    ws = torch.empty(nbytes, device=cuda_device, dtype=torch.uint8)
    _lib.check(lib.dabsn_hip_norm_bwd(
        code, ops._code(wdtype), layer, rows, h, x.data_ptr(), h, w.data_ptr(), stats.data_ptr(),
        grad.data_ptr(), h, add.data_ptr(), dx.data_ptr(), dw.data_ptr(), p(db), ws.data_ptr(), nbytes,
        dense.stream(x)), "norm backward")
    check(x, w, b, grad, eps, layer, out, dx, dw, db, add)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_weight_of_two_calls_gets_both_gradients(cuda_device, dtype):
    x, w, _, grad = case(7, 60, 203, dtype, dtype, False)
    parts = []
    for rows, g in ((x[:30], grad[:30]), (x[30:], grad[30:])):
        leaf = w.clone().requires_grad_(True)
        parts += torch.autograd.grad(rms_norm(rows, leaf), leaf, g)
    leaf = w.clone().requires_grad_(True)
    (both,) = torch.autograd.grad([rms_norm(x[:30], leaf), rms_norm(x[30:], leaf)], leaf, [grad[:30], grad[30:]])
    assert torch.equal(both, parts[0] + parts[1])
