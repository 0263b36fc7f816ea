"""Calls of the linear layer and the MLP that no formula covers: what is refused inside autocast."""

from __future__ import annotations

import pytest
import torch

from dabsn_amd import fused_linear, fused_mlp

BF16, FP32 = torch.bfloat16, torch.float32


@pytest.fixture
def autocast():
    """Autocast to bfloat16 as ``torch.autocast("cuda")`` sets it, also where there is no device."""
    dtype, enabled = torch.get_autocast_dtype("cuda"), torch.is_autocast_enabled("cuda")
    torch.set_autocast_dtype("cuda", BF16)
    torch.set_autocast_enabled("cuda", True)
    yield
    torch.set_autocast_enabled("cuda", enabled)
    torch.set_autocast_dtype("cuda", dtype)


@pytest.mark.parametrize("residual,error", [
    (torch.zeros(5), ValueError), (torch.zeros(1, 5), ValueError), (torch.zeros(3, 1), ValueError),
    (torch.zeros(2, 3, 5), ValueError), (torch.zeros(3, 5, dtype=torch.float64), TypeError),
    (torch.zeros(3, 5, dtype=torch.float16), TypeError), (torch.zeros(5, dtype=BF16), ValueError)])
def test_autocast_refuses_the_residuals_that_are_refused_outside(autocast, residual, error):
    """Of another type the residual is added by itself, which would broadcast it."""
    with pytest.raises(error, match="residual"):
        fused_linear(torch.zeros(3, 4), torch.zeros(5, 4), residual=residual)


def test_autocast_refuses_an_mlp_that_does_not_lead_back(autocast):
    with pytest.raises(ValueError, match="w2"):
        fused_mlp(torch.zeros(3, 4), torch.zeros(5, 4), torch.zeros(1, 5))


def test_autocast_asks_for_the_residuals_device(autocast):
    with pytest.raises(RuntimeError, match="device"):
        fused_linear(torch.zeros(3, 4), torch.zeros(5, 4), residual=torch.zeros(3, 5))


def test_library_refuses_wide_results_that_no_kernel_forms():
    """fp32 results beside bf16 operands: the rows' gradient alone, without a slope, in whole eights."""
    import ctypes

    from dabsn_amd import _lib

    lib, one = _lib.load(), 1 << 20
    good = dict(dtype=1, transB=1, wideC=1, M=4, N=8, K=16, A=one, B=one, C=one, lda=16, ldb=8, ldc=8)
    for bad in (dict(dtype=0), dict(transB=0, ldb=16), dict(transA=1, lda=8), dict(ldc=9), dict(ldc=12),
                dict(slope=one, slope_kind=1, lds=8)):
        assert lib.dabsn_hip_linear(ctypes.byref(_lib.LinearCall(**{**good, **bad})), None) == -2, bad
        assert lib.dabsn_hip_linear_workspace_bytes(ctypes.byref(_lib.LinearCall(**{**good, **bad}))) == 0
