"""Tangents of forward-mode differentiation are refused, not dropped, by the operators of the MLP and of
the vocabulary, with leaves that want gradients and without."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import dabsn_amd

IDS = torch.tensor([1, 4, 0])


def _rand(*shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(len(shape)))


CALLS = {
    "layer_norm": (lambda x, w: dabsn_amd.layer_norm(x, w), (3, 5), (5,)),
    "rms_norm": (lambda x, w: dabsn_amd.rms_norm(x, w), (3, 5), (5,)),
    "fused_linear": (lambda x, w: dabsn_amd.fused_linear(x, w), (3, 5), (7, 5)),
    "fused_linear residual": (lambda x, w: dabsn_amd.fused_linear(x, _rand(5, 5), residual=w), (3, 5), (3, 5)),
    "fused_mlp": (lambda x, w: dabsn_amd.fused_mlp(x, w, _rand(5, 7)), (3, 5), (7, 5)),
    "fused_mlp norm": (lambda x, w: dabsn_amd.fused_mlp(x, _rand(7, 5), _rand(5, 7), norm_weight=w), (3, 5), (5,)),
    "token_logprobs": (lambda x, w: dabsn_amd.token_logprobs(x, IDS), (3, 5), None),
    "chunked_linear_token_logprobs":
        (lambda x, w: dabsn_amd.chunked_linear_token_logprobs(x, w, None, IDS), (3, 5), (7, 5)),
    "distillation_from_logits":
        (lambda x, w: dabsn_amd.distillation_from_logits(x, _rand(3, 2), torch.tensor([[0, 1]] * 3)), (3, 5), None),
    "scaled_embedding": (lambda x, w: dabsn_amd.scaled_embedding(IDS, x, scale=2.0), (5, 8), None),
}


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("name", CALLS)
def test_tangents_are_refused(name, which, grad):
    call, *shapes = CALLS[name]
    if shapes[which] is None:
        pytest.skip("one differentiable tensor")
    tensors = [None if s is None else _rand(*s).requires_grad_(grad) for s in shapes]
    with forward_ad.dual_level():
        tensors[which] = forward_ad.make_dual(tensors[which], torch.ones(shapes[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(*tensors)


@pytest.mark.parametrize("name", CALLS)
def test_other_tensors_pass_inside_a_level(name):
    """Without a tangent the calls go on to their next check."""
    call, *shapes = CALLS[name]
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="device"):
            call(*(None if s is None else _rand(*s) for s in shapes))
