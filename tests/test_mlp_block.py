"""The block's MLP as callers meet it: blocks from older files, replaced and hooked layers, memory files."""

from __future__ import annotations

import io

import torch

import dabsn_amd


def test_a_block_pickled_before_the_choices_existed_runs():
    """An older pickle holds no ``mlp_activation`` and ``mlp_bias``."""
    torch.manual_seed(0)
    block = dabsn_amd.DABSNBlock(8, 8, 8, mlp_ratio=2.0)
    torch.nn.init.normal_(block.mlp_fc2.weight)
    h = torch.randn(2, 3, 8, requires_grad=True)
    want = block.forward_mlp(h)
    for name in ("mlp_activation", "mlp_bias"):
        block.__dict__.pop(name)
    file = io.BytesIO()
    torch.save(block, file)
    file.seek(0)
    old = torch.load(file, weights_only=False)  # written above
    assert "mlp_activation" not in old.__dict__
    assert torch.equal(old.forward_mlp(h), want)
