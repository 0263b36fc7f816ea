"""The block's MLP as callers meet it: blocks from older files, replaced and hooked layers, memory files."""

from __future__ import annotations

import io

import pytest
import torch
import torch.nn.functional as F
from torch.nn.utils import parametrize, prune

import dabsn_amd
from dabsn_amd import memory as mem

ACTS = {"none": lambda z: z, "relu2": lambda z: F.relu(z) ** 2, "gelu": F.gelu, "silu": F.silu}


def _block(act, norm="layer", bias=True):
    torch.manual_seed(0)
    block = dabsn_amd.DABSNBlock(8, 8, 8, mlp_ratio=2.0, mlp_activation=act, mlp_norm=norm, mlp_bias=bias)
    for p in (block.mlp_fc1, block.mlp_fc2, block.mlp_norm):
        for q in p.parameters():
            torch.nn.init.normal_(q)
    return block


def _parts(block, h, act):
    return h + block.mlp_fc2(ACTS[act](block.mlp_fc1(block.mlp_norm(h))))


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


@pytest.mark.parametrize("act,norm,bias", [("relu2", "rms", False), ("gelu", "layer", True), ("silu", "rms", True),
                                           ("none", "layer", False)])
@pytest.mark.parametrize("layer", ["mlp_norm", "mlp_fc1", "mlp_fc2"])
def test_hooks_of_its_layers_run(layer, act, norm, bias):
    block, h = _block(act, norm, bias), torch.randn(2, 3, 8)
    handle = getattr(block, layer).register_forward_hook(lambda m, a, out: out + 1)
    want = _parts(block, h, act)
    assert torch.equal(block.forward_mlp(h), want)
    with torch.no_grad():
        assert torch.equal(block.forward_mlp(h), want)
    handle.remove()
    with pytest.raises(RuntimeError, match="device"):  # the fused call again
        block.forward_mlp(h)
    seen = []
    for register in ("register_forward_pre_hook", "register_full_backward_hook",
                     "register_full_backward_pre_hook"):
        handle = getattr(getattr(block, layer), register)(lambda *a: seen.append(register))
        block.forward_mlp(h.clone().requires_grad_(True)).sum().backward()
        assert seen == [register]
        seen.clear()
        handle.remove()


class Doubled(torch.nn.Linear):
    def forward(self, x):
        return 2 * super().forward(x)


def test_replaced_and_pruned_layers_run():
    block, h = _block("gelu"), torch.randn(2, 3, 8)
    base = _parts(block, h, "gelu")
    fc2 = block.mlp_fc2
    block.mlp_fc2 = Doubled(16, 8)
    block.mlp_fc2.load_state_dict(fc2.state_dict())
    assert torch.allclose(block.forward_mlp(h), h + 2 * (base - h), atol=1e-5)
    block.mlp_fc2 = torch.nn.Sequential(fc2)
    assert torch.equal(block.forward_mlp(h), base)
    block.mlp_fc2 = fc2
    fc2.forward = lambda x: torch.zeros(2, 3, 8)
    assert torch.equal(block.forward_mlp(h), h)
    del fc2.forward
    prune.random_unstructured(block.mlp_fc1, "weight", amount=0.5)
    for _ in range(2):  # pruning forms the weight anew in each call
        block.forward_mlp(h).sum().backward()
    assert bool((block.mlp_fc1.weight_orig.grad[block.mlp_fc1.weight_mask == 0] == 0).all())


def test_a_hook_for_all_modules_runs():
    block, h, seen = _block("silu"), torch.randn(2, 3, 8), []
    handle = torch.nn.modules.module.register_module_forward_hook(lambda m, a, out: seen.append(m))
    try:
        block.forward_mlp(h)
    finally:
        handle.remove()
    assert seen == [block.mlp_norm, block.mlp_fc1, block.mlp_fc2]


def test_a_parametrized_layer_is_fused():
    class Half(torch.nn.Module):
        def forward(self, w):
            return w / 2

    block = _block("silu")
    parametrize.register_parametrization(block.mlp_fc1, "weight", Half())
    with pytest.raises(RuntimeError, match="device"):
        block.forward_mlp(torch.randn(2, 3, 8))


@pytest.mark.gpu
@pytest.mark.parametrize("act,norm,bias", [("relu2", "rms", False), ("gelu", "layer", True), ("silu", "rms", True),
                                           ("none", "layer", False)])
def test_one_by_one_is_the_same_function(cuda_device, act, norm, bias):
    """fp32 sums of at most 16 terms of order one on both sides: some 2^-20 of the values' 1 to 100."""
    block, h = _block(act, norm, bias).cuda(), torch.randn(2, 3, 8, device=cuda_device)
    fused = block.forward_mlp(h)
    handle = block.mlp_fc1.register_forward_hook(lambda m, a, out: None)
    parts = block.forward_mlp(h)
    handle.remove()
    assert not torch.equal(fused, h)
    assert float((fused - parts).abs().max()) <= 1e-5 * float(parts.abs().max())


def _lm(**mlp):
    torch.manual_seed(3)
    return dabsn_amd.DABSNSequenceLM(40, 24, 2, residual=True, mlp_ratio=2.0, **mlp)


def _carried(model):
    """A memory of the model's architecture, as if two tokens had been read."""
    layers = []
    for block in model.blocks:
        bank = mem.BankStore(1, int(block.state_dim), device="cpu", dtype=torch.float32)
        bank.append(torch.ones(1, 2, int(block.state_dim)), torch.ones(1, 2, 6))
        state = lambda: tuple(torch.zeros(1, int(block.state_dim)) for _ in range(3))  # noqa: E731
        layers.append(mem.LayerMemory(bank=bank, core=state(), long=state()))
    return mem.DABSNMemory(layers=layers, position=2, batch_size=1, fingerprint=mem.fingerprint_of(model))


def test_memory_files_of_the_reference_mlp_cross_load(tmp_path):
    """``mlp_activation="relu2"`` with the RMS norm and no bias has the reference's parameters and
    function: its files carry the reference's fingerprint and load into either model, as do the plain
    model's. Other kinds are still refused, in both directions."""
    plain, fused, other = _lm(), _lm(mlp_activation="relu2"), _lm(mlp_activation="gelu")
    biased = _lm(mlp_activation="relu2", mlp_bias=True)
    for source in (plain, fused):
        path = mem.save(_carried(source), tmp_path / "a.dmem")
        payload = torch.load(path, weights_only=True)
        assert payload["fingerprint"] == mem.fingerprint_of(plain)
        for target in (plain, fused):
            loaded = mem.load(path, model=target)
            assert loaded.fingerprint == mem.fingerprint_of(target) and loaded.entries == 2
        torch.save({"model": {}}, tmp_path / "c.pt")
        mem.embed_in_checkpoint(mem.load(path), tmp_path / "c.pt")
        for target in (plain, fused):
            assert mem.extract_from_checkpoint(tmp_path / "c.pt", model=target).entries == 2
        for target in (other, biased):
            with pytest.raises(ValueError, match="mlp"):
                mem.load(path, model=target)
    for source in (other, biased):
        path = mem.save(_carried(source), tmp_path / "b.dmem")
        assert mem.load(path, model=source).entries == 2
        for target in (plain, fused, *({other, biased} - {source})):
            with pytest.raises(ValueError, match="mlp"):
                mem.load(path, model=target)


def test_a_callers_model_that_names_its_activation_has_a_fingerprint():
    model = _lm()

    class Own:
        mlp_activation = "gelu"

        def __getattr__(self, name):
            if name in ("mlp_norm", "mlp_bias"):
                raise AttributeError(name)
            return getattr(model, name)

    assert mem.fingerprint_of(Own()) == {**mem.fingerprint_of(model), "mlp": "rms gelu"}
