"""PICO_LINEAR_8BIT=1 reads a layer's modules instead of calling them: what that would pass by is an error before anything is computed, and a layer called by itself computes in 8 bits too."""
from types import SimpleNamespace

import pytest
import torch
import torch.nn as nn


@pytest.fixture
def layer(monkeypatch):
    import picotron_amd.process_group_manager as pgm
    from picotron_amd import model as M
    monkeypatch.setenv("DEVICE", "cpu")
    monkeypatch.setenv("CONTEXT_PARALLEL", "0")
    for name in ("FLASH_ATTEN", "PICO_FUSED_PROJ", "PICO_FUSED_RESIDUAL"):
        monkeypatch.delenv(name, raising=False)
    monkeypatch.setenv("PICO_LINEAR_8BIT", "1")
    pgm.setup_process_group_manager(1, 1, 1, 1)
    config = SimpleNamespace(hidden_size=64, num_attention_heads=2, num_key_value_heads=2, num_hidden_layers=1, intermediate_size=96, vocab_size=50, max_position_embeddings=16, rms_norm_eps=1e-5,
                             rope_theta=10000.0)
    return M.DecoderLayer(config, 0).to(torch.bfloat16)


@pytest.fixture
def calls(monkeypatch, layer):
    """The layers in 8 bits in place of which plain torch writes down what they are given."""
    from picotron_amd import model as M
    seen = []
    def norm_linear(x, residual, norm_weight, eps, weight, packed=None, parts=()):
        h = x if residual is None else x + residual
        seen.append(("norm", weight.shape))
        return torch.nn.functional.linear(h, weight), h
    def swiglu_linear(gate_up, weight, packed=None):
        seen.append(("swiglu", weight.shape))
        return torch.nn.functional.linear(gate_up.chunk(2, -1)[0], weight)
    monkeypatch.setattr(M, "rms_norm_linear_8bit", norm_linear)
    monkeypatch.setattr(M, "swiglu_linear_8bit", swiglu_linear)
    monkeypatch.setattr(M.Attention, "from_qkv", lambda self, qkv, cos, sin: qkv[..., :64])
    return seen


X = torch.ones(1, 8, 64, dtype=torch.bfloat16)
NAMES = ["input_layernorm", "post_attention_layernorm", "attention", "mlp", "mlp.down_proj"]


def test_a_layer_by_itself_is_in_8_bits(layer, calls):
    branch, residual = layer.forward_chained(X, None)
    chained = list(calls)
    calls.clear()
    assert torch.equal(layer(X), residual + branch)
    assert calls == chained == [("norm", (192, 64)), ("norm", (192, 64)), ("swiglu", (64, 96))]


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("hook", ["register_forward_hook", "register_forward_pre_hook", "register_full_backward_hook", "register_full_backward_pre_hook"])
def test_hooks_that_would_be_silent(layer, calls, name, hook):
    handle = getattr(layer.get_submodule(name), hook)(lambda *a: None)
    for call in (lambda: layer(X), lambda: layer.forward_chained(X, None)):
        with pytest.raises(RuntimeError, match=f"reads {name} without calling it"):
            call()
    assert not calls
    handle.remove()
    layer(X)
    assert len(calls) == 3


class Adapter(nn.Module):
    def __init__(self, inside):
        super().__init__()
        self.inside, self.weight = inside, inside.weight if hasattr(inside, "weight") else None

    def forward(self, *a, **k):
        return 2 * self.inside(*a, **k)


@pytest.mark.parametrize("name", NAMES)
def test_modules_in_another_ones_place(layer, calls, name):
    parent, _, last = name.rpartition(".")
    inside = layer.get_submodule(name)
    setattr(layer.get_submodule(parent), last, Adapter(inside))
    with pytest.raises(RuntimeError, match=f"reads {name} as"):
        layer(X)
    setattr(layer.get_submodule(parent), last, inside)
    inside.forward = lambda *a, **k: None
    with pytest.raises(RuntimeError, match=f"reads {name} as"):
        layer(X)
    assert not calls


def test_projections_and_norms_of_other_kinds(layer, calls):
    from picotron_amd import model as M
    down = layer.mlp.down_proj
    layer.mlp.down_proj = nn.Linear(96, 64, bias=False).to(torch.bfloat16)       # (the same product)
    layer(X)
    layer.mlp.down_proj = nn.Linear(96, 64).to(torch.bfloat16)
    with pytest.raises(RuntimeError, match="without a bias"):
        layer(X)
    layer.mlp.down_proj = down
    layer.post_attention_layernorm = M.LlamaRMSNorm(64).to(torch.bfloat16)
    with pytest.raises(RuntimeError, match="plain TritonRMSNorm"):
        layer(X)


def test_a_layer_by_itself_without_the_adds_inside_the_norms(layer, calls, monkeypatch):
    monkeypatch.setenv("PICO_FUSED_RESIDUAL", "0")
    with pytest.raises(RuntimeError, match="inside the norms"):
        layer(X)
    monkeypatch.setenv("PICO_FUSED_PROJ", "0")
    monkeypatch.delenv("PICO_FUSED_RESIDUAL")
    with pytest.raises(RuntimeError, match="fused projections"):
        layer(X)


def test_without_the_switch_hooks_and_modules_are_called(layer, calls, monkeypatch):
    monkeypatch.delenv("PICO_LINEAR_8BIT")
    seen = []
    for name in ("input_layernorm", "attention", "post_attention_layernorm", "mlp"):
        module = layer.get_submodule(name)
        module.forward = lambda x, *a, **k: x
        module.register_forward_hook(lambda m, a, out, name=name: seen.append(name))
    layer(X)
    assert seen == ["input_layernorm", "attention", "post_attention_layernorm", "mlp"] and not calls


def test_subclasses_count_by_what_they_compute(layer, calls):
    from picotron_amd import model as M

    class Named(M.MLP):
        label = "mine"

    class Doubled(M.MLP):
        def forward(self, x):
            return 2 * super().forward(x)

    layer.mlp.__class__ = Named
    layer(X)
    assert len(calls) == 3
    layer.mlp.__class__ = Doubled
    with pytest.raises(RuntimeError, match="plain MLP"):
        layer(X)


def test_a_parametrized_projection_is_read_through_its_parametrization(layer, calls, monkeypatch):
    from picotron_amd import model as M
    got = []
    monkeypatch.setattr(M, "swiglu_linear_8bit", lambda gate_up, weight, packed=None: (got.append(weight), gate_up[..., :64])[1])

    class Doubled(nn.Module):
        def forward(self, w):
            return 2 * w

    plain = layer.mlp.down_proj.weight.detach().clone()
    nn.utils.parametrize.register_parametrization(layer.mlp.down_proj, "weight", Doubled())
    layer(X)
    assert torch.equal(got[0], 2 * plain) and got[0].requires_grad
