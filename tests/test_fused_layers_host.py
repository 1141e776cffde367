"""The pass over fused layers on the CPU, with torch's own operations in place of the operators: the
same loss and gradients as the model's own layers, and what is refused."""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

from test_uncaptured_host import _grads, _same, _step, on_the_cpu  # noqa: F401  (a fixture)
from verification.computation import operators
from verification.prover.step import uncaptured_step


def _torch_norm(x, weight, *, eps, residual=None, out_dtype=None):
    t = x if residual is None else x + residual
    y = (t * (t.square().mean(-1, keepdim=True) + eps).rsqrt() * weight).to(out_dtype)
    return y if residual is None else (y, t)


def _torch_rotary(q, k, positions, frequencies):
    angle = positions[:, None] * frequencies
    c, s = angle.cos(), angle.sin()

    def turned(x):
        u, v = x.chunk(2, -1)
        return torch.cat([u * c - v * s, u * s + v * c], -1)

    return turned(q), turned(k)


def _torch_sgd(weights, gradients, eta, *, max_norm):
    norm = torch.stack([g.norm() for g in gradients]).norm()
    with torch.no_grad():
        for w, g in zip(weights, gradients):
            w -= eta * min(1.0, max_norm / float(norm)) * g
    return norm


@pytest.fixture(autouse=True)
def step_on_the_cpu(monkeypatch, on_the_cpu):  # noqa: F811
    monkeypatch.setattr(operators, "rms_norm", _torch_norm)
    monkeypatch.setattr(operators, "rotary", _torch_rotary)
    monkeypatch.setattr(operators, "gated_silu", lambda g, u: F.silu(g) * u)
    monkeypatch.setattr(operators, "sgd_step", _torch_sgd)


@pytest.mark.parametrize("bias", [True, False])
def test_fused_layers_are_the_models_own(bias):
    c, model, records = _step(bias)
    want_loss = c.loss(model, records)
    want = _grads(model, want_loss)
    got = c.uncaptured_loss(model, records, fused=True)
    assert abs(float((got - want_loss).detach())) <= 1e-5 * float(want_loss.detach())
    _same(_grads(model, got), want)


def test_a_step_on_the_cpu():
    c, model, records = _step(True)
    before = {n: p.detach().clone() for n, p in model.named_parameters()}
    want = _grads(model, c.loss(model, records))
    norm = torch.stack([g.norm() for g in want.values()]).norm()
    loss, got = uncaptured_step(c, model, records, max_norm=float(norm) / 2)
    assert not loss.requires_grad and abs(float(got - norm)) <= 1e-4 * float(norm)
    for n, p in model.named_parameters():
        assert p.grad is None
        assert torch.allclose(p, before[n] - c.eta / 2 * want[n], atol=1e-7, rtol=1e-6), n


def test_what_fused_layers_refuse():
    c, model, records = _step(False)
    model.train()
    model.gradient_checkpointing_enable()
    with pytest.raises(ValueError, match="checkpointed"):
        c.uncaptured_loss(model, records, fused=True)
    c, model, records = _step(False)
    model.config.hidden_act = "gelu"
    with pytest.raises(ValueError, match="activation"):
        c.uncaptured_loss(model, records, fused=True)
    c, model, records = _step(True)
    model.model.layers[1].self_attn.sliding_window = 8
    with pytest.raises(ValueError, match="sliding"):
        c.uncaptured_loss(model, records, fused=True)
    c, model, records = _step(True)
    model.train()
    model.model.layers[1].self_attn.attention_dropout = 0.1
    with pytest.raises(ValueError, match="dropout"):
        c.uncaptured_loss(model, records, fused=True)
    c, model, records = _step(True)
    model.model.rotary_emb.rope_type = "dynamic"
    with pytest.raises(ValueError, match="rotary"):
        c.uncaptured_loss(model, records, fused=True)
    with torch.no_grad(), pytest.raises(RuntimeError, match="grad mode"):
        uncaptured_step(c, model, records)
    from verification.computation.instances.mlp import MLPComputation
    with pytest.raises(ValueError, match="no uncaptured pass"):
        uncaptured_step(MLPComputation([4, 4], n_s=2, eta=0.1), model, records)


@pytest.mark.parametrize("kind", ["qwen3", "granite", "mistral"])
def test_layers_of_other_models_are_refused(kind):
    """Their modules have the same names and do more between them: heads' norms, branches that are scaled."""
    import transformers
    from verification.computation.instances.attention import register
    c, _, records = _step(False)
    cfg = transformers.CONFIG_MAPPING[kind](
        vocab_size=c.n_v, hidden_size=c.d, intermediate_size=c.d_f, num_hidden_layers=c.L,
        num_attention_heads=c.n_h, num_key_value_heads=c.n_kv, head_dim=c.d_h, hidden_act="silu",
        max_position_embeddings=64)
    cfg._attn_implementation = register()
    model = transformers.AutoModelForCausalLM.from_config(cfg).eval()
    with pytest.raises(ValueError, match=kind):
        c.uncaptured_loss(model, records, fused=True)
