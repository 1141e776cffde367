"""A step that leaves no transcript (prover.step.uncaptured_step) and the fused pass under it,
against the captured step's arithmetic on the same model and batch."""

from __future__ import annotations

import math

import pytest
import torch

import step_operators_oracle as O
from test_uncaptured_gpu import _grads, _step
from verification.computation import operators
from verification.computation.interface import load_weights, snapshot_weights
from verification.prover.step import prove_step, uncaptured_step

pytestmark = pytest.mark.gpu

# As in test_uncaptured_gpu: in fp32 a sum of at most d_f + n + n_v terms, through 2 layers there and
# back; in bf16 each of the 12 tensors that a layer rounds there and back is off by half a step. The
# model's own angles are fp32 products of positions up to 36: 2^-19 of a turn's radian, through the
# same layers.
BOUNDS = [(torch.float32, 4 * (128 + 37 + 500) * 2.0**-24 + 4 * 2.0**-19),
          (torch.bfloat16, 2 * 24 * 2.0**-8)]


@pytest.mark.parametrize("tied, bias", [(True, True), (True, False), (False, True)])
@pytest.mark.parametrize("dtype, bound", BOUNDS)
def test_the_captured_step_and_the_fused_pass_agree(tied, bias, dtype, bound):
    c, model, records = _step(tied, bias, dtype)
    want = c.loss(model, records)
    want_g = _grads(model, want)
    got = c.uncaptured_loss(model, records, fused=True)
    got_g = _grads(model, got)
    assert got.dtype == torch.float32 and got_g.keys() == want_g.keys()
    assert abs(float((got - want).detach())) <= bound * abs(float(want.detach()))
    total = torch.stack([g.norm() for g in want_g.values()]).norm()
    for name, g in want_g.items():
        assert float((got_g[name] - g).norm()) <= bound * float(g.norm() + total), name
    with torch.no_grad():
        assert torch.equal(c.uncaptured_loss(model, records, fused=True), got.detach())


@pytest.mark.parametrize("dtype, bound", BOUNDS)
@pytest.mark.parametrize("clipped", [False, True])
def test_a_step(dtype, bound, clipped):
    """The weights after it: the captured step's, or those of its gradient scaled to the bound."""
    c, model, records = _step(True, True, dtype)
    w_t = snapshot_weights(c, model)
    want_loss = c.loss(model, records)
    grads = _grads(model, want_loss)
    norm = float(torch.stack([g.norm() for g in grads.values()]).norm())
    max_norm = norm / 3 if clipped else math.inf
    loss, got_norm = uncaptured_step(c, model, records, max_norm=max_norm)
    assert abs(float(loss) - float(want_loss.detach())) <= bound * abs(float(want_loss.detach()))
    assert abs(float(got_norm) - norm) <= 2 * bound * norm
    assert all(p.grad is None for p in model.parameters())
    factor = c.eta * (1 / 3 if clipped else 1)
    for name, p in model.named_parameters():
        want = w_t[name].double() - factor * grads[name]
        # the gradient's difference, the factor's, and half a step of the weights
        off = float((p.detach().double() - want).norm())
        assert off <= factor * 4 * bound * norm + 2.0**-23 * float(want.norm()), name
    if not clipped:
        load_weights(c, model, w_t)
        proved = prove_step(c, model, w_t, records)
        assert abs(proved.loss - float(loss)) <= bound * abs(proved.loss)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("clipped", [False, True])
def test_the_update_of_a_step(dtype, clipped):
    """Each weight is the one before less its own gradient of the fused pass, which gives the same bits
    again, by the factor and eta, within the roundings of that one formula."""
    c, model, records = _step(True, True, dtype)
    before = [p.detach().clone() for p in model.parameters()]
    loss = c.uncaptured_loss(model, records, fused=True)
    loss.backward()
    grads = [p.grad.clone() for p in model.parameters()]
    norm = float(O.total_norm(grads)[0])
    max_norm = norm / 3 if clipped else math.inf
    got, got_norm = uncaptured_step(c, model, records, max_norm=max_norm)
    assert torch.equal(got, loss.detach())
    O.within(got_norm, O.total_norm(grads), "norm")
    names = [n for n, _ in model.named_parameters()]
    for name, p, want in zip(names, model.parameters(), O.changed(grads, max_norm, before, c.eta)):
        O.within(p.detach(), want, name)


@pytest.mark.parametrize("tied, bias", [(True, True), (False, False)])
def test_fused_gradients_in_bf16_are_as_near_as_the_captured_step_s(tied, bias):
    """Against fp32, tensor by tensor: both passes round like tensors to bf16, the fused one fewer of them, so
    that each's error is a sum of like many independent roundings; three times the other's allows
    for their chance, and one rounding for a gradient that the other has by luck. A term that is missing, or has
    the wrong sign, is as large as the gradient, a hundred times that."""
    single, model, records = _step(tied, bias, torch.float32)
    exact = _grads(model, single.loss(model, records))
    weights = dict(model.named_parameters())
    c, model, records = _step(tied, bias, torch.bfloat16)
    assert all(torch.equal(p, weights[n]) for n, p in model.named_parameters())
    captured = _grads(model, c.loss(model, records))
    fused = _grads(model, c.uncaptured_loss(model, records, fused=True))
    for name, g in exact.items():
        off, other = float((fused[name] - g).norm()), float((captured[name] - g).norm())
        assert off <= 3 * other + 2.0**-8 * float(g.norm()), (name, off, other, float(g.norm()))


def test_steps_are_deterministic():
    c, model, records = _step(True, False, torch.float32)
    w_t = snapshot_weights(c, model)
    runs = []
    for _ in range(2):
        load_weights(c, model, w_t)
        for _ in range(3):
            loss, norm = uncaptured_step(c, model, records, max_norm=1.0)
        runs.append((loss, norm, snapshot_weights(c, model)))
    assert torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][1], runs[1][1])
    for name, w in runs[0][2].items():
        assert torch.equal(w, runs[1][2][name]), name


def test_frozen_weights_stay():
    c, model, records = _step(True, True, torch.bfloat16)
    frozen = {n for n, _ in model.named_parameters() if "layers.0" in n or n == "model.norm.weight"}
    for n, p in model.named_parameters():
        p.requires_grad_(n not in frozen)
    before = {n: p.detach().clone() for n, p in model.named_parameters()}
    uncaptured_step(c, model, records, max_norm=1.0)
    for n, p in model.named_parameters():
        assert torch.equal(p.detach(), before[n]) == (n in frozen), n


def test_a_proved_step_notices_a_step_on_its_leaves():
    """The update is a write like any other: a transcript whose weights it changes says so."""
    from verification.prover.capture import MutatedCaptureError
    c, model, records = _step(True, True, torch.float32)
    proved = prove_step(c, model, snapshot_weights(c, model), records)
    proved.assert_unmodified()
    w = list(proved.w_next.values())
    operators.sgd_step(w, [torch.ones_like(t) for t in w], 0.1)
    with pytest.raises(MutatedCaptureError):
        proved.assert_unmodified()
