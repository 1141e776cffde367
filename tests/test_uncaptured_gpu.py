"""A decoder's pass that leaves no transcript (DecoderComputation.uncaptured_loss) against the
captured step's loss on the same model and batch: the same loss and gradients, up to the
roundings of the compute format."""

from __future__ import annotations

import pytest
import torch

from setup.records import Record
from verification.computation.instances.attention import ATTENTION
from verification.computation.instances.decoder import DecoderComputation

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _step(tied, bias, dtype, *, L=2, d=64, n_h=4, n_kv=2, n_v=500, n_s=3, n=37):
    c = DecoderComputation(L=L, d=d, d_f=2 * d, n_h=n_h, n_kv=n_kv, n_v=n_v, n_s=n_s, n=n,
                           tied=tied, qkv_bias=bias, compute_dtype=dtype)
    torch.manual_seed(0)
    with torch.device(DEV):
        model = c.build_model()
    g = torch.Generator().manual_seed(1)
    records = []
    for _ in range(n_s):
        ids = torch.randint(0, n_v, (n,), generator=g, dtype=torch.int32)
        mask = (torch.rand(n, generator=g) < 0.7).int()
        records.append(Record(ids, torch.roll(ids, -1), mask))
    return c, model, records


def _grads(model, loss):
    model.zero_grad(set_to_none=True)
    loss.backward()
    return {name: p.grad.double() for name, p in model.named_parameters()}


# Both passes are one computation whose operations round differently. In fp32 a sum of at most
# d_f + n + n_v terms is off by as many half steps, through 2 layers there and back; in bf16 each of
# the 12 tensors that a layer rounds there and back is off by half a step.
@pytest.mark.parametrize("tied, bias", [(True, True), (True, False), (False, True)])
@pytest.mark.parametrize("dtype, bound", [(torch.float32, 4 * (128 + 37 + 500) * 2.0**-24),
                                          (torch.bfloat16, 2 * 24 * 2.0**-8)])
def test_the_captured_step_and_the_uncaptured_pass_agree(tied, bias, dtype, bound):
    c, model, records = _step(tied, bias, dtype)
    want = c.loss(model, records)
    want_g = _grads(model, want)
    got = c.uncaptured_loss(model, records)
    assert model.config._attn_implementation == ATTENTION  # the captured core is back
    got_g = _grads(model, got)
    assert got.dtype == torch.float32
    assert abs(float((got - want).detach())) <= bound * abs(float(want.detach()))
    total = torch.stack([g.norm() for g in want_g.values()]).norm()
    assert got_g.keys() == want_g.keys()
    for name, g in want_g.items():
        # (a bias's gradient may be the difference of larger terms: against the whole gradient)
        assert float((got_g[name] - g).norm()) <= bound * float(g.norm() + total), name
    with torch.no_grad():
        assert torch.equal(c.uncaptured_loss(model, records), got.detach())


def test_a_step_of_training_lowers_the_loss():
    c, model, records = _step(True, True, torch.bfloat16)
    first = c.uncaptured_loss(model, records)
    first.backward()
    with torch.no_grad():
        for p in model.parameters():
            p -= 0.5 * p.grad
        assert float(c.uncaptured_loss(model, records)) < float(first.detach())


@pytest.mark.parametrize("reentrant", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_checkpointed_layers_give_the_same_gradients(dtype, reentrant):
    """The layers run again in the backward pass, with the same operators: the same bits."""
    c, model, records = _step(True, True, dtype)
    loss = c.uncaptured_loss(model, records)
    want = _grads(model, loss)
    model.train()
    model.gradient_checkpointing_enable(
        gradient_checkpointing_kwargs={"use_reentrant": reentrant})
    again = c.uncaptured_loss(model, records)
    assert torch.equal(again.detach(), loss.detach())
    got = _grads(model, again)
    for name, g in want.items():
        assert torch.equal(got[name], g), name
