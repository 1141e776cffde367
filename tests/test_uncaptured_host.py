"""A decoder's pass that leaves no transcript, on the CPU with torch's own operations in place of
the operators: which attention each pass runs, whatever else runs on the same model."""

from __future__ import annotations

import threading

import pytest
import torch
import torch.nn.functional as F

from setup.records import Record
from verification.computation import operators
from verification.computation.instances import attention as A
from verification.computation.instances.decoder import DecoderComputation

# One computation in two orders of its sums, in fp32: of at most 64 + 24 + 50 terms, through two
# layers there and back, and three of the operators.
CLOSE = 8 * (64 + 24 + 50) * 2.0**-24


def _torch_attention(q, k, v, *, causal=True, lengths=None, scale=None):
    n, rep = q.shape[2], q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(rep, 1), v.repeat_interleave(rep, 1)
    s = q @ k.transpose(2, 3) * scale
    s = s.masked_fill(torch.ones(n, n, dtype=torch.bool).triu(1), -torch.inf)
    return s.softmax(-1) @ v


def _torch_loss(x, w, targets, weights):
    return (F.cross_entropy(x @ w.T, targets, reduction="none") * weights).sum()


@pytest.fixture(autouse=True)
def on_the_cpu(monkeypatch):
    monkeypatch.setattr(operators, "attention", _torch_attention)
    monkeypatch.setattr(operators, "vocab_loss", _torch_loss)
    monkeypatch.setattr(operators, "embedding", lambda ids, w: F.embedding(ids, w))


def _step(bias):
    c = DecoderComputation(L=2, d=32, d_f=64, n_h=4, n_kv=2, n_v=50, n_s=2, n=24, tied=True,
                           qkv_bias=bias)
    torch.manual_seed(0)
    model = c.build_model()
    g = torch.Generator().manual_seed(1)
    records = []
    for _ in range(2):
        ids = torch.randint(0, 50, (24,), generator=g, dtype=torch.int32)
        records.append(Record(ids, torch.roll(ids, -1), (ids % 3 > 0).int()))
    return c, model, records


def _grads(model, loss):
    model.zero_grad(set_to_none=True)
    loss.backward()
    return {name: p.grad.clone() for name, p in model.named_parameters()}


def _same(got, want):
    total = torch.stack([g.norm() for g in want.values()]).norm()
    for name, g in want.items():
        assert float((got[name] - g).norm()) <= CLOSE * float(g.norm() + total), name


@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("reentrant", [None, True, False])
def test_layers_that_are_computed_again(bias, reentrant):
    """Checkpointed layers run a second time in the backward pass: the same attention then."""
    c, model, records = _step(bias)
    want_loss = c.loss(model, records)
    want = _grads(model, want_loss)
    if reentrant is not None:
        model.train()
        model.gradient_checkpointing_enable(
            gradient_checkpointing_kwargs={"use_reentrant": reentrant})
    loss = c.uncaptured_loss(model, records)
    assert abs(float(loss.detach() - want_loss.detach())) <= CLOSE * float(want_loss.detach())
    _same(_grads(model, loss), want)


class _Pass(threading.Thread):
    """The uncaptured loss in a thread of its own, held in its first layer until `go_on`."""

    def __init__(self, c, model, records):
        super().__init__()
        self.args, self.result = (c, model, records), None
        self.entered, self.go_on = threading.Event(), threading.Event()

    def run(self):
        c, model, records = self.args
        self.result = float(c.uncaptured_loss(model, records).detach())

    def hold(self):
        self.start()
        assert self.entered.wait(60)
        return self

    def end(self):
        self.go_on.set()
        self.join(60)
        assert not self.is_alive()
        return self.result


@pytest.fixture
def held(monkeypatch):
    def attention(*args, **kw):
        t = threading.current_thread()
        if isinstance(t, _Pass) and not t.entered.is_set():
            t.entered.set()
            assert t.go_on.wait(60)
        return _torch_attention(*args, **kw)

    monkeypatch.setattr(operators, "attention", attention)


def test_two_passes_at_once(held):
    """The first to begin ends while the second is in its first layer."""
    c, model, records = _step(True)
    want = float(c.uncaptured_loss(model, records).detach())
    captured = float(c.loss(model, records).detach())
    one = _Pass(c, model, records).hold()
    two = _Pass(c, model, records).hold()
    assert one.end() == want and two.end() == want
    assert model.config._attn_implementation == A.ATTENTION
    assert float(c.loss(model, records).detach()) == captured


def test_a_captured_step_beside_an_uncaptured_pass(held):
    """The captured core, with its probabilities, and under a mask of its caller's."""
    c, model, records = _step(True)
    ids = torch.stack([r.ids for r in records]).long()
    pad = torch.ones(2, 24, dtype=torch.long)
    pad[0, :7] = 0

    def masked():
        return model(input_ids=ids, attention_mask=pad).logits.detach()

    want = masked()
    captured = float(c.loss(model, records).detach())
    beside = _Pass(c, model, records).hold()
    try:
        got = masked(), float(c.loss(model, records).detach())
    finally:
        beside.end()
    assert torch.equal(got[0], want) and got[1] == captured
    assert float((want - model(input_ids=ids).logits.detach()).abs().max()) > 0.01


def test_what_the_uncaptured_attention_refuses():
    """Nothing that the operator would leave out goes through it unseen."""
    c, model, _ = _step(True)
    module = model.model.layers[0].self_attn
    q, k = torch.randn(1, 4, 5, 8), torch.randn(1, 2, 5, 8)
    mask = A.uncaptured_mask(q.device)
    out, probs = A.attention_forward(module, q, k, k, mask, 0.3)
    assert out.shape == (1, 5, 4, 8) and probs is None
    want, _ = A.attention_forward(module, q, k, k,
                                  torch.full((5, 5), -torch.inf).triu(1)[None, None], 0.3)
    assert torch.allclose(out, want, atol=CLOSE)
    for kw in ({"dropout": 0.1}, {"sliding_window": 3}):
        with pytest.raises(ValueError):
            A.attention_forward(module, q, k, k, mask, 0.3, **kw)


def test_a_model_of_another_attention_is_refused():
    c, model, records = _step(True)
    model.config._attn_implementation = "eager"
    with pytest.raises(ValueError, match="attention"):
        c.uncaptured_loss(model, records)
