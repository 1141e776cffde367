"""What the operators refuse, without a GPU: the Python calls' checks, and the entry points'
own, which come before any work is enqueued."""

from __future__ import annotations

import ctypes
import math
from pathlib import Path

import pytest
import torch

from verification.computation import operators as ops

LIB = Path(__file__).resolve().parents[1] / "pots-2.0_amd" / "libpots_mi355x.so"
E_ARG = -4


@pytest.fixture(scope="module")
def abi():
    if not LIB.exists():
        pytest.fail(f"{LIB} is not built")
    lib = ctypes.CDLL(str(LIB))
    for op in ("attention", "vocab_loss", "embedding"):
        getattr(lib, f"pots_{op}_forward").restype = ctypes.c_int
        getattr(lib, f"pots_{op}_backward").restype = ctypes.c_int
        getattr(lib, f"pots_{op}_backward_work").restype = ctypes.c_uint64
    return lib


def _t(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


Q, KV = (2, 4, 5, 8), (2, 2, 5, 8)


@pytest.mark.parametrize("q, k, v, kw", [
    (Q, (2, 3, 5, 8), (2, 3, 5, 8), {}),               # heads not a multiple
    (Q, (2, 2, 6, 8), KV, {}),                         # another length of keys
    (Q, KV, (2, 2, 5, 9), {}),                         # another width of values
    (Q[1:], KV, KV, {}),                               # three dimensions
    ((2, 4, 5, 129), (2, 2, 5, 129), (2, 2, 5, 129), {}),
    ((2, 4, 5, 0), (2, 2, 5, 0), (2, 2, 5, 0), {}),
    (Q, KV, KV, {"scale": 0.0}), (Q, KV, KV, {"scale": -1.0}),
    (Q, KV, KV, {"scale": math.nan}), (Q, KV, KV, {"scale": math.inf}),
    (Q, KV, KV, {"lengths": _t(2, dtype=torch.int64)}),
    (Q, KV, KV, {"lengths": _t(3, dtype=torch.int32)}),
    (Q, KV, KV, {}),                                   # not on a GPU
])
def test_attention_refuses(q, k, v, kw):
    with pytest.raises(ValueError):
        ops.attention_forward(_t(*q), _t(*k), _t(*v), **kw)


def test_types_are_refused():
    h = torch.float16
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        ops.attention_forward(_t(*Q, dtype=h), _t(*KV, dtype=h), _t(*KV, dtype=h))
    with pytest.raises(ValueError, match="must be torch.float32"):
        ops.attention_forward(_t(*Q), _t(*KV, dtype=torch.bfloat16), _t(*KV))
    with pytest.raises(ValueError):
        ops.vocab_loss_forward(_t(3, 4, dtype=h), _t(5, 4, dtype=h), _t(3, dtype=torch.int64))
    with pytest.raises(ValueError):
        ops.embedding_forward(_t(3, dtype=torch.int64), _t(5, 4, dtype=h))


def test_attention_backward_refuses():
    q, k = _t(*Q), _t(*KV)
    lse = _t(2, 4, 5)
    with pytest.raises(ValueError, match="dout"):
        ops.attention_backward(_t(2, 4, 6, 8), q, k, k, q, lse)
    with pytest.raises(ValueError):
        ops.attention_backward(q, q, k, k, q, _t(2, 4, 6))


@pytest.mark.parametrize("x, w, t", [
    (_t(3, 4), _t(5, 6), _t(3, dtype=torch.int64)),
    (_t(3, 4), _t(5, 4), _t(4, dtype=torch.int64)),
    (_t(3, 4), _t(5, 4), _t(3)),
    (_t(3, 4), _t(0, 4), _t(3, dtype=torch.int64)),
    (_t(3, 4, 1), _t(5, 4), _t(3, dtype=torch.int64)),
    (_t(3, 4), _t(5, 4), _t(3, dtype=torch.int64)),    # not on a GPU
])
def test_vocab_loss_refuses(x, w, t):
    with pytest.raises(ValueError):
        ops.vocab_loss_forward(x, w, t)
    with pytest.raises(ValueError):
        ops.vocab_loss_backward(_t(3), x, w, t, _t(3))


def test_embedding_refuses():
    ids = _t(3, dtype=torch.int64)
    for bad in (lambda: ops.embedding_forward(_t(3), _t(5, 4)),
                lambda: ops.embedding_forward(ids, _t(5)),
                lambda: ops.embedding_forward(ids, _t(0, 4)),
                lambda: ops.embedding_backward(ids, _t(4, 4), 5),
                lambda: ops.embedding_backward(ids, _t(3, 4), 0),
                lambda: ops.embedding_backward(ids, _t(3, 4), 5, add_to=_t(6, 4)),
                lambda: ops.embedding_backward(ids, _t(3, 4), 5, add_to=_t(4, 5).t()),
                lambda: ops.embedding_backward(ids, _t(3, 4), 5, add_to=_t(1, 4).expand(5, 4)),
                lambda: ops.embedding_forward(ids, _t(5, 4))):
        with pytest.raises(ValueError):
            bad()


def _attention(**kw):
    a = dict(b=2, h=4, kv=2, n=5, d=8, dtype=0, causal=1, scale=1.0, ptr=0)
    a.update(kw)
    heads = (a["ptr"], 8, 8, 8) * 8
    return ops._ATTENTION.pack(*heads, a["ptr"], 0, a["b"], a["h"], a["kv"], a["n"], a["d"],
                               a["dtype"], a["causal"], a["scale"])


@pytest.mark.parametrize("kw", [dict(kv=3), dict(kv=0), dict(h=0), dict(d=0), dict(d=129),
                                dict(dtype=2), dict(scale=0.0), dict(scale=math.nan),
                                dict(scale=math.inf), dict(n=0x40000001), dict(b=1 << 20), {}])
def test_attention_entry_points_refuse(abi, kw):
    """Sizes out of range; with none, null pointers."""
    a = _attention(**kw)
    assert abi.pots_attention_forward(a, None) == E_ARG
    assert abi.pots_attention_backward(a, None, None) == E_ARG


def _loss(**kw):
    a = dict(rows=3, dim=4, vocab=5, dtype=0)
    a.update(kw)
    return ops._LOSS.pack(*(0,) * 8, 4, 4, 4, 4, a["rows"], a["dim"], a["vocab"], a["dtype"])


@pytest.mark.parametrize("kw", [dict(dim=0), dict(vocab=0), dict(dtype=2), dict(dim=65537),
                                dict(rows=(1 << 24) + 1), dict(vocab=(1 << 24) + 1),
                                dict(rows=1 << 24, vocab=1 << 24), {}])
def test_vocab_loss_entry_points_refuse(abi, kw):
    a = _loss(**kw)
    assert abi.pots_vocab_loss_forward(a, None, None) == E_ARG
    assert abi.pots_vocab_loss_backward(a, None, None) == E_ARG


def _embedding(**kw):
    a = dict(tokens=3, dim=4, vocab=5, dtype=0, scale=1.0)
    a.update(kw)
    return ops._EMBEDDING.pack(0, 0, 0, 4, 4, a["tokens"], a["dim"], a["vocab"], a["dtype"], 0,
                               a["scale"])


@pytest.mark.parametrize("kw", [dict(dim=0), dict(vocab=0), dict(dtype=2),
                                dict(dim=(1 << 20) + 1), dict(tokens=(1 << 24) + 1),
                                dict(vocab=(1 << 30) + 1), dict(scale=math.nan), {}])
def test_embedding_entry_points_refuse(abi, kw):
    a = _embedding(**kw)
    assert abi.pots_embedding_forward(a, None) == E_ARG
    assert abi.pots_embedding_backward(a, None, None) == E_ARG
    assert abi.pots_attention_forward(None, None) == E_ARG
    assert abi.pots_vocab_loss_forward(None, None, None) == E_ARG
    assert abi.pots_embedding_forward(None, None) == E_ARG


def test_nothing_to_do_is_no_error(abi):
    assert abi.pots_attention_forward(_attention(n=0), None) == 0
    assert abi.pots_attention_backward(_attention(b=0), None, None) == 0
    assert abi.pots_attention_backward_work(_attention(n=0)) == 0
    assert abi.pots_vocab_loss_forward(_loss(rows=0), None, None) == 0
    assert abi.pots_embedding_forward(_embedding(tokens=0), None) == 0


# ---- what autograd is given ---------------------------------------------------------------------

@pytest.fixture
def plain_loss(monkeypatch):
    """The loss's two calls as plain formulas, on the CPU."""
    calls = []

    def forward(x, w, t):
        calls.append("forward")
        s = x @ w.T
        lse = s.logsumexp(1)
        return torch.where(t < 0, 0.0, lse - s.gather(1, t.clamp(min=0)[:, None])[:, 0]), lse

    def backward(weights, x, w, t, lse):
        calls.append("backward")
        g = (x @ w.T - lse[:, None]).exp()
        g[t >= 0, t[t >= 0]] -= 1
        g = g * (weights * (t >= 0))[:, None]
        return g @ w, g.T @ x

    monkeypatch.setattr(ops, "vocab_loss_forward", forward)
    monkeypatch.setattr(ops, "vocab_loss_backward", backward)
    return calls


def test_vocab_loss_weights_have_a_gradient(plain_loss):
    """Each row's loss: the sum is linear in the weights. A row of weight zero has one too, unless it
    holds what no loss comes of."""
    g = torch.Generator().manual_seed(0)
    x, w = torch.randn(6, 4, generator=g), torch.randn(9, 4, generator=g)
    t = torch.tensor([3, 0, -100, 8, 5, 2])
    weights = torch.tensor([0.5, 0.25, 1.0, 0.0, -1.0, 0.0])
    x[5] = math.nan
    want = ops.vocab_loss_forward(x, w, t)[0]
    want[5] = 0.0
    weights.requires_grad_()
    (3 * ops.vocab_loss(x, w, t, weights)).backward()
    assert torch.equal(weights.grad, 3 * want) and "backward" not in plain_loss
    # by differences, of the weights that are not zero and of one that is
    for i in (0, 1, 2, 3, 4):
        step = torch.zeros(6)
        step[i] = 0.25
        up, down = (float(ops.vocab_loss(x, w, t, weights.detach() + s * step)) for s in (1, -1))
        # (linear: six terms of a sum in fp32, each way)
        assert abs((up - down) / 0.5 - float(want[i])) <= 4 * 12 * 2.0**-24 * (abs(up) + abs(down))
    xg = x.nan_to_num().requires_grad_()
    a, b = torch.autograd.grad(ops.vocab_loss(xg, w, t, weights), (xg, weights))
    assert torch.equal(a, ops.vocab_loss_backward(weights.detach(), x.nan_to_num(), w, t,
                                                  (x.nan_to_num() @ w.T).logsumexp(1))[0])
    assert bool((b != 0)[[0, 1, 3, 4, 5]].all())


@pytest.mark.parametrize("n", [0, 1, 5, 1 << 16, (1 << 16) + 1, 70000, 1 << 20])
def test_the_sum_of_many_losses(n):
    t = torch.randn(n, generator=torch.Generator().manual_seed(n))
    got = ops._sum(t)
    # (no order of adding up n values is further off)
    assert got.shape == () and abs(float(got) - float(t.double().sum())) <= \
        n * 2.0**-24 * float(t.double().abs().sum())


class _NoLibrary:
    @staticmethod
    def get():
        return _NoLibrary

    @staticmethod
    def operator(name, args, device):
        raise AssertionError("out-of-range sizes reached the library")


@pytest.fixture
def without_gpu(monkeypatch):
    """The calls' own checks on tensors without memory."""
    monkeypatch.setattr(ops, "_on_gpu", lambda t: None)
    monkeypatch.setattr(ops, "native", _NoLibrary)


def _meta(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="meta")


BIG = 1 << 32


@pytest.mark.parametrize("scale", [1e39, 3.5e38, 1e-60])
def test_attention_refuses_scales_that_fp32_does_not_hold(without_gpu, scale):
    q, k = _meta(*Q), _meta(*KV)
    with pytest.raises(ValueError, match="scale"):
        ops.attention_forward(q, k, k, scale=scale)
    with pytest.raises(ValueError, match="scale"):
        ops.attention_backward(q, q, k, k, q, _meta(2, 4, 5, dtype=torch.float32), scale=scale)


@pytest.mark.parametrize("scale", [1e39, -3.5e38, math.inf, math.nan])
def test_embedding_refuses_scales_that_fp32_does_not_hold(without_gpu, scale):
    ids = _meta(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="scale"):
        ops.embedding_forward(ids, _meta(5, 4), scale=scale)
    with pytest.raises(ValueError, match="scale"):
        ops.embedding_backward(ids, _meta(3, 4), 5, scale=scale)


def test_sizes_past_32_bits_are_refused(without_gpu):
    ids, x = _meta(BIG, dtype=torch.int64), _meta(BIG, 1)
    q, f = _meta(1, 1, BIG, 8), _meta(BIG, dtype=torch.float32)
    for call in (lambda: ops.attention_forward(q, q, q),
                 lambda: ops.attention_forward(q[..., :3], q[..., :3], q[..., :3]),
                 lambda: ops.attention_backward(q, q, q, q, q, f.view(1, 1, BIG)),
                 lambda: ops.vocab_loss_forward(x, _meta(5, 1), ids),
                 lambda: ops.vocab_loss_forward(_meta(3, 1), x, _meta(3, dtype=torch.int64)),
                 lambda: ops.vocab_loss_backward(f, x, _meta(5, 1), ids, f),
                 lambda: ops.embedding_forward(ids, _meta(5, 1)),
                 lambda: ops.embedding_backward(ids, x, 5),
                 lambda: ops.embedding_backward(ids[:3], x[:3], BIG)):
        with pytest.raises(ValueError):
            call()


def test_a_loss_of_no_matrix_is_refused():
    with pytest.raises(ValueError):
        ops.vocab_loss(torch.tensor(1.0), _t(5, 4), _t(3, dtype=torch.int64), _t(3))


def test_added_gradients_of_single_values_and_single_rows(monkeypatch, without_gpu):
    """One value a row has no distance to the next one, and one row none to another row."""
    calls = []
    monkeypatch.setattr(_NoLibrary, "operator",
                        staticmethod(lambda name, args, device: calls.append(name)))
    ids = _meta(3, dtype=torch.int64)
    for dim, into in ((1, _meta(1, 5).t()), (4, _meta(5, 4)), (4, _meta(4).as_strided((1, 4), (0, 1))),
                      (1, _meta(8)[:1, None].as_strided((1, 1), (0, 0)))):
        got = ops.embedding_backward(ids, _meta(3, dim), into.shape[0], add_to=into)
        assert got is into
    assert calls == ["embedding_backward"] * 4
    for into in (_meta(4, 5).t(), _meta(4).expand(5, 4), _meta(8).as_strided((5, 1), (0, 1))):
        with pytest.raises(ValueError):
            ops.embedding_backward(ids, _meta(3, into.shape[1]), 5, add_to=into)
