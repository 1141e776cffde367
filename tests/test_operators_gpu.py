"""The training pass's operators against their formulas in 64 bits, at the sizes, masks, strides
and values where a tiled kernel can go wrong. Bounds come from the formulas' own sums
(operators_oracle)."""

from __future__ import annotations

import math

import pytest
import torch

import operators_oracle as R
from verification.computation import operators as ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


def _rand(g, *shape, dtype, std=1.0):
    return (torch.randn(*shape, generator=g) * std).to(dtype).to(DEV)


def _gen(seed):
    return torch.Generator().manual_seed(seed)


# ---- attention ------------------------------------------------------------------------------

def _attention_inputs(seed, dtype, b, h, kv, d, n):
    g = _gen(seed)
    return (_rand(g, b, h, n, d, dtype=dtype), _rand(g, b, kv, n, d, dtype=dtype),
            _rand(g, b, kv, n, d, dtype=dtype), _rand(g, b, h, n, d, dtype=dtype))


def _attention_check(q, k, v, g, **kw):
    out, lse = ops.attention_forward(q, k, v, **kw)
    dq, dk, dv = ops.attention_backward(g, q, k, v, out, lse, **kw)
    want = R.attention(q, k, v, g, **kw)
    for name, got in (("out", out), ("lse", lse), ("dq", dq), ("dk", dk), ("dv", dv)):
        R.within(got, want[name], name)
    return out, lse, dq, dk, dv


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("b, h, kv, d, n", [
    (1, 1, 1, 1, 1), (2, 4, 2, 8, 16), (1, 2, 1, 24, 2), (3, 3, 3, 32, 31), (1, 6, 2, 33, 32),
    (2, 7, 1, 64, 33), (1, 4, 4, 64, 63), (2, 3, 1, 80, 64), (1, 2, 2, 96, 65),
    (2, 2, 1, 100, 127), (1, 6, 1, 128, 129), (1, 2, 1, 128, 257), (2, 14, 2, 64, 200)])
def test_attention_sizes(dtype, causal, b, h, kv, d, n):
    _attention_check(*_attention_inputs(n, dtype, b, h, kv, d, n), causal=causal)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("b, h, kv, n", [(8, 16, 8, 257), (8, 16, 2, 65)])
def test_attention_of_many_heads(dtype, d, b, h, kv, n):
    """Enough rows for blocks of four and of two waves."""
    _attention_check(*_attention_inputs(d, dtype, b, h, kv, d, n), causal=True)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d, h", [(64, 4), (40, 4), (64, 48)])
def test_attention_lengths(dtype, causal, d, h):
    """Lengths of nothing, of one, inside a tile and at its end, and out of range; what lies past
    them is not read."""
    lens = [0, 1, 31, 32, 33, 95, 96, 300, -4]
    n = 97
    q, k, v, g = _attention_inputs(3, dtype, len(lens), h, 2, d, n)
    for t in (q, k, v, g):
        for i, m in enumerate(lens):
            t[i, :, max(0, min(m, n)):] = math.nan
    lengths = torch.tensor(lens, dtype=torch.int32, device=DEV)
    out, lse = ops.attention_forward(q, k, v, causal=causal, lengths=lengths)
    back = ops.attention_backward(g, q, k, v, out, lse, causal=causal, lengths=lengths)
    want = R.attention(*(t.nan_to_num(0.0) for t in (q, k, v, g)), causal=causal,
                       lengths=lengths)
    for name, got in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *back)):
        R.within(got, want[name], name)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("d", [64, 20])
def test_attention_strides(dtype, d):
    """Heads beside each other, heads in reverse of memory order, rows that are not 16-byte
    aligned, one row for all positions and a last stride that is not one."""
    b, h, kv, n = 2, 4, 2, 70
    q, k, v, g = _attention_inputs(5, dtype, b, h, kv, d, n)
    want = R.attention(q, k, v, g, causal=True)

    def beside(t):
        return t.transpose(1, 2).contiguous().transpose(1, 2)

    def odd(t):
        big = torch.empty(*t.shape[:3], d + 3, dtype=dtype, device=DEV)[..., 1:d + 1]
        return big.copy_(t)

    def last(t):
        return t.transpose(2, 3).contiguous().transpose(2, 3)

    def outer(t):
        return t.permute(2, 1, 0, 3).contiguous().permute(2, 1, 0, 3)

    for lay in (beside, odd, last, outer):
        args = [lay(t) for t in (q, k, v, g)]
        out, lse = ops.attention_forward(*args[:3])
        got = (out, lse, *ops.attention_backward(args[3], *args[:3], lay(out), lse))
        for name, x in zip(("out", "lse", "dq", "dk", "dv"), got):
            R.within(x, want[name], f"{name} {lay.__name__}")
    g1 = g[:, :, :1].expand(b, h, n, d)
    out, lse = ops.attention_forward(q, k, v)
    got = ops.attention_backward(g1, q, k, v, out, lse)
    want = R.attention(q, k, v, g1, causal=True)
    for name, x in zip(("dq", "dk", "dv"), got):
        R.within(x, want[name], f"{name} of a broadcast gradient")


@pytest.mark.parametrize("dtype", [F32, BF])
def test_attention_scale_and_large_scores(dtype):
    q, k, v, g = _attention_inputs(6, dtype, 1, 2, 1, 64, 130)
    _attention_check(q, k, v, g, causal=True, scale=0.37)
    _attention_check(q * 16, k * 16, v, g, causal=False, scale=0.01)
    # scores in the thousands: one key takes each row, and no exponential overflows
    out, lse = ops.attention_forward(q * 64, k * 64, v, causal=False, scale=1.0)
    assert bool(out.isfinite().all()) and bool(lse.isfinite().all())


@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("h", [2, 96])
def test_attention_gradients_where_few_keys_are_seen(d, h):
    """What all values of such rows have in common changes no gradient of q and k: no more comes
    of it than the rounding of fp32 sums, though out, rounded to bf16, is off by far more."""
    q, k, v, g = _attention_inputs(d, BF, 8, h, 2, d, 32)
    v = (v + 64).contiguous()
    out, lse = ops.attention_forward(q, k, v)
    dq, dk, _ = ops.attention_backward(g, q, k, v, out, lse)
    want = R.attention(q, k, v, g, causal=True)
    Q, K, V, G = (t.double().cpu() for t in (q, k, v, g))
    rep, scale = h // 2, d ** -0.5
    K, V = K.repeat_interleave(rep, 1), V.repeat_interleave(rep, 1)
    s = (Q @ K.mT * scale).masked_fill(torch.ones(32, 32).triu(1).bool(), -math.inf)
    p = s.softmax(-1)
    dp = G @ V.mT
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    # scores and statistics as in the oracle; a relative error of all p of a row changes their sum
    size = (Q.abs() @ K.abs().mT * scale).amax(-1, keepdim=True)
    rp = (2 * (d + 4) * size + 32 + 8 + 8 * (size + s.logsumexp(-1, keepdim=True).abs())) * R.E32
    edp = (d + 4) * R.E32 * (G.abs() @ V.abs().mT).amax(-1, keepdim=True)
    eds = p * (3 * rp * dp.abs().amax(-1, keepdim=True) + 3 * edp)
    eds = eds + (R.U[BF] + rep * 40 * R.E32) * (ds.abs() + eds)

    def shared(t):
        return t.view(8, 2, rep, 32, d).sum(2)

    R.within(dq, (want["dq"][0], eds @ K.abs() * scale + R.U[BF] * want["dq"][0].abs()), "dq")
    R.within(dk, (want["dk"][0], shared(eds.mT @ Q.abs()) * scale
                  + R.U[BF] * want["dk"][0].abs()), "dk")


@pytest.mark.parametrize("dtype", [F32, BF])
def test_attention_rows_whose_scores_are_all_minus_infinity(dtype):
    """Such a row has no largest score to subtract: zero, like one that sees nothing."""
    q, k, v, g = _attention_inputs(7, dtype, 1, 1, 1, 32, 40)
    q[:], k[:] = 1.0, 1.0
    k[0, 0, :3] = -math.inf
    out, lse = ops.attention_forward(q, k, v)
    assert bool((out[0, 0, :3] == 0).all()) and bool((lse[0, 0, :3] == -math.inf).all())
    assert bool(out[0, 0, 3:].isfinite().all())
    _, _, dv = ops.attention_backward(g, q, k, v, out, lse)
    assert bool(dv.isfinite().all()) and bool((dv[0, 0, :3] == 0).all())


def test_attention_nan_reaches_its_rows():
    q, k, v, _ = _attention_inputs(8, BF, 2, 2, 1, 64, 100)
    q[0, 1, 50] = math.nan
    out, lse = ops.attention_forward(q, k, v)
    assert bool(out[0, 1, 50].isnan().all()) and bool(lse[0, 1, 50].isnan())
    out[0, 1, 50], lse[0, 1, 50] = 0.0, 0.0
    assert bool(out.isfinite().all()) and bool(lse.isfinite().all())


@pytest.mark.parametrize("dtype", [F32, BF])
def test_attention_of_a_large_tensor(dtype):
    """Offsets past 32 bits, in bytes and in elements."""
    n, d = 3, 32
    q, k, v, g = _attention_inputs(9, dtype, 2, 2, 1, d, n)
    step = (1 << 31) + 64
    flat = torch.empty(3 * step, dtype=dtype, device=DEV)

    def far(t):
        return flat.as_strided(t.shape, (256, 2048, step, 1), 4096).copy_(t)

    want = R.attention(q, k, v, g, causal=True)
    for i, name in enumerate(("q", "k", "v")):
        args = [q, k, v]
        args[i] = far(args[i])
        out, lse = ops.attention_forward(*args)
        got = (out, lse, *ops.attention_backward(g, *args, out, lse))
        for x, y in zip(("out", "lse", "dq", "dk", "dv"), got):
            R.within(y, want[x], f"{x} far {name}")


@pytest.mark.parametrize("dtype", [F32, BF])
def test_attention_gradients_against_differences(dtype):
    """Along a direction, the 64-bit output's central difference."""
    q, k, v, g = _attention_inputs(10, dtype, 1, 4, 2, 16, 37)
    _, _, dq, dk, dv = _attention_check(q, k, v, g, causal=True)
    want = R.attention(q, k, v, g, causal=True)
    rnd = _gen(11)
    for i, (name, got) in enumerate((("dq", dq), ("dk", dk), ("dv", dv))):
        args = [t.double().cpu() for t in (q, k, v)]
        way = torch.randn(args[i].shape, generator=rnd, dtype=torch.float64)
        vals = []
        for eps in (1e-4, -1e-4):
            moved = list(args)
            moved[i] = args[i] + eps * way
            o = R.attention(*(m.float().double() if False else _Exact(m) for m in moved),
                            _Exact(g.double().cpu()), causal=True)["out"][0]
            vals.append(float((o * g.double().cpu()).sum()))
        diff = (vals[0] - vals[1]) / 2e-4
        bound = float((want[name][1] * way.abs()).sum()) + 1e-5 * (1 + abs(diff))
        assert abs(float((got.double().cpu() * way).sum()) - diff) <= bound, name


class _Exact:
    """A 64-bit tensor where the oracle takes one of the operators' types."""

    def __init__(self, t):
        self.t, self.dtype, self.shape = t, F32, t.shape

    def double(self):
        return self.t


# ---- the loss -------------------------------------------------------------------------------

def _loss_inputs(seed, dtype, rows, d, vocab):
    g = _gen(seed)
    x, w = _rand(g, rows, d, dtype=dtype), _rand(g, vocab, d, dtype=dtype, std=1.5 / d**0.5)
    t = torch.randint(0, vocab, (rows,), generator=g)
    weights = torch.rand(rows, generator=g) / max(rows, 1)
    if rows > 3:
        weights[torch.rand(rows, generator=g) < 0.25] = 0
        t[1], t[rows // 2] = -100, vocab - 1
    return x, w, t.to(DEV), weights.to(DEV)


def _loss_check(x, w, t, weights):
    loss, lse = ops.vocab_loss_forward(x, w, t)
    dx, dw = ops.vocab_loss_backward(weights, x, w, t, lse)
    want = R.vocab_loss(x, w, t, weights)
    for name, got in (("loss", loss), ("lse", lse), ("dx", dx), ("dw", dw)):
        R.within(got, want[name], name)
    return loss, lse, dx, dw


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("rows, d, vocab", [
    (1, 1, 1), (1, 32, 90), (2, 100, 128), (7, 64, 129), (33, 288, 255), (127, 8, 1000),
    (128, 128, 256), (129, 63, 257), (300, 65, 511), (257, 576, 2049), (513, 192, 1025)])
def test_loss_sizes(dtype, rows, d, vocab):
    _loss_check(*_loss_inputs(rows, dtype, rows, d, vocab))


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("rows", [5, 140])
def test_loss_of_several_pieces(dtype, rows):
    """A vocabulary longer than a piece of it, of a last piece that is odd."""
    _loss_check(*_loss_inputs(21, dtype, rows, 64, 40003))


@pytest.mark.parametrize("rows", [1, 32, 33, 64, 65, 210, 768, 769])
@pytest.mark.parametrize("d, vocab", [(32, 90), (576, 257), (2048, 1300)])
def test_loss_of_fp32_rows_read_where_they_lie(rows, d, vocab):
    """Whole stages on 16-byte borders, rows apart from each other, and around the number of rows
    from which operands are laid out instead."""
    x, w, t, wt = _loss_inputs(rows + d, F32, rows, d, vocab)
    far_x = torch.full((rows, d + 32), math.nan, device=DEV)[:, 32:].copy_(x)
    far_w = torch.full((vocab, d + 4), math.nan, device=DEV)[:, 4:].copy_(w)
    want = R.vocab_loss(x, w, t, wt)
    for a, b in ((x, w), (far_x, far_w), (far_x[:, 1:], far_w[:, 1:])):
        if a.shape[1] < d:
            want = R.vocab_loss(a, b, t, wt)
        loss, lse = ops.vocab_loss_forward(a, b, t)
        R.within(loss, want["loss"], "loss")
        R.within(lse, want["lse"], "lse")
    w[vocab // 2, d - 1] = math.inf
    loss, lse = ops.vocab_loss_forward(x.abs(), w, t)
    assert bool((lse == math.inf).all() | lse.isnan().all())


@pytest.mark.parametrize("rows", [1, 32, 33, 70, 256, 257])
@pytest.mark.parametrize("d, vocab", [(32, 90), (576, 257), (896, 1300)])
def test_loss_gradients_of_few_fp32_rows(rows, d, vocab):
    """One row, the ends of tiles of 32 and 256 rows, and rows apart from each other."""
    _loss_check(*_loss_inputs(rows + d, F32, rows, d, vocab))
    x, w, t, wt = _loss_inputs(rows, F32, rows, d, vocab)
    _loss_check(torch.zeros(rows, d + 3, device=DEV)[:, 3:].copy_(x),
                torch.zeros(vocab, d + 4, device=DEV)[:, 4:].copy_(w), t, wt)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_loss_strides(dtype):
    x, w, t, wt = _loss_inputs(22, dtype, 70, 64, 300)
    want = R.vocab_loss(x, w, t, wt)
    big = torch.full((300, 201), math.nan, dtype=dtype, device=DEV)
    for at in (8, 3):  # rows on 16-byte borders or not
        wide = big[:, at:at + 64].copy_(w)
        tall = torch.empty(70, 67, dtype=dtype, device=DEV)[:, :64].copy_(x)
        for a, b in ((x, wide), (tall, w), (x.t().contiguous().t(), w.t().contiguous().t())):
            loss, lse = ops.vocab_loss_forward(a, b, t)
            dx, dw = ops.vocab_loss_backward(wt, a, b, t, lse)
            for name, got in (("loss", loss), ("lse", lse), ("dx", dx), ("dw", dw)):
                R.within(got, want[name], name)
    R.within(ops.vocab_loss_forward(x, w, t.int())[0], want["loss"], "int32 targets")


@pytest.mark.parametrize("row", [(1 << 22) - 64, (1 << 22) + 64])
def test_loss_of_rows_far_apart(row):
    """Rows of the vocabulary on either side of what a tile's offsets reach."""
    x, w, t, wt = _loss_inputs(28, BF, 40, 64, 600)
    far = torch.empty(600 * row, dtype=BF, device=DEV).as_strided((600, 64), (row, 1)).copy_(w)
    want = R.vocab_loss(x, w, t, wt)
    loss, lse = ops.vocab_loss_forward(x, far, t)
    dx, dw = ops.vocab_loss_backward(wt, x, far, t, lse)
    for name, got in (("loss", loss), ("lse", lse), ("dx", dx), ("dw", dw)):
        R.within(got, want[name], name)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_loss_rows_that_count_for_nothing(dtype):
    """Rows of weight zero or without a target may hold anything."""
    x, w, t, wt = _loss_inputs(23, dtype, 150, 96, 400)
    t[5], wt[9], t[149], wt[149] = -1, 0.0, -100, 1.0
    dead = (t < 0) | (wt == 0)
    want = R.vocab_loss(x, w, t, wt)
    junk = x.clone()
    junk[dead] = math.nan
    _, lse = ops.vocab_loss_forward(junk, w, t)
    dx, dw = ops.vocab_loss_backward(wt, junk, w, t, lse)
    R.within(dx, want["dx"], "dx")
    R.within(dw, want["dw"], "dw")
    total = ops.vocab_loss(junk, w, t, wt)
    assert bool(total.isfinite())
    dx, dw = ops.vocab_loss_backward(torch.zeros_like(wt), junk, w, t, lse)
    assert bool((dx == 0).all()) and bool((dw == 0).all())


def test_loss_of_no_rows():
    _, w, _, _ = _loss_inputs(24, BF, 1, 64, 300)
    x, t = torch.empty(0, 64, dtype=BF, device=DEV), torch.empty(0, dtype=torch.int64, device=DEV)
    wt = torch.empty(0, device=DEV)
    loss, lse = ops.vocab_loss_forward(x, w, t)
    dx, dw = ops.vocab_loss_backward(wt, x, w, t, lse)
    assert loss.shape == (0,) and dx.shape == (0, 64) and bool((dw == 0).all())


@pytest.mark.parametrize("dtype", [F32, BF])
def test_loss_targets_past_the_vocabulary_and_infinite_features(dtype):
    x, w, t, wt = _loss_inputs(25, dtype, 40, 64, 300)
    wt[:] = 1.0
    t[3] = 300
    loss, lse = ops.vocab_loss_forward(x, w, t)
    assert bool(loss[3].isnan()) and int(loss.isnan().sum()) == 1
    dx, _ = ops.vocab_loss_backward(wt, x, w, t, lse)
    assert bool(dx[3].isnan().all()) and int(dx.isnan().any(1).sum()) == 1
    t[3] = 5
    x[7] = math.nan
    loss, _ = ops.vocab_loss_forward(x, w, t)
    assert bool(loss[7].isnan()) and int(loss.isnan().sum()) == 1


@pytest.mark.parametrize("dtype", [F32, BF])
def test_loss_large_logits(dtype):
    """Logits in the thousands: the maximum is taken out before any exponential."""
    x, w, t, wt = _loss_inputs(26, dtype, 66, 64, 700)
    loss, lse = ops.vocab_loss_forward(x * 512, w * 8, t)
    want = R.vocab_loss(x * 512, w * 8, t, wt)
    R.within(loss, want["loss"], "loss")
    R.within(lse, want["lse"], "lse")


# ---- the embedding --------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("tokens, d, vocab", [
    (1, 1, 1), (1, 32, 90), (15, 100, 7), (16, 64, 300), (17, 8, 3), (1024, 576, 500),
    (2047, 36, 90), (2048, 32, 5000), (2049, 30, 1), (5000, 288, 1000), (70001, 4, 64)])
def test_embedding(dtype, tokens, d, vocab):
    g = _gen(tokens)
    ids = torch.randint(-1, vocab + 1, (tokens,), generator=g).to(DEV)
    table, dout = _rand(g, vocab, d, dtype=dtype), _rand(g, tokens, d, dtype=dtype)
    out = ops.embedding_forward(ids, table, scale=0.75)
    inside = (ids >= 0) & (ids < vocab)
    want = table[ids.clamp(0, vocab - 1)].double() * 0.75
    want[~inside] = math.nan
    R.within(out, (want.cpu(), R.U[dtype] * want.abs().cpu()), "rows")
    R.within(ops.embedding_backward(ids, dout, vocab, scale=0.75),
             R.embedding(ids, dout, vocab, 0.75), "gradient")
    into = table.clone()
    got = ops.embedding_backward(ids, dout, vocab, add_to=into)
    assert got is into
    R.within(into, R.embedding(ids, dout, vocab, 1.0, table), "added gradient")


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("tokens", [255, 256, 257, 16384, 16385])
def test_embedding_around_the_counts_that_change_its_path(dtype, tokens):
    g = _gen(tokens)
    ids = (torch.rand(tokens, generator=g) ** 3 * 700).long().to(DEV)
    dout = _rand(g, tokens, 24, dtype=dtype)
    R.within(ops.embedding_backward(ids, dout, 701), R.embedding(ids, dout, 701, 1.0), "gradient")
    into = _rand(g, 701, 24, dtype=dtype)
    want = R.embedding(ids, dout, 701, 1.0, into)
    R.within(ops.embedding_backward(ids, dout, 701, add_to=into), want, "added gradient")


def test_embedding_gradient_of_a_large_table():
    """A dense gradient too large for any cache: every row that no token has is zero."""
    vocab, d = 70001, 1024
    ids = torch.tensor([0, 70000, 35000, 0, 69999], device=DEV)
    dout = _rand(_gen(33), 5, d, dtype=F32)
    torch.full((vocab, d), math.nan, device=DEV)  # what the allocator may hand out again
    got = ops.embedding_backward(ids, dout, vocab)
    assert torch.equal(got[35000], dout[2]) and torch.equal(got[0], dout[0] + dout[3])
    assert torch.equal(got[70000], dout[1]) and torch.equal(got[69999], dout[4])
    assert int((got != 0).any(1).sum()) == 4


def test_embedding_of_frequent_tokens():
    """One token for every position, and one that many pieces of the sorted list share."""
    g = _gen(31)
    for ids in (torch.zeros(40000, dtype=torch.int64),
                torch.where(torch.rand(40000, generator=g) < 0.7, 5,
                            torch.randint(0, 900, (40000,), generator=g))):
        dout = _rand(g, 40000, 20, dtype=F32)
        R.within(ops.embedding_backward(ids.to(DEV), dout, 901),
                 R.embedding(ids, dout, 901, 1.0), "gradient")


@pytest.mark.parametrize("dtype", [F32, BF])
def test_embedding_strides_and_shapes(dtype):
    g = _gen(32)
    ids = torch.randint(0, 50, (3, 7), generator=g).to(DEV)
    wide = _rand(g, 50, 41, dtype=dtype)
    for table in (wide[:, :40], wide[:, 1:33], wide.t()[:, :41]):
        out = ops.embedding_forward(ids.int(), table)
        assert torch.equal(out, table[ids.clamp(max=table.shape[0] - 1)]) or \
            table.shape[0] < 50
    dout = _rand(g, 3, 7, 33, dtype=dtype)[..., :32]
    grad = torch.zeros(50, 40, dtype=dtype, device=DEV)[:, 3:35]
    ops.embedding_backward(ids, dout, 50, add_to=grad)
    R.within(grad, R.embedding(ids, dout, 50, 1.0, torch.zeros(50, 32)), "added gradient")
    none = torch.empty(0, dtype=torch.int64, device=DEV)
    assert ops.embedding_forward(none, wide).shape == (0, 41)
    assert bool((ops.embedding_backward(none, wide[:0], 50) == 0).all())
    one = torch.ones(1, 32, dtype=dtype, device=DEV).expand(21, 32)
    R.within(ops.embedding_backward(ids.reshape(-1), one, 50),
             R.embedding(ids, one, 50, 1.0), "gradient of a broadcast row")


# ---- all of them ----------------------------------------------------------------------------

def _pass(q, k, v, g, x, w, t, wt, ids, rows):
    out, lse = ops.attention_forward(q, k, v)
    loss, l2 = ops.vocab_loss_forward(x, w, t)
    return (out, lse, *ops.attention_backward(g, q, k, v, out, lse), loss, l2,
            *ops.vocab_loss_backward(wt, x, w, t, l2), ops.embedding_forward(ids, w),
            ops.embedding_backward(ids, rows, w.shape[0]))


def _pass_inputs(seed, dtype):
    g = _gen(seed)
    return (*_attention_inputs(seed, dtype, 2, 6, 2, 64, 150),
            *_loss_inputs(seed, dtype, 300, 96, 20001),
            torch.randint(0, 20001, (5000,), generator=g).to(DEV),
            _rand(g, 5000, 96, dtype=dtype))


@pytest.mark.parametrize("dtype", [F32, BF])
def test_same_bits_every_time_and_on_another_stream(dtype):
    args = _pass_inputs(41, dtype)
    first = _pass(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = _pass(*args)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, second):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_captured_and_replayed(dtype):
    """Replays on new inputs, the eager calls between them."""
    args = _pass_inputs(42, dtype)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _pass(*args)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = _pass(*args)
    for seed in (43, 44, 45):
        for a, b in zip(args, _pass_inputs(seed, dtype)):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, _pass(*args)):
            assert torch.equal(a, b)


def test_differentiable_calls():
    """Through autograd: the same gradients as the calls beneath, tensors that need none get
    none, and scaled and broadcast output gradients."""
    q, k, v, g, x, w, t, wt, ids, rows = _pass_inputs(46, F32)
    for a in (q, k, v, x, w):
        a.requires_grad_()
    (ops.attention(q, k, v) * g).sum().backward()
    out, lse = ops.attention_forward(q.detach(), k.detach(), v.detach())
    for a, b in zip((q, k, v), ops.attention_backward(g, q.detach(), k.detach(), v.detach(), out,
                                                      lse)):
        assert torch.equal(a.grad, b)
    (2 * ops.vocab_loss(x, w, t, wt)).backward()
    want = R.vocab_loss(x.detach(), w.detach(), t, 2 * wt)
    R.within(x.grad, want["dx"], "dx")
    R.within(w.grad, want["dw"], "dw")
    w.grad = None
    (ops.embedding(ids, w, scale=0.5) * rows).sum().backward()
    R.within(w.grad, R.embedding(ids, rows, w.shape[0], 0.5), "embedding")
    ops.attention(q.detach(), k, v.detach()).sum().backward()
    assert q.grad is not None and v.grad is not None


@pytest.mark.parametrize("shape", ["width", "device"])
def test_refusals_on_the_gpu(shape):
    q, k, v, g = _attention_inputs(47, F32, 1, 2, 1, 16, 5)
    with pytest.raises(ValueError):
        if shape == "width":
            ops.attention_forward(q, k[..., :8], v)
        else:
            ops.attention_forward(q, k.cpu(), v)


# ---- what else autograd and strides do ---------------------------------------------------------

@pytest.mark.parametrize("which", [0, 1, 2])
def test_only_the_tensor_that_wants_a_gradient_gets_one(which):
    q, k, v, g, x, w, t, wt, ids, rows = _pass_inputs(48, F32)
    out, lse = ops.attention_forward(q, k, v)
    want = ops.attention_backward(g, q, k, v, out, lse)[which]
    (q, k, v)[which].requires_grad_()
    (ops.attention(q, k, v) * g).sum().backward()
    for i, a in enumerate((q, k, v)):
        assert (a.grad is None) == (i != which)
    assert torch.equal((q, k, v)[which].grad, want)
    _, lse = ops.vocab_loss_forward(x, w, t)
    want = (*ops.vocab_loss_backward(wt, x, w, t, lse), ops.vocab_loss_forward(x, w, t)[0])[which]
    (x, w, wt)[which].requires_grad_()
    ops.vocab_loss(x, w, t, wt).backward()
    for i, a in enumerate((x, w, wt)):
        assert (a.grad is None) == (i != which)
    assert torch.equal((x, w, wt)[which].grad, want)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_embedding_of_a_transposed_table(dtype):
    g = _gen(49)
    table = _rand(g, 41, 50, dtype=dtype).t()
    ids = torch.randint(-2, 60, (3, 40), generator=g).to(DEV)
    inside = (ids >= 0) & (ids < 50)
    out = ops.embedding_forward(ids, table)
    assert table.shape == (50, 41) and 0 < int(inside.sum()) < 120
    assert torch.equal(out[inside], table[ids[inside]]) and bool(out[~inside].isnan().all())


@pytest.mark.parametrize("dtype", [F32, BF])
def test_loss_weights_gradient_against_the_formula(dtype):
    x, w, t, wt = _loss_inputs(50, dtype, 70, 64, 300)
    x[69], wt[69] = math.nan, 0.0
    wt.requires_grad_()
    (0.5 * ops.vocab_loss(x, w, t, wt)).backward()
    want, bound = R.vocab_loss(x[:69], w, t[:69], wt[:69].detach())["loss"]
    R.within(wt.grad[:69], (0.5 * want, 0.5 * bound), "the weights' gradient")
    assert float(wt.grad[69]) == 0.0 and int((wt[:69] == 0).sum()) > 0
