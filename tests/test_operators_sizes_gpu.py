"""The training pass's operators at sizes past one launch, one piece or one cache, and on the tiles
that large products take. Which launches the sizes reach is asserted in test_operator_launches.py."""

from __future__ import annotations

import math

import pytest
import torch

import operators_oracle as R
from verification.computation import operators as ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


def _gen(seed):
    return torch.Generator().manual_seed(seed)


# ---- the embedding --------------------------------------------------------------------------

def test_embedding_of_rows_past_a_launch():
    """2^32 chunks of 16 bytes, 64 GiB."""
    tokens, d, vocab = 1 << 24, 1024, 1000
    g = torch.Generator(device=DEV).manual_seed(1)
    table = torch.randn(vocab, d, generator=g, device=DEV)
    ids = torch.randint(0, vocab, (tokens,), generator=g, device=DEV)
    out = ops.embedding_forward(ids, table)
    for part in (slice(i, i + (1 << 18)) for i in range(0, tokens, 1 << 18)):
        assert torch.equal(out[part], table[ids[part]])


@pytest.mark.parametrize("tokens", [3, 300])
def test_embedding_gradient_of_a_table_past_a_launch(tokens):
    """16 rows of zeros a block would be 2^32 threads."""
    vocab, d = (1 << 28) + 5, 8
    ids = torch.randint(0, vocab, (tokens,), generator=_gen(tokens))
    ids[0], ids[1], ids[2] = vocab - 1, 0, 1 << 27
    dout = torch.randn(tokens, d, generator=_gen(2)).to(BF)
    torch.full((vocab, d), math.nan, dtype=BF, device=DEV)  # what the allocator hands out again
    got = ops.embedding_backward(ids.to(DEV), dout.to(DEV), vocab)
    rows, at = ids.unique(return_inverse=True)
    want, bound = R.embedding(at, dout, len(rows), 1.0)
    R.within(got[rows.to(DEV)], (want, bound), "rows with tokens")
    got[rows.to(DEV)] = 0
    for part in got.split(1 << 24):
        assert not bool(part.any())  # (a NaN is not zero)


# tokens, dim, vocab of fp32 tables past the last cache, whose zeros are written beside the ordering
# (and the merge), the sums and the joins
TABLES = [(300, 1024, 70001), (5000, 1024, 70001), (20000, 700, 110003)]


@pytest.mark.parametrize("tokens, d, vocab", TABLES)
def test_embedding_gradient_of_large_tables_beside_the_ordering(tokens, d, vocab):
    g = _gen(tokens)
    ids = (torch.rand(tokens, generator=g, dtype=torch.float64) ** 3 * vocab).long()
    ids[0], ids[1], ids[2], ids[3] = vocab - 1, 0, vocab, -1
    dout = torch.randn(tokens, d, generator=g)
    torch.full((vocab, d), math.nan, device=DEV)  # what the allocator hands out again
    got = ops.embedding_backward(ids.to(DEV), dout.to(DEV), vocab, scale=0.5)
    R.within(got, R.embedding(ids, dout, vocab, 0.5), "gradient")


@pytest.mark.parametrize("dtype", [F32, BF])
def test_embedding_added_to_single_values_and_to_a_single_row(dtype):
    g = _gen(5)
    ids = torch.randint(-1, 301, (700,), generator=g)
    one = torch.randn(700, 1, generator=g).to(dtype)
    into = torch.randn(1, 300, generator=g).to(dtype).to(DEV).t()
    want = R.embedding(ids, one, 300, 1.0, into)
    assert ops.embedding_backward(ids.to(DEV), one.to(DEV), 300, add_to=into) is into
    R.within(into, want, "single values")
    rows = torch.randn(700, 40, generator=g).to(dtype)
    into = torch.randn(40, generator=g).to(dtype).to(DEV).as_strided((1, 40), (0, 1))
    want = R.embedding(ids, rows, 1, 1.0, into)
    ops.embedding_backward(ids.to(DEV), rows.to(DEV), 1, add_to=into)
    R.within(into, want, "a single row")


# ---- the loss -------------------------------------------------------------------------------

def _loss_inputs(seed, dtype, rows, d, vocab):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(rows, d, generator=g, device=DEV).to(dtype)
    w = (torch.randn(vocab, d, generator=g, device=DEV) * (1.5 / d**0.5)).to(dtype)
    t = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
    weights = torch.rand(rows, generator=g, device=DEV) / rows
    weights[torch.rand(rows, generator=g, device=DEV) < 0.25] = 0
    t[1], t[rows // 2], t[rows - 1] = -100, vocab - 1, vocab - 2
    return x, w, t, weights


# dtype, rows, dim, vocab; then what they reach: the tiles of the forward pass, of the backward
# pass's two products, and the pieces of the vocabulary each way.
DIRECT, NARROW_DIRECT = "128u, 64u, 4u, 1u, 2u, true", "256u, 32u, 8u, 1u, 4u, true"
LARGE, MEDIUM, NARROW = "256u, 256u", "128u, 128u", "256u, 32u, 8u, 1u, 4u, false"
TRIMMED, NARROW_X = "192u, 256u", "256u, 32u, 8u, 1u, 2u"
LOSSES = [
    (BF, 300, 64, 32769, LARGE, TRIMMED, TRIMMED, 1, 1),
    (F32, 300, 64, 32769, DIRECT, TRIMMED, TRIMMED, 1, 1),
    (BF, 300, 256, 32769, LARGE, LARGE, LARGE, 1, 1),
    (F32, 300, 256, 32769, DIRECT, LARGE, LARGE, 1, 1),
    (BF, 1100, 1536, 17001, LARGE, LARGE, LARGE, 1, 1),
    (F32, 1024, 576, 49152, LARGE, TRIMMED, TRIMMED, 1, 1),
    (F32, 900, 1001, 20003, LARGE, LARGE, LARGE, 1, 1),
    # several pieces, the last one odd
    (F32, 2049, 64, 90001, LARGE, TRIMMED, TRIMMED, 1, 3),
    (BF, 4097, 200, 66001, LARGE, LARGE, LARGE, 1, 2),
    (F32, 33, 2001, 46001, MEDIUM, MEDIUM, MEDIUM, 2, 2),
    (F32, 7, 64, 360001, NARROW_DIRECT, NARROW_X, LARGE, 1, 2),
    (F32, 7, 2001, 46001, NARROW, NARROW_X, LARGE, 2, 2),
    (BF, 100, 64, 1200001, MEDIUM, MEDIUM, MEDIUM, 1, 2),
]


@pytest.mark.parametrize("dtype, rows, d, vocab", [case[:4] for case in LOSSES])
def test_loss_on_every_tile_and_over_pieces(dtype, rows, d, vocab):
    x, w, t, weights = _loss_inputs(rows + d, dtype, rows, d, vocab)
    loss, lse = ops.vocab_loss_forward(x, w, t)
    dx, dw = ops.vocab_loss_backward(weights, x, w, t, lse)
    want = R.vocab_loss(x, w, t, weights)
    for name, got in (("loss", loss), ("lse", lse), ("dx", dx), ("dw", dw)):
        R.within(got, want[name], name)


def test_loss_of_more_tiles_than_a_launch():
    """2^23 tiles of 512 threads: several pieces of the vocabulary, though w is read where it lies.
    Some rows against the oracle."""
    rows, d, vocab = (1 << 20) + 5, 64, (1 << 19) + 3
    x, w, t, weights = _loss_inputs(3, BF, rows, d, vocab)
    loss, lse = ops.vocab_loss_forward(x, w, t)
    some = torch.cat([torch.arange(20), torch.arange(rows // 2 - 10, rows // 2 + 10),
                      torch.arange(rows - 10, rows)]).to(DEV)
    want = R.vocab_loss(x[some], w, t[some], weights[some])
    R.within(loss[some], want["loss"], "loss")
    R.within(lse[some], want["lse"], "lse")
    assert bool(loss.isfinite().all()) and bool(lse.isfinite().all())


def test_loss_gradients_of_as_many_rows_as_it_takes():
    """2^24 rows, whose sums one launch of a block a row could not join."""
    rows, d, vocab = 1 << 24, 8, 100
    x, w, t, weights = _loss_inputs(4, BF, rows, d, vocab)
    _, lse = ops.vocab_loss_forward(x, w, t)
    dx = torch.full((rows, d), math.nan, dtype=BF, device=DEV)  # what the allocator hands out again
    del dx
    dx, dw = ops.vocab_loss_backward(weights, x, w, t, lse)
    half = rows // 2
    some = torch.cat([torch.arange(50), torch.arange(half - 50, half + 50),
                      torch.arange(rows - 50, rows)]).to(DEV)
    R.within(dx[some], R.vocab_loss(x[some], w, t[some], weights[some])["dx"], "dx")
    assert bool(dw.isfinite().all()) and not bool(dx.isnan().any())
    assert bool(((dx == 0).all(1) == ((weights == 0) | (t < 0))).all())
