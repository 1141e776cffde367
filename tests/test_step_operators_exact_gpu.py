"""Norms of small integers, whose sums are the same in any order and in 32 bits as in more: every
value of every sum is pinned, in every column and row, at widths and row counts where a launch's blocks
go round.

A sum of integers (or of eighths) below 2^24 of its steps is exact. What is left after it is counted
rounding by rounding, each 2^-24 relative at the most (E32), and does not grow with the row."""

from __future__ import annotations

import pytest
import torch

import step_operators_oracle as R
from verification.computation import operators as ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32
E4M3, I8 = torch.float8_e4m3fn, torch.int8
EPS = 1e-6
E32 = R.E32

# s = 1/sqrt(S·(1/d) + eps): the reciprocal of d, the product, eps itself and its addition, halved by
# the root; then the root, improved once (half of one, and one): 3.5. Two products more for y.
OFF_S, OFF_Y = 4 * E32, 6 * E32


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _ints(g, rows, d, most, dtype):
    return torch.randint(-most, most + 1, (rows, d), generator=g, device=DEV,
                         dtype=torch.int8).to(dtype)


def _powers(g, n, lowest, highest, dtype):
    """Powers of two."""
    some = torch.tensor([2.0**i for i in range(lowest, highest + 1)], dtype=dtype, device=DEV)
    return some[torch.randint(len(some), (n,), generator=g, device=DEV)]


def _within(got, value, bound, what):
    """:func:`step_operators_oracle.within`, on the GPU."""
    assert got.shape == value.shape, what
    off = (got.double() - value).abs() - bound
    assert bool((off <= 0).all()), (what, float(off.max()), int((~(off <= 0)).sum()),
                                    (~(off <= 0)).nonzero()[:4].tolist())


# Rows of up to 64, 128 and 1024 columns are 16, 8 and 4 to a block, wider ones one; a launch has at
# most 4096 blocks forward and 1536 backward: each of these goes round twice and a little, both ways.
MANY = [(131083, 9), (131083, 64), (65541, 100), (32771, 200), (32771, 300), (32771, 700),
        (32771, 1000), (8197, 1100), (8197, 2048), (8197, 2052), (8197, 4100), (8197, 8200)]
# Columns around the ends of lanes', waves' and rows' shares.
WIDE = [(5, d) for d in (1, 2, 3, 5, 63, 257, 511, 513, 769, 1023, 1025, 2047, 2049, 4095, 4097, 6001, 8191,
                         8193, 12289, 16381, 16383, 16384)]


@pytest.mark.parametrize("rows, d", MANY + WIDE)
@pytest.mark.parametrize("xt, rt, ot", [(BF, F32, BF), (F32, None, F32)])
def test_norms_of_integers(rows, d, xt, rt, ot):
    """sum t^2 <= 9 · 16384."""
    g = _gen(rows + d)
    x = _ints(g, rows, d, 2 if rt else 3, xt)
    res = None if rt is None else _ints(g, rows, d, 1, rt)
    w = _powers(g, d, -1, 1, F32)
    y, total, rstd = ops.rms_norm_forward(x, w, eps=EPS, residual=res, out_dtype=ot)
    t = x.double() if res is None else x.double() + res.double()
    assert torch.equal(total.double(), t)
    s = (t.square().sum(1) / d + EPS).rsqrt()
    _within(rstd, s, OFF_S * s, "rstd")
    want = t * s[:, None] * w.double()
    _within(y, want, (OFF_Y + R.U[ot]) * want.abs(), "y")


@pytest.mark.parametrize("rows, d", MANY + WIDE)
@pytest.mark.parametrize("xt, tt, yt, dtotal", [(BF, F32, BF, True), (F32, F32, F32, False)])
def test_norm_gradients_of_integers(rows, d, xt, tt, yt, dtotal):
    """With rstd a power of two (it is the call's argument) dy·h are quarters of at most 6, of at most 131083
    rows, and g·h eighths of at most 12, of at most 16384 columns: both sums are exact."""
    g = _gen(3 * rows + d)
    t, dy = _ints(g, rows, d, 3, tt), _ints(g, rows, d, 2, yt)
    w, s = _powers(g, d, -1, 1, F32), _powers(g, rows, -2, 0, F32)
    dt = _ints(g, rows, d, 3, tt) if dtotal else None
    dx, dres, dw = ops.rms_norm_backward(dy, t, w, s, dtotal=dt, x_dtype=xt)
    h = t.double() * s.double()[:, None]
    assert torch.equal(dw.double(), (dy.double() * h).sum(0))
    gain = dy.double() * w.double()
    hm = h * ((gain * h).sum(1, keepdim=True) / d)
    turned = s.double()[:, None] * (gain - hm)
    want = turned if dt is None else turned + dt.double()
    # the mean: 1 / d and the product (and the two's own); the difference, and the sum with dtotal
    bound = 3 * E32 * (s.double()[:, None] * hm.abs()) + 2 * E32 * turned.abs() + E32 * want.abs()
    _within(dres, want, bound + R.U[tt] * want.abs(), "dresidual")
    _within(dx, want, bound + R.U[xt] * want.abs(), "dx")


@pytest.mark.parametrize("rows, d", MANY + WIDE)
@pytest.mark.parametrize("block", [None, 128])
@pytest.mark.parametrize("dtype", [E4M3, I8])
def test_quantized_norms_of_integers(rows, d, block, dtype):
    """Each row has its largest value in another column than its neighbours, and of another size."""
    g = _gen(5 * rows + d)
    x = _ints(g, rows, d, 1, BF)
    i = torch.arange(rows, device=DEV)
    x[i, i * 37 % d] = (2.0 ** (1 + i % 6)).to(BF)  # sum t^2 <= 16384 + 4096
    w = torch.ones(d, device=DEV)
    q, scales, _ = ops.rms_norm_quantized(x, w, eps=EPS, dtype=dtype, block=block)
    most = 448.0 if dtype == E4M3 else 127.0
    t = x.double()
    y = t * (t.square().sum(1, keepdim=True) / d + EPS).rsqrt()
    groups = torch.nn.functional.pad(y, (0, -d % (block or d))).unflatten(1, (-1, block or d))
    want = (groups.abs().amax(2) / most).clamp(min=2.0**-126)
    # the division by 448 or 127: a step, two roundings
    _within(scales, want, (OFF_Y + 2 * E32) * want, "scales")
    v = (groups / want[:, :, None]).flatten(1)[:, :d]
    half = torch.full_like(v, 0.5) if dtype == I8 else \
        torch.maximum(v.abs() * 2.0**-4, torch.full_like(v, 2.0**-10))
    # y's, the scale's and the division's
    _within(q.float(), v, half + (2 * OFF_Y + 4 * E32) * v.abs(), "q")
