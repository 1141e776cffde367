"""What a step does between its products and after them, against the formulas in 64 bits
(step_operators_oracle), at the sizes, types, strides and values where a kernel can go wrong."""

from __future__ import annotations

import itertools
import math

import pytest
import torch

import step_operators_oracle as R
from verification.computation import operators as ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32
E4M3, I8 = torch.float8_e4m3fn, torch.int8
EPS = 1e-6


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _rand(g, *shape, dtype=F32, std=1.0):
    return (torch.randn(*shape, generator=g) * std).to(dtype).to(DEV)


# ---- the norm -------------------------------------------------------------------------------

def _norm_check(x, w, residual, out_dtype, *, eps=EPS, dy=None, dtotal=None):
    y, total, rstd = ops.rms_norm_forward(x, w, eps=eps, residual=residual, out_dtype=out_dtype)
    want = R.norm(x, w, residual, eps, out_dtype)
    for name, got in (("y", y), ("total", total), ("rstd", rstd)):
        R.within(got, want[name], name)
    assert y.dtype == out_dtype and total.dtype == (x if residual is None else residual).dtype
    if dy is None:
        return
    got = ops.rms_norm_backward(dy, total, w, rstd, dtotal=dtotal, x_dtype=x.dtype)
    want = R.norm_backward(dy, total, w, eps, dtotal, x.dtype)
    for name, t, like in zip(("dx", "dresidual", "dweight"), got, (x, total, w)):
        R.within(t, want[name], name)
        assert t.dtype == like.dtype


def _norm_inputs(seed, rows, d, xt, rt, wt, ot):
    g = _gen(seed)
    x = _rand(g, rows, d, dtype=xt)
    res = None if rt is None else _rand(g, rows, d, dtype=rt, std=3.0)
    total = xt if rt is None else rt
    return (x, (1 + _rand(g, d, std=0.3)).to(wt), res, ot), \
        {"dy": _rand(g, rows, d, dtype=ot), "dtotal": _rand(g, rows, d, dtype=total)}


WIDTHS = [1, 2, 3, 4, 5, 6, 7, 8, 63, 64, 255, 256, 257, 511, 513, 896, 1000, 1025, 1536, 1537, 2047,
          2049, 4095, 4097, 8191, 8193, 16383, 16384]


@pytest.mark.parametrize("d", WIDTHS)
@pytest.mark.parametrize("xt, rt, wt, ot", [(BF, F32, F32, BF), (F32, None, BF, F32)])
def test_norm_widths(d, xt, rt, wt, ot):
    args, grads = _norm_inputs(d, 5, d, xt, rt, wt, ot)
    _norm_check(*args, **grads)


@pytest.mark.parametrize("xt, rt, wt, ot",
                         itertools.product([F32, BF], [None, F32, BF], [F32, BF], [F32, BF]))
@pytest.mark.parametrize("d", [130, 2500])
def test_norm_types(xt, rt, wt, ot, d):
    args, grads = _norm_inputs(7, 37, d, xt, rt, wt, ot)
    _norm_check(*args, **grads)
    _norm_check(*args, dy=grads["dy"])


@pytest.mark.parametrize("rows, d", [(1, 896), (2, 3), (4, 64), (2049, 40), (70001, 9), (9000, 257),
                                     (1100, 2052), (600, 8200)])
def test_norm_rows(rows, d):
    """More rows than a launch has waves, in both directions."""
    args, grads = _norm_inputs(rows, rows, d, BF, F32, F32, BF)
    _norm_check(*args, **grads)


@pytest.mark.parametrize("d", [96, 101])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_norm_strides(d, dtype):
    """Rows inside wider rows at odd offsets, one row for all, columns that do not follow each
    other, and more than two dimensions."""
    g = _gen(d)
    w = _rand(g, 2 * d, dtype=dtype)[::2]
    wide = [_rand(g, 3, 7, d + 5, dtype=dtype) for _ in range(4)]
    x, res, dy, dt = (t[..., 3:d + 3] for t in wide)
    _norm_check(x, w, res, dtype, dy=dy, dtotal=dt)
    _norm_check(x[:1, :1].expand(3, 7, d), w, res, dtype, dy=dy[:, :1].expand(3, 7, d), dtotal=dt)
    t = _rand(g, d, 21, dtype=dtype).t()
    _norm_check(t, w, t.flip(0), dtype, dy=t, dtotal=t.flip(0))
    # consecutive values at every offset from a 16-byte border
    flat = _rand(g, 9 * d + 8, dtype=dtype)
    for at in range(8):
        _norm_check(flat[at:at + 9 * d].view(9, d), w, None, dtype)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_norm_special_rows(dtype):
    """A row of zeros is zeros, and NaN and infinities stay in their rows."""
    g = _gen(0)
    x, w = _rand(g, 8, 300, dtype=dtype), _rand(g, 300, dtype=dtype)
    x[1] = 0
    x[3, 17], x[5, 299], x[6, 0] = math.nan, math.inf, 2.0**-120
    y, _, rstd = ops.rms_norm_forward(x, w, eps=1e-5)
    good = [0, 1, 2, 4, 6, 7]
    want = R.norm(x[good], w, None, 1e-5, dtype)
    R.within(y[good], want["y"], "y")
    R.within(rstd[good], want["rstd"], "rstd")
    assert bool((y[1] == 0).all()) and bool(y[3].isnan().all()) and bool(y[5, 299].isnan())
    assert bool((y[5, :299] == 0).all()) and float(rstd[5]) == 0.0
    dy = _rand(g, 8, 300, dtype=dtype)
    dx, _, dw = ops.rms_norm_backward(dy, x, w, rstd)
    assert bool(dx[3].isnan().all()) and bool(dw[17].isnan())
    R.within(dx[good], R.norm_backward(dy[good], x[good], w, 1e-5, None, dtype)["dx"], "dx")


def test_norm_of_no_rows():
    w = torch.ones(8, device=DEV)
    x = torch.zeros(2, 0, 8, device=DEV)
    y, total, rstd = ops.rms_norm_forward(x, w, residual=x)
    assert y.shape == total.shape == x.shape and rstd.shape == (2, 0)
    dx, _, dw = ops.rms_norm_backward(y, total, w, rstd, x_dtype=BF)
    assert dx.shape == x.shape and bool((dw == 0).all())
    q, scales, _ = ops.rms_norm_quantized(x, w, block=32)
    assert q.shape == x.shape and scales.shape == (2, 0, 1)


def test_norm_rows_past_32_bits():
    """Rows 2^31 elements apart, in every tensor that may lie so."""
    g = _gen(1)
    d, far = 260, (1 << 31) + 8
    big = torch.zeros(far + 1024, dtype=BF, device=DEV)

    def apart(at):
        t = big.as_strided((2, d), (far, 1), at)
        return t.copy_(_rand(g, 2, d, dtype=BF))

    x, res, dy = (apart(at) for at in (0, 261, 522))
    _norm_check(x, _rand(g, d), res, BF, dy=dy)
    y, _, rstd = ops.rms_norm_forward(x, _rand(g, d))
    w = torch.ones(d, device=DEV)
    dx = ops.rms_norm_backward(dy, x, w, rstd, dtotal=res)[0]
    R.within(dx, R.norm_backward(dy, x, w, EPS, res, BF)["dx"], "dx")


@pytest.mark.parametrize("rt", [None, F32, BF])
def test_norm_gradients_by_differences(rt):
    """The differentiable form against slopes of the formula itself."""
    g = _gen(3)
    rows, d = 6, 44
    leaves = [_rand(g, rows, d), _rand(g, d), None if rt is None else _rand(g, rows, d, dtype=rt)]
    out = [_rand(g, rows, d), _rand(g, rows, d)]
    for t in leaves:
        if t is not None:
            t.requires_grad_()
    if rt is None:
        y = ops.rms_norm(leaves[0], leaves[1], eps=EPS)
        (y * out[0]).sum().backward()
    else:
        y, total = ops.rms_norm(leaves[0], leaves[1], eps=EPS, residual=leaves[2])
        ((y * out[0]).sum() + (total.float() * out[1]).sum()).backward()
    values = [None if t is None else t.detach().double().cpu() for t in leaves]
    o = [t.double().cpu() for t in out]

    def f(which, v):
        x, w, r = (v if i == which else t for i, t in enumerate(values))
        t = x if r is None else x + r
        y = t * (t.square().mean(1, keepdim=True) + EPS).rsqrt() * w
        return (y * o[0]).sum() + (0 if r is None else (t * o[1]).sum())

    for i, t in enumerate(leaves):
        if t is None:
            continue
        along = torch.randn(values[i].shape, generator=g, dtype=torch.float64)
        want = R.difference(lambda v: f(i, v), values[i], along)
        got = float((t.grad.double().cpu() * along).sum())
        # dots of at most 264 terms of gradients that are off by the sum's rounding to its type
        size = float((t.grad.double().cpu() * along).abs().sum())
        off = 4 * R.U[BF if rt == BF else F32] + (d + 16) * R.E32 * 4
        assert abs(got - want) <= off * size + 1e-6, i


@pytest.mark.parametrize("dtype", [F32, BF])
def test_norm_gradients_of_broadcast_inputs(dtype):
    """One row for all of a batch, one weight for two norms, and one tensor as branch and residual."""
    g = _gen(13)
    rows, d = 50, 70
    row, w = _rand(g, 1, d, dtype=dtype).requires_grad_(), _rand(g, d).requires_grad_()
    res = _rand(g, rows, d)
    o = [_rand(g, rows, d, dtype=dtype), _rand(g, 1, d, dtype=dtype)]
    y, total = ops.rms_norm(row.expand(rows, d), w, residual=res)
    z, double = ops.rms_norm(row, w, residual=row)
    torch.autograd.backward([y, z], o)
    first = R.norm_backward(o[0], total.detach(), w.detach(), 1e-6, None, dtype)
    other = R.norm_backward(o[1], double.detach(), w.detach(), 1e-6, None, dtype)
    R.within(w.grad, tuple(a + b for a, b in zip(first["dweight"], other["dweight"])), "dw")
    # torch adds up the rows' gradients and the three shares, in fp32 or rounding each sum to the type
    shares = [(first["dx"][0], first["dx"][1]), (2 * other["dx"][0], 2 * other["dx"][1])]
    value = sum(v.sum(0, keepdim=True) for v, _ in shares)
    size = sum(v.abs().sum(0, keepdim=True) for v, _ in shares)
    bound = sum(b.sum(0, keepdim=True) for _, b in shares)
    R.within(row.grad, (value, bound + (rows * R.E32 + 3 * R.U[dtype]) * size), "dx")


def test_norm_gradients_where_one_output_is_unused():
    g = _gen(4)
    x, r = _rand(g, 3, 40, dtype=BF).requires_grad_(), _rand(g, 3, 40).requires_grad_()
    w = _rand(g, 40).requires_grad_()
    o = _rand(g, 3, 40)
    _, total = ops.rms_norm(x, w, residual=r)
    (total * o).sum().backward()
    assert torch.equal(r.grad, o) and torch.equal(x.grad, o.to(BF)) and w.grad is None
    r.grad = None
    y, total = ops.rms_norm(x, w, residual=r)
    (dr,) = torch.autograd.grad((y.float() * o).sum(), [r])
    R.within(dr, R.norm_backward(o.to(BF), total.detach(), w.detach(), 1e-6, None, F32)["dx"], "dr")


@pytest.mark.parametrize("rows, d", [(3, 40), (2000, 300), (700, 2100), (300, 9000)])
@pytest.mark.parametrize("residual", [False, True])
def test_norm_gradients_without_the_weights(rows, d, residual, monkeypatch):
    """A gain that is frozen has no gradient, and nothing is summed for it; the others' bits are the same."""
    from verification.commitment import native
    g = _gen(15)
    x, w = _rand(g, rows, d, dtype=BF), _rand(g, d)
    res, o = _rand(g, rows, d) if residual else None, _rand(g, rows, d, dtype=BF)
    calls = []
    lib = native.get()
    run = lib.operator

    def operator(name, args, device):
        calls.append((name, args))
        return run(name, args, device)

    monkeypatch.setattr(lib, "operator", operator)
    got = []
    for frozen in (False, True):
        leaves = [t.detach().clone().requires_grad_() for t in (x, res) if t is not None]
        gain = w.clone().requires_grad_(not frozen)
        y = ops.rms_norm(leaves[0], gain, residual=leaves[1] if residual else None)
        (y[0] if residual else y).backward(o)
        got.append([t.grad for t in leaves])
        name, args = calls.pop()
        assert name == "rms_norm_backward" and (gain.grad is None) == frozen
        assert (ops._NORM.unpack(args)[11] == 0) == frozen  # where dweight goes
    for a, b in zip(*got):
        assert torch.equal(a, b)


# ---- 8 bits ---------------------------------------------------------------------------------

def _quantized_check(x, w, residual, dtype, block):
    q, scales, total = ops.rms_norm_quantized(x, w, eps=EPS, residual=residual, dtype=dtype,
                                              block=block)
    want = R.quantized(x, w, residual, EPS, dtype, block)
    assert q.dtype == dtype and torch.equal(total.cpu(), R.added(x, residual))
    R.within(scales, want["scales"], "scales")
    R.within(q.float(), want["q"], "q")


@pytest.mark.parametrize("d", [1, 2, 3, 5, 31, 33, 64, 127, 129, 256, 260, 897, 1536, 2050, 4100,
                               8192, 9001, 16384])
@pytest.mark.parametrize("block", [None, 32, 64, 128, 256])
@pytest.mark.parametrize("dtype", [E4M3, I8])
def test_quantized_widths(d, block, dtype):
    args, _ = _norm_inputs(d, 5, d, BF, F32, F32, BF)
    _quantized_check(*args[:3], dtype, block)


@pytest.mark.parametrize("xt, rt, wt", itertools.product([F32, BF], [None, F32, BF], [F32, BF]))
@pytest.mark.parametrize("dtype", [E4M3, I8])
def test_quantized_types(xt, rt, wt, dtype):
    args, _ = _norm_inputs(9, 300, 700, xt, rt, wt, BF)
    _quantized_check(*args[:3], dtype, None)
    _quantized_check(*args[:3], dtype, 64)


@pytest.mark.parametrize("dtype", [E4M3, I8])
@pytest.mark.parametrize("block", [None, 32])
def test_quantized_special_blocks(dtype, block):
    """Zeros; a NaN, an infinity and the smallest numbers in one block of a row."""
    g = _gen(5)
    x = _rand(g, 6, 96)
    w = torch.ones(96, device=DEV)
    x[0] = 0
    q, scales, _ = ops.rms_norm_quantized(x, w, dtype=dtype, block=block)
    assert bool((q[0].float() == 0).all()) and bool((scales[0] == 2.0**-126).all())
    w[40] = math.nan
    q, scales, _ = ops.rms_norm_quantized(x[1:], w, dtype=dtype, block=block)
    if block is None:
        assert bool(scales.isnan().all())
    else:
        assert bool(scales[:, 1].isnan().all()) and bool(scales[:, ::2].isfinite().all())
        plain = ops.rms_norm_quantized(x[1:], torch.ones(96, device=DEV), dtype=dtype, block=block)
        assert torch.equal(q[:, :32].float(), plain[0][:, :32].float())
        assert torch.equal(scales[:, ::2], plain[1][:, ::2])
    w[40] = math.inf
    q, scales, _ = ops.rms_norm_quantized(x[1:], w, dtype=dtype, block=block)
    part = scales if block is None else scales[:, 1:2]
    assert bool(part.isinf().all()) and bool((q[:, 41:64].float() == 0).all())
    w.fill_(1e-37)  # sizes whose scale would be no normal number
    q, scales, _ = ops.rms_norm_quantized(x[1:], w, dtype=dtype, block=block)
    assert bool((scales == 2.0**-126).all())
    R.within(q.float(), R.quantized(x[1:], w, None, 1e-6, dtype, block)["q"], "q")


@pytest.mark.parametrize("dtype", [E4M3, I8])
def test_quantized_numbers_that_are_none(dtype):
    """Where y / scale is NaN, the type's NaN or -128; int8 has that number for nothing else."""
    x, w = _rand(_gen(14), 5, 96), torch.ones(96, device=DEV)

    def none(q):
        return q.float().isnan() if dtype == E4M3 else q == -128

    q, _, _ = ops.rms_norm_quantized(x, w, dtype=dtype, block=32)
    assert not bool(none(q).any())
    for bad in (math.nan, math.inf, -math.inf):
        w[40] = bad
        q, _, _ = ops.rms_norm_quantized(x, w, dtype=dtype, block=32)
        want = torch.zeros(96, dtype=torch.bool, device=DEV)
        want[slice(32, 64) if math.isnan(bad) else 40] = True
        assert torch.equal(none(q), want.expand(5, 96))
        if not math.isnan(bad):
            assert bool((q[:, 32:64].float()[:, torch.arange(32) != 8] == 0).all())


# ---- rotary positions -----------------------------------------------------------------------

def _rotary_check(q, k, positions, f, **kw):
    b, _, n, _ = q.shape
    sections, adjacent = kw.get("sections"), kw.get("adjacent", False)
    at = positions[None] if sections is None else positions
    at = (at[:, None] if at.dim() == 2 else at).expand(-1, b, n)
    counts = sections or (f.numel(),)
    for call, inverse in ((ops.rotary_forward, False), (ops.rotary_backward, True)):
        for got, t, name in zip(call(q, k, positions, f, **kw), (q, k), "qk"):
            assert got.dtype == t.dtype and got.transpose(1, 2).is_contiguous()
            R.within(got, R.rotary(t, at, f, counts, adjacent, inverse), name)


def _heads(g, b, h, kv, d, n, dtype):
    return _rand(g, b, h, n, d, dtype=dtype), _rand(g, b, kv, n, d, dtype=dtype)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("d, width", [(2, 2), (3, 2), (4, 4), (6, 6), (7, 4), (8, 8), (10, 10), (14, 14),
                                      (16, 16), (20, 18), (24, 24), (31, 16), (32, 8), (40, 2),
                                      (64, 64), (80, 80), (96, 32), (100, 100), (128, 126),
                                      (129, 128), (256, 256), (1000, 500), (1024, 1024)])
def test_rotary_widths(dtype, adjacent, d, width):
    q, k = _heads(_gen(d), 2, 3, 1, d, 5, dtype)
    at = torch.randint(-50, 5000, (2, 5), generator=_gen(1)).to(DEV)
    _rotary_check(q, k, at, R.by_frequency(width).to(DEV), adjacent=adjacent)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("b, h, kv, d, n", [(1, 1, 1, 64, 1), (16, 14, 2, 64, 1), (3, 6, 2, 32, 257),
                                            (2, 14, 2, 64, 1021), (1, 9, 9, 128, 2050),
                                            (300, 2, 1, 16, 33), (1, 70, 3, 64, 7), (5, 1, 1, 4, 4000)])
def test_rotary_sizes(dtype, b, h, kv, d, n):
    """One token and many, each block full of them or not."""
    g = _gen(n)
    q, k = _heads(g, b, h, kv, d, n, dtype)
    _rotary_check(q, k, torch.arange(n, device=DEV), R.by_frequency(d).to(DEV))
    at = torch.randint(0, 1 << 20, (b, n), generator=g).to(DEV)
    _rotary_check(q, k, at, R.by_frequency(d).float().to(DEV), adjacent=True)


@pytest.mark.parametrize("sections", [(24,), (4, 20), (8, 8, 8), (0, 24, 0), (1, 2, 3, 18), (3, 0, 21)])
@pytest.mark.parametrize("shape", ["tokens", "batch", "strided", "int32"])
@pytest.mark.parametrize("adjacent", [False, True])
def test_rotary_axes(sections, shape, adjacent):
    b, n, axes = 3, 29, len(sections)
    g = _gen(2)
    q, k = _heads(g, b, 4, 2, 50, n, BF)
    if shape == "tokens":
        at = torch.randint(0, 900, (axes, n), generator=g)
    elif shape == "strided":
        at = torch.randint(0, 900, (n, b, 2 * axes), generator=g).permute(2, 1, 0)[::2]
    else:
        at = torch.randint(-9, 900, (axes, b, n), generator=g)
    if shape == "int32":
        at = at.int()
    _rotary_check(q, k, at.to(DEV), R.by_frequency(48).to(DEV), sections=sections,
                  adjacent=adjacent)


def test_rotary_far_positions():
    """Of 2^31 a fast pair makes 3e8 turns: 64 bits still hold the angle."""
    g = _gen(6)
    q, k = _heads(g, 1, 2, 1, 64, 6, F32)
    for at in ([0, 1, 1 << 20, (1 << 24) + 1, (1 << 31) - 1, -(1 << 31)],):
        at = torch.tensor(at)
        _rotary_check(q, k, at.to(DEV), R.by_frequency(64, 5e5).to(DEV))
        _rotary_check(q, k, at.int().to(DEV), R.by_frequency(64).to(DEV), adjacent=True)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_rotary_strides(dtype):
    b, h, kv, d, n = 2, 4, 2, 40, 19
    g = _gen(8)
    f, at = R.by_frequency(d).to(DEV), torch.arange(n, device=DEV)

    def beside(c):  # a projection's heads
        return _rand(g, b, n, c, d, dtype=dtype).transpose(1, 2)

    def odd(c):
        return _rand(g, b, c, n, d + 3, dtype=dtype)[..., 1:d + 1]

    def last(c):
        return _rand(g, b, c, d, n, dtype=dtype).transpose(2, 3)

    def one(c):
        return _rand(g, b, 1, n, d, dtype=dtype).expand(b, c, n, d)

    for lay in (beside, odd, last, one):
        _rotary_check(lay(h), lay(kv), at, f)
        _rotary_check(lay(h), lay(kv), at, f[::2], adjacent=True)
    joined = _rand(g, b, n, (h + 2 * kv) * d, dtype=dtype)  # q, k and v of one product
    q, k = (joined[..., i * d:j * d].view(b, n, -1, d).transpose(1, 2)
            for i, j in ((0, h), (h, h + kv)))
    _rotary_check(q, k, at, f)


def test_rotary_of_nothing():
    q, k = torch.zeros(2, 3, 0, 8, device=DEV), torch.zeros(2, 1, 0, 8, device=DEV)
    f = R.by_frequency(8).to(DEV)
    a, b = ops.rotary_forward(q, k, torch.arange(0, device=DEV), f)
    assert a.shape == q.shape and b.shape == k.shape
    a, b = ops.rotary_forward(q[:0], k[:0], torch.zeros(0, 0, dtype=torch.int32, device=DEV), f)
    assert a.shape == (0, 3, 0, 8)


def test_rotary_heads_past_32_bits():
    g = _gen(9)
    far = (1 << 31) + 8
    big = torch.zeros(far + 4096, dtype=BF, device=DEV)
    q = big.as_strided((1, 2, 3, 64), (0, far, 64, 1)).copy_(_rand(g, 1, 2, 3, 64))
    k = big.as_strided((2, 1, 3, 64), (far, 64, 64, 1), 1000).copy_(_rand(g, 2, 1, 3, 64))
    f, at = R.by_frequency(64).to(DEV), torch.arange(3, device=DEV)
    _rotary_check(q, q[:, :1], at, f)
    _rotary_check(k.expand(2, 1, 3, 64), k, at, f)


def test_rotary_gradients():
    """By differences, with a key head that several heads share and q from one product with k."""
    g = _gen(10)
    b, h, n, d = 2, 3, 5, 12
    x = _rand(g, b, n, (h + 1) * d).requires_grad_()
    f, at = R.by_frequency(d).to(DEV), torch.tensor([[0, 3, 9, 11, 2], [7, 7, 1, 0, 5]], device=DEV)
    o = _rand(g, b, h, n, d), _rand(g, b, h, n, d)
    q = x[..., :h * d].view(b, n, h, d).transpose(1, 2)
    k = x[..., h * d:].view(b, n, 1, d).transpose(1, 2).expand(b, h, n, d)
    y = ops.rotary(q, k, at, f)
    sum((a * c).sum() for a, c in zip(y, o)).backward()
    value = x.detach().double().cpu()
    angle = at.cpu()[:, None, :, None].double() * f.cpu()

    def turned(t):
        u, v = t[..., :d // 2], t[..., d // 2:]
        return torch.cat([u * angle.cos() - v * angle.sin(), u * angle.sin() + v * angle.cos()], -1)

    def fn(v):
        q = v[..., :h * d].view(b, n, h, d).transpose(1, 2)
        k = v[..., h * d:].view(b, n, 1, d).transpose(1, 2).expand(b, h, n, d)
        return sum((turned(t) * c.double().cpu()).sum() for t, c in zip((q, k), o))

    along = torch.randn(value.shape, generator=g, dtype=torch.float64)
    got = (x.grad.double().cpu() * along)
    # (linear in x: the difference is exact but for its own rounding)
    assert abs(float(got.sum()) - R.difference(fn, value, along)) <= 1e-6 + 16 * R.E32 * float(
        got.abs().sum()) + 16 * R.E32 * float(along.abs().sum()) * 8


# ---- the gated activation -------------------------------------------------------------------

def _gated_check(gate, up, dout):
    want = R.gated(gate, up, dout)
    got = {"out": ops.gated_silu_forward(gate, up)}
    got["dgate"], got["dup"] = ops.gated_silu_backward(dout, gate, up)
    for name, t in got.items():
        assert t.dtype == gate.dtype and t.is_contiguous()
        R.within(t, want[name], name)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("shape", [(1,), (3,), (7, 1), (5, 2), (4, 3), (2, 5, 7), (9, 8), (3, 9), (33, 100),
                                   (1, 4097), (257, 1023), (1030, 1536), (3, 1, 8960)])
def test_gated_shapes(dtype, shape):
    g = _gen(len(shape))
    _gated_check(*(_rand(g, *shape, dtype=dtype, std=2.0) for _ in range(3)))


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("rows, f", [(1, 5), (6, 96), (31, 101), (2, 3), (300, 4099)])
def test_gated_strides(dtype, rows, f):
    g = _gen(f)
    gate, up = _rand(g, rows, 2 * f, dtype=dtype).split(f, 1)
    dout = _rand(g, rows, f + 3, dtype=dtype)[:, 1:f + 1]
    _gated_check(gate, up, dout)
    _gated_check(gate, up[:1].expand(rows, f), dout[:, :1].expand(rows, f))
    _gated_check(gate.t(), up.t(), dout.t())
    flat = _rand(g, rows * f + 8, dtype=dtype)
    for at in range(8):
        t = flat[at:at + rows * f].view(rows, f)
        _gated_check(t, t, t)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_gated_values(dtype):
    """Far to both sides, where e^-g overflows and where it vanishes; special values as the formula
    has them."""
    x = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 20, -20, 87, -87, -89, -104, -120, 200, -1e30, 1e38],
                     device=DEV).to(dtype)
    one = torch.ones_like(x)
    _gated_check(x, one, one)
    _gated_check(x, 0.5 * one, -3 * one)
    bad = torch.tensor([math.nan, math.inf, -math.inf, 1.0], device=DEV, dtype=dtype)
    got = ops.gated_silu_forward(bad, torch.ones_like(bad))
    assert got[0].isnan() and float(got[1]) == math.inf and got[2].isnan() and got[3].isfinite()
    got = ops.gated_silu_forward(torch.ones_like(bad), bad)
    assert got[0].isnan() and float(got[1]) == math.inf and float(got[2]) == -math.inf


def test_gated_of_nothing_and_rows_past_32_bits():
    x = torch.zeros(0, 5, device=DEV)
    assert ops.gated_silu_forward(x, x).shape == (0, 5)
    assert ops.gated_silu_backward(x.t(), x.t(), x.t())[0].shape == (5, 0)
    g = _gen(11)
    far = (1 << 31) + 8
    big = torch.zeros(far + 4096, dtype=BF, device=DEV)
    gate, up, dout = (big.as_strided((2, 700), (far, 1), at).copy_(_rand(g, 2, 700))
                      for at in (0, 701, 1402))
    _gated_check(gate, up, dout)


def test_gated_gradients_round_no_more_than_their_formula():
    """By their RMS, counted in roundings of 2^-24 · 0.425 each (half a step at most, mantissas as they
    come). d gate is the product of dout and up, the slope of silu, and the product of those two: three roundings, of
    which the slope's counts 1.7 times in the square, since it is most often near 1, where a step is largest.
    The exponential and the products of small g(1 - sigma) are what is left: one and a half, 5.2 in all."""
    n, g = 1 << 20, torch.Generator(device=DEV).manual_seed(21)
    gate, up = (1.5 * torch.randn(n, generator=g, device=DEV) for _ in range(2))
    dout = torch.randn(n, generator=g, device=DEV)
    dgate, _ = ops.gated_silu_backward(dout, gate, up)
    x, v, dy = gate.double(), up.double(), dout.double()
    want = dy * v * torch.sigmoid(x) * (1 + x * torch.sigmoid(-x))
    off = float((dgate.double() - want).norm() / want.norm())
    assert off <= 0.425 * R.E32 * math.sqrt(5.5), off


@pytest.mark.parametrize("dtype", [F32, BF])
def test_gated_slopes_far_out(dtype):
    """To the ends of the type, where g(1 - sigma) and sigma differ by all that it holds."""
    ends = torch.tensor([3e38, -3e38, 1.8e38, -1.8e38, 1e37, -1e37, 1e-38, -1e-38], device=DEV).to(dtype)
    x = torch.cat([ends, torch.linspace(-110, 110, 2201, device=DEV).to(dtype)])
    _gated_check(x, torch.ones_like(x), torch.ones_like(x))


def test_gated_rows_of_more_than_2_30_values():
    """One tensor without rows, as long as it likes, and rows of such a length."""
    n = (1 << 30) + 11
    x = torch.zeros(2, n, dtype=BF, device=DEV)
    for at in ((1 << 30) - 5, n - 3):  # on both sides of 2^30, and at the end
        x[:, at:at + 8] = _rand(_gen(at % 7), 2, min(8, n - at), dtype=BF)
    ends = [slice((1 << 30) - 9, (1 << 30) + 8), slice(n - 5, n), slice(0, 9)]
    for t in (x[1], x):
        up = t.flip(0) if t.dim() == 2 else t
        out = ops.gated_silu_forward(t, up)
        dg, du = ops.gated_silu_backward(up, t, up)
        for part in ends:
            want = R.gated(t[..., part], up[..., part], up[..., part])
            for name, got in (("out", out), ("dgate", dg), ("dup", du)):
                R.within(got[..., part], want[name], name)
        assert int(out.count_nonzero()) == sum(int(out[..., p].count_nonzero()) for p in ends[:2])
        del out, dg, du


def test_gated_gradients():
    g = _gen(12)
    leaves = [_rand(g, 4, 13).requires_grad_(), _rand(g, 1, 13).requires_grad_()]
    o = _rand(g, 4, 13)
    (ops.gated_silu(leaves[0], leaves[1].expand(4, 13)) * o).sum().backward()
    values = [t.detach().double().cpu() for t in leaves]
    for i, t in enumerate(leaves):
        along = torch.randn(t.shape, generator=g, dtype=torch.float64)

        def f(v):
            gate, up = (v if i == j else x for j, x in enumerate(values))
            return (gate * torch.sigmoid(gate) * up * o.double().cpu()).sum()

        got = t.grad.double().cpu() * along
        # four rows are added up for the broadcast one
        assert abs(float(got.sum()) - R.difference(f, values[i], along)) <= \
            1e-6 + 40 * R.E32 * float(got.abs().sum() + along.abs().sum() * 40)


# ---- the whole gradient ---------------------------------------------------------------------

SHAPES = [(1,), (3,), (7, 5), (0,), (4095,), (4096,), (4097,), (64, 65), (3, 5, 11), (8193,),
          (1023, 33), (1,), (12288,), (2, 2)]


def _gradients(seed, shapes=SHAPES, types=(F32, BF), std=0.1):
    g = _gen(seed)
    return [_rand(g, *s, dtype=types[i % len(types)], std=std) for i, s in enumerate(shapes)]


def _change_check(grads, max_norm, weights=None, eta=1.0, *, out=False):
    want_norm = R.total_norm(grads)
    want = R.changed(grads, max_norm, weights, eta)
    like = grads if weights is None else weights
    to = [torch.full_like(t, 7.0) for t in like] if out else like
    kept = [t.clone() for t in grads] + ([] if weights is None else [t.clone() for t in weights])
    kw = {"out": to} if out else {}
    if weights is None:
        norm = ops.clip_gradients(grads, max_norm, **kw)
    else:
        norm = ops.sgd_step(weights, grads, eta, max_norm=max_norm, **kw)
    assert norm.shape == () and norm.dtype == F32
    R.within(norm, want_norm, "norm")
    for i, (t, w) in enumerate(zip(to, want)):
        R.within(t, w, i)
    for i, (a, b) in enumerate(zip(kept, grads + (weights or []))):
        if out or (weights is not None and i < len(grads)):
            assert torch.equal(a, b), "an input changed"


@pytest.mark.parametrize("types", [(F32,), (BF,), (F32, BF), (BF, F32, F32)])
@pytest.mark.parametrize("max_norm", [0.25, 1e6])
@pytest.mark.parametrize("out", [False, True])
def test_clip(types, max_norm, out):
    grads = _gradients(1, types=types)
    R.within(ops.gradient_norm(grads), R.total_norm(grads), "norm")
    _change_check(grads, max_norm, out=out)


@pytest.mark.parametrize("types", [(F32,), (BF,), (F32, BF, BF)])
@pytest.mark.parametrize("weight_types", [(F32,), (BF,), (BF, F32)])
@pytest.mark.parametrize("max_norm", [0.25, math.inf])
@pytest.mark.parametrize("out", [False, True])
def test_sgd(types, weight_types, max_norm, out):
    _change_check(_gradients(2, types=types), max_norm, _gradients(3, types=weight_types, std=1.0),
                  0.37, out=out)


@pytest.mark.parametrize("count", [1, 95, 96, 97, 160, 161, 337, 700])
def test_tensors_past_a_launch(count):
    shapes = [SHAPES[(i * 5) % len(SHAPES)] for i in range(count)]
    _change_check(_gradients(count, shapes), 0.5)
    _change_check(_gradients(count, shapes), 0.5, _gradients(count + 1, shapes, (F32,)), 0.1, out=True)


@pytest.mark.parametrize("size", [(1 << 23) + 4095, (1 << 23) + 1, 3 * (1 << 23) + 5000])
def test_tensors_of_more_chunks_than_blocks(size):
    grads = _gradients(4, [(size,), (70,), (size // 3, 2)])
    _change_check(grads, 1.0)
    _change_check(grads, 1.0, _gradients(5, [(size,), (70,), (size // 3, 2)], (F32,)), 0.1)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_tensors_that_start_anywhere(dtype):
    """Slices of one buffer at every offset, in place: what lies between them is not touched."""
    sizes = [1, 2, 3, 5, 8, 13, 4097, 21, 4096, 34, 7]
    flat = _rand(_gen(6), sum(sizes) + 2 * len(sizes), dtype=dtype)
    before, at, parts, gaps = flat.clone(), 0, [], []
    for n in sizes:
        parts.append(flat[at:at + n])
        gaps += [at + n, at + n + 1]
        at += n + 2
    want = R.changed(parts, 2.0)
    ops.clip_gradients(parts, 2.0)
    for i, (t, w) in enumerate(zip(parts, want)):
        R.within(t, w, i)
    assert torch.equal(flat[gaps], before[gaps])


def test_a_norm_within_its_bound_changes_nothing():
    grads = _gradients(7)
    kept = [t.clone() for t in grads]
    norm = float(ops.clip_gradients(grads, 1e3))
    assert all(torch.equal(a, b) for a, b in zip(grads, kept)) and norm < 1e3
    # at the bound itself the factor is one, just below it is not
    assert float(ops.clip_gradients([torch.tensor([3.0, 4.0], device=DEV)], 5.0)) == 5.0
    t = torch.tensor([3.0, 4.0], device=DEV)
    ops.clip_gradients([t], 2.5)
    assert t.tolist() == [1.5, 2.0]


def test_sizes_of_gradients():
    """Squares outside fp32 on both sides, and a norm outside it."""
    for size in (1e30, 1e-30, 2e38):
        t = torch.full((1000,), size, device=DEV)
        norm = ops.gradient_norm([t])
        want = size * math.sqrt(1000)
        if want > 3.4e38:
            assert float(norm) == math.inf
            # the factor is taken in 64 bits; at 1.6e-40 a step of fp32 is 2^-149, 9e-6 of it
            ops.clip_gradients([t], 1.0)
            assert torch.allclose(t, torch.full_like(t, 1 / math.sqrt(1000)), rtol=5e-6)
        else:
            assert abs(float(norm) - want) <= 4 * R.E32 * want


def test_norms_that_are_not_finite():
    a, b = torch.ones(5, device=DEV), torch.tensor([1.0, math.inf], device=DEV)
    assert float(ops.clip_gradients([a, b], 1.0)) == math.inf
    assert bool((a == 0).all()) and float(b[0]) == 0 and bool(b[1].isnan())
    a, b = torch.ones(5, device=DEV), torch.tensor([1.0, math.nan], device=DEV, dtype=BF)
    assert math.isnan(float(ops.clip_gradients([a, b], 1.0)))
    assert bool(a.isnan().all()) and bool(b.isnan().all())
    w = torch.ones(5, device=DEV)
    assert math.isnan(float(ops.sgd_step([w], [torch.full((5,), math.nan, device=DEV)], 0.1)))
    assert bool(w.isnan().all())


@pytest.mark.parametrize("types", [(F32, F32), (BF, F32), (BF, BF)])
def test_without_a_bound_values_are_their_own(types):
    """No clip: what is not finite in one gradient is in its own weight alone, in place or not."""
    for bad in (math.nan, math.inf, -math.inf):
        g = [torch.tensor([1.0, bad, -2.0], device=DEV).to(types[0]),
             torch.ones(5000, device=DEV, dtype=types[0])]
        w = [torch.full(t.shape, 3.0, device=DEV, dtype=types[1]) for t in g]
        want = [a.double() - 0.5 * b.double() for a, b in zip(w, g)]  # exact where it is finite
        out = [torch.empty_like(t) for t in w]
        norms = [ops.sgd_step(w, g, 0.5, out=out), ops.sgd_step(w, g, 0.5, max_norm=1e39),
                 ops.clip_gradients(g, math.inf), ops.gradient_norm(g)]
        for to in (out, w):
            assert all(torch.equal(a.double().nan_to_num(7e9, 8e9, 9e9), b.nan_to_num(7e9, 8e9, 9e9))
                       for a, b in zip(to, want))
        for n in norms:
            assert math.isnan(float(n)) if math.isnan(bad) else float(n) == math.inf
        assert bool((g[1] == 1).all()) and g[0][::2].tolist() == [1.0, -2.0]
        assert g[0][1].isnan() if math.isnan(bad) else float(g[0][1]) == bad
        # with a bound, however large, the norm's factor is everyone's
        ops.sgd_step(w, g, 0.5, max_norm=3e38, out=out)
        if math.isnan(bad):
            assert all(bool(t.isnan().all()) for t in out)
        else:
            assert torch.equal(out[1], w[1]) and out[0][1].isnan()


def test_gradients_of_nothing():
    empty = torch.zeros(0, 3, device=DEV)
    assert float(ops.gradient_norm([empty])) == 0.0
    assert float(ops.clip_gradients([empty, empty], 1.0)) == 0.0
    assert float(ops.sgd_step([empty], [empty], 1.0)) == 0.0
    z = torch.zeros(5, device=DEV)
    assert float(ops.clip_gradients([z], 1.0)) == 0.0 and bool((z == 0).all())


def test_gradients_that_are_not_contiguous():
    """Read as they are, with the results elsewhere; written, they are refused."""
    g = _gen(8)
    grads = [_rand(g, 30, 7).t(), _rand(g, 1, 9).expand(4, 9), _rand(g, 20)[::2]]
    _change_check(grads, 0.5, [_rand(g, *t.shape) for t in grads], 0.1)
    R.within(ops.gradient_norm(grads), R.total_norm(grads), "norm")
    to = [torch.empty(t.shape, device=DEV) for t in grads]
    ops.clip_gradients(grads, 0.5, out=to)
    for t, w in zip(to, R.changed(grads, 0.5)):
        R.within(t, w, "out")
    with pytest.raises(ValueError, match="contiguous"):
        ops.clip_gradients(grads, 0.5)


def test_what_overlaps_is_refused():
    t = torch.ones(64, device=DEV)
    u = torch.ones(64, device=DEV)
    for call in (lambda: ops.clip_gradients([t, t], 1.0),
                 lambda: ops.clip_gradients([t[:40], t[30:]], 1.0),
                 lambda: ops.clip_gradients([t[:32], u[:32]], 1.0, out=[u[:32], t[:32]]),
                 lambda: ops.clip_gradients([t[:32]], 1.0, out=[t[1:33]]),
                 lambda: ops.sgd_step([t, t], [u, u], 1.0),
                 lambda: ops.sgd_step([t[:32]], [t[16:48]], 1.0),
                 lambda: ops.sgd_step([t[:16].view(BF)], [t[:32]], 1.0)):
        with pytest.raises(ValueError):
            call()
    assert bool((t == 1).all()) and bool((u == 1).all())
    # one gradient read twice, and one tensor that is its own weight
    assert abs(float(ops.gradient_norm([t, t])) - math.sqrt(128)) <= 1e-5
    ops.sgd_step([t], [t], 0.5)
    assert bool((t == 0.5).all())


def test_tensors_of_two_devices_are_refused():
    a, b = torch.ones(4, device=DEV), torch.ones(4)
    for call in (lambda: ops.gradient_norm([a, b]), lambda: ops.clip_gradients([a], 1.0, out=[b]),
                 lambda: ops.sgd_step([a], [b], 1.0), lambda: ops.sgd_step([b], [a], 1.0),
                 lambda: ops.rms_norm_forward(a, b), lambda: ops.rms_norm_forward(a, a, residual=b),
                 lambda: ops.gated_silu_forward(a, b),
                 lambda: ops.rotary_forward(a.view(1, 1, 1, 4), a.view(1, 1, 1, 4), b[:1].long(), a[:2])):
        with pytest.raises(ValueError):
            call()


def test_autograd_sees_the_writes():
    w = torch.ones(8, device=DEV, requires_grad=True)
    g = torch.ones(8, device=DEV)
    y = (w * w).sum()
    versions = w._version, g._version
    ops.sgd_step([w], [g], 0.5)
    ops.clip_gradients([g], 0.5)
    assert w._version > versions[0] and g._version > versions[1]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_inference_tensors():
    """They have no version to count, and are written like others."""
    with torch.inference_mode():
        w, g = torch.ones(8, device=DEV), torch.full((8,), 2.0, device=DEV)
        x = torch.randn(3, 8, device=DEV)
        ops.sgd_step([w], [g], 0.25)
        y, total = ops.rms_norm(x, w, residual=x)
        ops.gated_silu(y, total)
    v = torch.ones(8, device=DEV)
    version = v._version
    ops.sgd_step([w, v], [g, g], 0.25)
    assert bool((w == 0).all()) and bool((v == 0.5).all()) and v._version > version


# ---- more than 2^31 values ------------------------------------------------------------------

LAST = slice(-3, None)


def _large(rows, d, seed):
    """bf16 rows beyond 2^31 values, of which the first and last few differ from the others."""
    t = torch.zeros(rows, d, dtype=BF, device=DEV)
    g = _gen(seed)
    t[:3], t[LAST] = _rand(g, 3, d, dtype=BF), _rand(g, 3, d, dtype=BF)
    return t


def test_large_norms():
    rows, d = (1 << 31) // 2050 + 9, 2050
    x, w = _large(rows, d, 1), _rand(_gen(2), d)
    y, total, rstd = ops.rms_norm_forward(x, w, residual=x)
    dx, _, dw = ops.rms_norm_backward(x, total, w, rstd)
    want, sums = [], []
    for part in (slice(0, 3), LAST):
        n = R.norm(x[part], w, x[part], 1e-6, BF)
        for name, t in (("y", y), ("total", total), ("rstd", rstd)):
            R.within(t[part], n[name], name)
        b = R.norm_backward(x[part], total[part], w, 1e-6, None, BF)
        R.within(dx[part], b["dx"], "dx")
        sums.append(b["dweight"])
    assert not bool(y[3:-3].any()) and not bool(dx[3:-3].any())
    R.within(dw, tuple(a + b for a, b in zip(*sums)), "dw")
    del y, total, dx
    for dtype in (E4M3, I8):
        q, scales, _ = ops.rms_norm_quantized(x, w, dtype=dtype, block=128)
        for part in (slice(0, 3), LAST):
            n = R.quantized(x[part], w, None, 1e-6, dtype, 128)
            R.within(q[part].float(), n["q"], "q")
            R.within(scales[part], n["scales"], "scales")
        assert bool((scales[3:-3] == 2.0**-126).all())


@pytest.mark.parametrize("rows", [1, (1 << 31) // 2049 + 7])
def test_large_activations(rows):
    d = 2049 if rows > 1 else (1 << 30) - 1  # (one row is as long as it may be)
    x = _large(max(rows, 6), d, 3) if rows > 1 else torch.zeros(1, d, dtype=BF, device=DEV)
    if rows == 1:
        x[0, -5:] = 1.5
    out = ops.gated_silu_forward(x, x)
    dg, du = ops.gated_silu_backward(x, x, x)
    for part in ((slice(0, 3), LAST) if rows > 1 else ((0, slice(-9, None)),)):
        want = R.gated(x[part], x[part], x[part])
        for name, t in (("out", out), ("dgate", dg), ("dup", du)):
            R.within(t[part], want[name], name)


def test_large_turns():
    b, h, n, d = 2, 9, 1 << 20, 128
    q = torch.zeros(b, n, h, d, dtype=BF, device=DEV).transpose(1, 2)
    g = _gen(4)
    q[:, :, :2], q[:, :, LAST] = _rand(g, b, h, 2, d), _rand(g, b, h, 3, d)
    f, at = R.by_frequency(d).to(DEV), torch.arange(n, device=DEV)
    got = ops.rotary_forward(q, q[:, :1], at, f)
    for part in (slice(0, 2), LAST):
        for t, x in zip(got, (q, q[:, :1])):
            want = R.rotary(x[:, :, part], at[part].expand(1, b, -1), f, (d // 2,), False, False)
            R.within(t[:, :, part], want, "turned")


def test_large_gradients():
    """A tensor of more than 2^31 values in front of a small one."""
    n = (1 << 31) + 12345
    big, small = torch.zeros(n, dtype=BF, device=DEV), _rand(_gen(5), 1000)
    big[:3], big[-3:] = 2.0, -4.0
    w = torch.zeros(n, dtype=BF, device=DEV)
    ends = torch.cat([big[:3], big[-3:]])
    norm, bound = R.total_norm([ends, small])
    R.within(ops.gradient_norm([big, small]), (norm, bound), "norm")
    ops.sgd_step([w, torch.zeros_like(small)], [big, small], 0.5, max_norm=1.0)
    want = R.changed([ends, small], 1.0, [torch.zeros_like(ends), torch.zeros_like(small)], 0.5)
    R.within(torch.cat([w[:3], w[-3:]]), want[0], "w")
    assert not bool(w[3:-3].any())


# ---- streams, repetition and graphs ---------------------------------------------------------

def _pass(x, w, res, dy, q, k, at, f, gate, up, grads, weights, out):
    """Every call once: a list of what came of it."""
    y, total, rstd = ops.rms_norm_forward(x, w, residual=res)
    back = ops.rms_norm_backward(dy, total, w, rstd, dtotal=res, x_dtype=BF)
    eight = ops.rms_norm_quantized(x, w, residual=res, block=128)
    turned = ops.rotary_forward(q, k, at, f)
    leaf = [t.detach().requires_grad_() for t in (gate, up)]
    act = ops.gated_silu(*leaf)
    dact = torch.autograd.grad(act, leaf, torch.ones_like(act))
    norm = ops.clip_gradients(grads, 0.5, out=out[0])
    step = ops.sgd_step(weights, grads, 0.1, max_norm=0.7, out=out[1])
    return [y, total, *back, eight[0].float(), *eight[1:], *turned, act.detach(), *dact, norm, step,
            ops.gradient_norm(grads), *(t.clone() for t in out[0] + out[1])]


def _pass_inputs(seed):
    g = _gen(seed)
    rows, d = 600, 1000
    grads, weights = _gradients(seed), _gradients(seed + 1, types=(F32,))
    return {"x": _rand(g, rows, d, dtype=BF), "w": _rand(g, d), "res": _rand(g, rows, d),
            "dy": _rand(g, rows, d, dtype=BF), "q": _rand(g, 2, 6, 100, 64, dtype=BF),
            "k": _rand(g, 2, 2, 100, 64, dtype=BF), "at": torch.arange(100, device=DEV),
            "f": R.by_frequency(64).to(DEV), "gate": _rand(g, 50, 1537, dtype=BF),
            "up": _rand(g, 50, 1537, dtype=BF), "grads": grads, "weights": weights,
            "out": ([torch.empty_like(t) for t in grads], [torch.empty_like(t) for t in weights])}


def test_the_same_bits_on_any_stream():
    s = _pass_inputs(20)
    want = _pass(**s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(side):
            got = _pass(**s)
        torch.cuda.current_stream().wait_stream(side)
        for i, (a, b) in enumerate(zip(got, want)):
            assert torch.equal(a, b), i


def test_two_passes_at_once():
    """Each call has scratch of its own."""
    inputs = [_pass_inputs(30), _pass_inputs(40)]
    want = [_pass(**s) for s in inputs]
    streams = [torch.cuda.Stream() for _ in inputs]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(4):
        got = []
        for st, s in zip(streams, inputs):
            with torch.cuda.stream(st):
                got.append(_pass(**s))
    for st in streams:
        torch.cuda.current_stream().wait_stream(st)
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_captured_passes():
    """Two graphs of the same calls, replayed in turn on new inputs, each replay against the eager
    calls; nothing in them is a memset."""
    from test_operators_capture_gpu import MEMSET, _kinds
    states = [_pass_inputs(50), _pass_inputs(60)]
    graphs, held = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in states:
            _pass(**s)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for s in states:
        graph = torch.cuda.CUDAGraph(keep_graph=True)
        with torch.cuda.graph(graph):
            held.append(_pass(**s))
        assert MEMSET not in _kinds(graph)
        graph.instantiate()
        graphs.append(graph)
    for turn in range(3):
        for i, s in enumerate(states):
            fresh = _pass_inputs(100 + 10 * turn + i)
            for name, t in s.items():
                if isinstance(t, torch.Tensor):
                    t.copy_(fresh[name])
                elif name != "out":
                    for a, b in zip(t, fresh[name]):
                        a.copy_(b)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for i, s in enumerate(states):
            got = [t.clone() for t in held[i]]
            for j, (a, b) in enumerate(zip(got, _pass(**s))):
                assert torch.equal(a, b), (turn, i, j)
