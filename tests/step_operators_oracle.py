"""The formulas of what a step does between its products and after them, in 64 bits, with bounds on
how far a computation that works in fp32 and rounds its results once may be from them.

A rounding is off by at most half a step: ``U[dtype]`` relative. A sum of n fp32 terms is off by at
most n half steps of the sum of their sizes, in whatever order. The device's exponential is taken as
two half steps; its sine and cosine of less than an eighth of a turn as two of one, 2^-24 each."""

from __future__ import annotations


import torch

E32 = 2.0**-24
U = {torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}


def added(x, residual):
    """The sum as the residual's type holds it, rounded to fp32 on the way: exact arithmetic, the
    same bits everywhere."""
    if residual is None:
        return x.cpu()
    return (x.cpu().float() + residual.cpu().float()).to(residual.dtype)


def norm(x, weight, residual, eps, out_dtype):
    """``{name: (value, bound)}`` of y, the sum and rstd."""
    total = added(x, residual)
    t, w = total.double(), weight.double().cpu()
    d = t.shape[-1]
    e = (d + 12) * E32  # a mean of squares, its root and reciprocal, and three products
    rstd = (t.square().mean(-1) + eps).rsqrt()
    y = t * rstd[..., None] * w
    return {"y": (y, y.abs() * (e + U[out_dtype])), "total": (total.double(), torch.zeros_like(t)),
            "rstd": (rstd, rstd * e)}


def norm_backward(dy, total, weight, eps, dtotal, x_dtype):
    u = {"dx": U[x_dtype], "dresidual": U[total.dtype]}
    dy, t, w = dy.double().cpu(), total.double().cpu(), weight.double().cpu()
    d = t.shape[-1]
    rows = t[..., 0].numel()
    e = (d + 12) * E32
    s = (t.square().mean(-1, keepdim=True) + eps).rsqrt()
    h, g = t * s, dy * w
    mean = (g * h).mean(-1, keepdim=True)
    size = (g * h).abs().mean(-1, keepdim=True)
    dt = s * (g - h * mean)
    bound = s * (g.abs() + h.abs() * (mean.abs() + size)) * 2 * e
    if dtotal is not None:
        dt = dt + dtotal.double().cpu()
    bound = bound + 2 * E32 * dt.abs()
    dw = (dy * h).reshape(-1, d).sum(0)
    bw = (dy * h).abs().reshape(-1, d).sum(0) * (e + (rows + 8) * E32)
    out = {x: (dt, bound + v * dt.abs()) for x, v in u.items()}
    return {**out, "dweight": (dw, bw + U[weight.dtype] * dw.abs())}


def quantized(x, weight, residual, eps, dtype, block):
    """(value before its rounding to 8 bits, bound) of q, and of the scales."""
    y, _ = norm(x, weight, residual, eps, torch.float32)["y"]
    d = y.shape[-1]
    e = (d + 16) * E32
    block = block or d
    most = 448.0 if dtype == torch.float8_e4m3fn else 127.0
    groups = torch.nn.functional.pad(y, (0, -d % block)).unflatten(-1, (-1, block))
    scales = (groups.abs().amax(-1) / most).clamp(min=2.0**-126)
    v = (groups / scales[..., None]).flatten(-2)[..., :d]
    if dtype == torch.int8:
        half = torch.full_like(v, 0.5)
    else:  # half a step of three bits, from 2^-6 up; below it steps are 2^-9
        half = torch.maximum(v.abs() * 2.0**-4, torch.full_like(v, 2.0**-10))
    return {"q": (v, half + 2 * e * v.abs()), "scales": (scales, scales * e)}


def rotary(x, positions, frequencies, counts, adjacent, inverse):
    """x [b, heads, n, d], positions [axes, b, n]."""
    u = U[x.dtype]
    x, f = x.double().cpu(), frequencies.double().cpu()
    pairs = f.numel()
    axis = torch.repeat_interleave(torch.arange(len(counts)), torch.tensor(counts))
    angle = positions.cpu()[axis].permute(1, 2, 0)[:, None].double() * f
    off = 6 * E32 + angle.abs() * 2.0**-50
    c, s = angle.cos(), angle.sin() * (-1 if inverse else 1)
    a = slice(0, 2 * pairs, 2) if adjacent else slice(0, pairs)
    b = slice(1, 2 * pairs, 2) if adjacent else slice(pairs, 2 * pairs)
    p, q = x[..., a], x[..., b]
    val, bound = x.clone(), torch.zeros_like(x)
    val[..., a], val[..., b] = p * c - q * s, p * s + q * c
    size = (p.abs() + q.abs()) * off
    bound[..., a] = size + u * val[..., a].abs()
    bound[..., b] = size + u * val[..., b].abs()
    return val, bound


def gated(gate, up, dout=None):
    u = U[gate.dtype]
    g, v = gate.double().cpu(), up.double().cpu()
    s = torch.sigmoid(g)
    out = g * s * v
    res = {"out": (out, out.abs() * (10 * E32 + u))}
    if dout is not None:
        dy = dout.double().cpu()
        rest = torch.sigmoid(-g)
        dg, du = dy * v * s * (1 + g * rest), dy * g * s
        res["dgate"] = (dg, (dy * v).abs() * s * (1 + g.abs() * rest) * 16 * E32 + u * dg.abs())
        res["dup"] = (du, du.abs() * (12 * E32 + u))
    return res


def total_norm(gradients):
    value = torch.stack([g.double().cpu().square().sum() for g in gradients]).sum().sqrt()
    return value, value * 2 * E32


def changed(gradients, max_norm, weights=None, eta=1.0):
    """What :func:`operators.clip_gradients` or ``sgd_step`` writes, per tensor."""
    factor = min(1.0, max_norm / float(total_norm(gradients)[0]))
    out = []
    for i, g in enumerate(gradients):
        v = g.double().cpu() * factor * eta
        if weights is None:
            out.append((v, v.abs() * (2 * E32 + U[g.dtype])))
        else:
            w = weights[i]
            new = w.double().cpu() - v
            out.append((new, v.abs() * 3 * E32 + new.abs() * (E32 + U[w.dtype])))
    return out


def within(got, want, what):
    value, bound = want
    got = got.double().cpu()
    assert got.shape == value.shape, (what, got.shape, value.shape)
    same = (got == value) | (got.isnan() & value.isnan())
    # the smallest normal number: what lies below it may be taken as zero
    off = torch.where(same, 0.0, (got - value).abs() - bound - 2.0**-126)
    assert bool((off <= 0).all()), (what, float(off.max()), int((~(off <= 0)).sum()))


def difference(f, at, along, step=1e-5):
    """A scalar function's slope along a direction, by central differences in 64 bits."""
    return float((f(at + step * along) - f(at - step * along)) / (2 * step))


def by_frequency(width, base=10000.0):
    return base ** (-torch.arange(0, width, 2, dtype=torch.float64) / width)
