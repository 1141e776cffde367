"""The operators' formulas in 64 bits, with bounds on how far a computation that rounds its
operands to the inputs' type and sums in fp32 may be from them.

A rounding is off by at most half a step: ``U[dtype]`` relative (2^-8 bf16, 2^-24 fp32). A sum
of n fp32 terms is off by at most n half steps of the sum of their sizes. ``2^x`` of the hardware
is taken as four half steps, and its argument carries half a step of its own size."""

from __future__ import annotations

import math

import torch

E32 = 2.0**-24
U = {torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}
DEV = "cuda"


def attention(q, k, v, dout, *, causal, lengths=None, scale=None):
    """``{name: (value, bound)}`` of out, lse, dq, dk and dv."""
    u = U[q.dtype]
    q, k, v, g = (t.double().cpu() for t in (q, k, v, dout))
    b, h, n, d = q.shape
    kv = k.shape[1]
    rep = h // kv
    scale = 1 / math.sqrt(d) if scale is None else scale
    val = {x: torch.zeros_like(t) for x, t in (("out", q), ("dq", q), ("dk", k), ("dv", v))}
    bnd = {x: torch.zeros_like(t) for x, t in val.items()}
    val["lse"] = torch.full((b, h, n), -math.inf, dtype=torch.float64)
    bnd["lse"] = torch.zeros(b, h, n, dtype=torch.float64)
    for i in range(b):
        m = n if lengths is None else max(0, min(n, int(lengths[i])))
        if m == 0:
            continue
        hide = torch.ones(m, m, dtype=torch.bool).triu_(1) if causal else \
            torch.zeros(m, m, dtype=torch.bool)
        for j in range(h):
            c = j // rep
            Q, K, V, G = q[i, j, :m], k[i, c, :m], v[i, c, :m], g[i, j, :m]
            s = (Q @ K.T * scale).masked_fill(hide, -math.inf)
            size = (Q.abs() @ K.abs().T * scale).masked_fill(hide, 0)
            es = ((d + 4) * E32 * size).amax(1, keepdim=True)
            lse = s.logsumexp(1, keepdim=True)
            big = size.amax(1, keepdim=True) + lse.abs()
            rp = 2 * es + (m + 8 + 8 * big) * E32  # of a probability, relative
            p = (s - lse).exp()
            o = p @ V
            n32 = (m + 8) * E32
            val["lse"][i, j, :m] = lse[:, 0]
            bnd["lse"][i, j, :m] = (es + (m + 8 + 8 * big) * E32)[:, 0]
            val["out"][i, j, :m] = o
            bo = (rp + u + n32) * (p @ V.abs()) + u * o.abs()
            bnd["out"][i, j, :m] = bo
            dv = p.T @ G
            val["dv"][i, c, :m] += dv
            bnd["dv"][i, c, :m] += (p * (rp + u + rep * n32)).T @ G.abs() + u * dv.abs()
            dp = G @ V.T
            D = (G * o).sum(1, keepdim=True)
            eD = (G.abs() * bo).sum(1, keepdim=True) + \
                (d + 4) * E32 * (G.abs() * o.abs()).sum(1, keepdim=True)
            edp = (d + 4) * E32 * (G.abs() @ V.abs().T)
            ds = p * (dp - D)
            eds = p * (rp * (dp.abs() + D.abs()) + edp + eD + 4 * E32 * (dp.abs() + D.abs()))
            eds = eds + (u + rep * n32) * (ds.abs() + eds)
            dq, dk = ds @ K * scale, ds.T @ Q * scale
            val["dq"][i, j, :m] = dq
            bnd["dq"][i, j, :m] = (eds @ K.abs()) * scale + 2 * u * dq.abs()
            val["dk"][i, c, :m] += dk
            bnd["dk"][i, c, :m] += (eds.T @ Q.abs()) * scale + 2 * u * dk.abs()
    return {x: (val[x], bnd[x]) for x in val}


def vocab_loss(x, w, targets, weights):
    """``{name: (value, bound)}`` of loss, lse, dx and dw; targets within the vocabulary or
    negative."""
    u = U[x.dtype]
    x, w, t, wt = x.double().cpu(), w.double().cpu(), targets.cpu(), weights.double().cpu()
    rows, d = x.shape
    vocab = w.shape[0]
    has = t >= 0
    s = x @ w.T
    size = x.abs() @ w.abs().T
    es = ((d + 16) * E32 * size).amax(1, keepdim=True) if rows else torch.zeros(0, 1)
    lse = s.logsumexp(1, keepdim=True)
    big = size.amax(1, keepdim=True) + lse.abs() if rows else torch.zeros(0, 1)
    el = es + (vocab // 32 + 64 + 8 * big) * E32
    st = s.gather(1, t.clamp(min=0)[:, None])
    loss = torch.where(has[:, None], lse - st, 0.0)[:, 0]
    p = (s - lse).exp()
    one = torch.zeros_like(p)
    one[has, t[has]] = 1
    weight = torch.where(has, wt, 0.0)[:, None]
    g = weight * (p - one)
    eg = weight.abs() * (p * (es + el + 8 * E32) + 4 * E32 * one) + u * g.abs()
    dx, dw = g @ w, g.T @ x
    bx = (eg + (vocab + 16) * E32 * g.abs()) @ w.abs() + u * dx.abs()
    bw = (eg + (rows + 16) * E32 * g.abs()).T @ x.abs() + u * dw.abs()
    return {"loss": (loss, (es + el)[:, 0] * 1.0), "lse": (lse[:, 0], el[:, 0]),
            "dx": (dx, bx), "dw": (dw, bw)}


def embedding(ids, dout, vocab, scale, add_to=None):
    """The table's gradient and its bound."""
    u = U[dout.dtype]
    ids, g = ids.cpu().reshape(-1), dout.double().cpu().reshape(-1, dout.shape[-1])
    ok = (ids >= 0) & (ids < vocab)
    val = torch.zeros(vocab, g.shape[1], dtype=torch.float64).index_add_(0, ids[ok], g[ok])
    size = torch.zeros_like(val).index_add_(0, ids[ok], g[ok].abs())
    count = torch.zeros(vocab, dtype=torch.float64).index_add_(
        0, ids[ok], torch.ones(int(ok.sum()), dtype=torch.float64))
    val, bound = val * scale, (count[:, None] + 3) * E32 * size * abs(scale)
    if add_to is not None:
        val = val + add_to.double().cpu()
    return val, bound + u * val.abs()


def within(got: torch.Tensor, want: tuple[torch.Tensor, torch.Tensor], what: str) -> None:
    value, bound = want
    got = got.double().cpu()
    assert got.shape == value.shape, what
    same = (got == value) | (got.isnan() & value.isnan())
    # the smallest normal number of either type: what lies below it may be taken as zero
    off = torch.where(same, 0.0, (got - value).abs() - bound - 2.0**-126)
    assert bool((off <= 0).all()), (what, float(off.max()), float(bound.flatten()[off.argmax()]),
                                    int((~(off <= 0)).sum()))
