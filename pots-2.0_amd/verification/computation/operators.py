"""The operators of a training pass that nobody audits: attention, the loss over a vocabulary
and the embedding, each with its gradient.

A captured step (``verification.prover``) keeps every product of the inventory, the attention
probabilities and the logits among them, because a verifier will ask for them. A step that
leaves no transcript (a warm-up, a held-out loss, the steps between audits) need not write
either to memory. These calls run such a pass on the same model, with the kernels of
``libpots_mi355x`` (``pots_attention_*``, ``pots_vocab_loss_*``, ``pots_embedding_*``):

- :func:`attention`, :func:`vocab_loss` and :func:`embedding` are differentiable;
- the ``*_forward`` and ``*_backward`` functions under them are the kernels' own calls, for
  programs that keep their own tape or only evaluate.

Tensors are on the GPU, in fp32 or bf16; sums, softmax statistics and losses are fp32. Calls
enqueue on the current stream and never wait for the GPU; outputs and scratch come from torch's
allocator on that stream, so a tensor made on another stream needs the usual
``wait_stream``. Results are the same bits on every run. Wrong shapes, types, sizes and devices raise
``ValueError``; ids and targets are not read on the host, so those outside the vocabulary show
in the result instead (NaN; a negative target is a row without a loss).
``verification.computation.instances.decoder.DecoderComputation.uncaptured_loss`` runs all three.

A differentiable call saves its inputs by reference. A backward pass that is captured into a
graph wants leaves that no other live tape has used on another stream, as with any torch
function.
"""

from __future__ import annotations

import math
import struct

import torch

from verification.commitment import native

__all__ = ["attention", "attention_forward", "attention_backward", "vocab_loss",
           "vocab_loss_forward", "vocab_loss_backward", "embedding", "embedding_forward",
           "embedding_backward", "MAX_HEAD_DIM"]

MAX_HEAD_DIM = 128

_DTYPES = {torch.float32: 0, torch.bfloat16: 1}
# pots_attention, pots_vocab_loss and pots_embedding (include/pots_mi355x.h)
_ATTENTION = struct.Struct("<32q2q7If")
_LOSS = struct.Struct("<12q4I")
_EMBEDDING = struct.Struct("<5q5If")
_NO_HEADS = (0, 0, 0, 0)
_MOST, _LEAST = torch.finfo(torch.float32).max, 2.0**-149  # of fp32, above zero


def _dtype(t: torch.Tensor, what: str) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"{what} must be float32 or bfloat16, not {t.dtype}")
    return code


def _on_gpu(t: torch.Tensor) -> None:
    if not t.is_cuda:
        raise ValueError("the operators run on the GPU: their tensors must be there")


def _like(t: torch.Tensor, ref: torch.Tensor, shape: tuple[int, ...], what: str) -> None:
    if t.shape != shape:
        raise ValueError(f"{what} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.dtype != ref.dtype or t.device != ref.device:
        raise ValueError(f"{what} must be {ref.dtype} on {ref.device}, not {t.dtype} on "
                         f"{t.device}")


def _floats(t: torch.Tensor, device: torch.device, shape: tuple[int, ...],
            what: str) -> torch.Tensor:
    if t.dtype != torch.float32 or t.device != device or t.shape != shape:
        raise ValueError(f"{what} must be float32 {tuple(shape)} on {device}")
    return t.contiguous()


def _packed(block: struct.Struct, *values) -> bytes:
    """An argument block. A size past its 32 bits is a size out of range like any other."""
    try:
        return block.pack(*values)
    except struct.error as e:
        raise ValueError(f"a size is out of range: {e}") from None


def _indices(t: torch.Tensor, device: torch.device, what: str) -> torch.Tensor:
    if t.dtype not in (torch.int64, torch.int32) or t.device != device:
        raise ValueError(f"{what} must be int64 or int32 on {device}")
    if t.dtype != torch.int64:
        t = t.to(torch.int64)
    return t if t.is_contiguous() else t.contiguous()


# ---- attention ------------------------------------------------------------------------------

def _laid_out(t: torch.Tensor, d: int) -> torch.Tensor:
    """``t`` as the kernels take it, its heads ``d`` wide (columns of zeros past its own): itself
    where its values follow each other and its positions lie on 16-byte borders, else a copy."""
    sb, sh, sn, sd = t.stride()
    own = t.shape[3]
    if (own == d and sd == 1 and sn < 1 << 22 and t.data_ptr() % 16 == 0
            and (sb | sh | sn) * t.element_size() % 16 == 0):
        return t
    b, h, n, _ = t.shape
    out = _new_heads(b, h, n, d, t)
    out[..., :own] = t
    if own < d:
        out[..., own:] = 0
    return out


def _heads(t: torch.Tensor) -> tuple[int, int, int, int]:
    sb, sh, sn, sd = t.stride()
    if sd != 1:
        raise ValueError("a position's values must follow each other")
    return t.data_ptr(), sb, sh, sn


def _call_attention(name: str, tensors: tuple[torch.Tensor, ...], d: int, pack) -> None:
    """Enqueue on the tensors as they lie, which the library accepts almost always and checks
    itself; where it does not, on copies."""
    lib, device = native.get(), tensors[0].device
    if tensors[0].shape[3] == d:
        try:
            return lib.operator(name, pack(*tensors), device)
        except ValueError:
            laid = [_laid_out(t, d) for t in tensors]
            if all(a is b for a, b in zip(laid, tensors)):
                raise
    else:
        laid = [_laid_out(t, d) for t in tensors]
    lib.operator(name, pack(*laid), device)


def _attention_args(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                    lengths: torch.Tensor | None, scale: float | None
                    ) -> tuple[int, torch.Tensor | None, float]:
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError("q, k and v must be [batch, heads, n, head_dim]")
    b, h, n, d = q.shape
    kv = k.shape[1]
    code = _dtype(q, "q")
    if kv < 1 or h < 1 or h % kv:
        raise ValueError(f"{h} query heads are not a multiple of {kv} key heads")
    if not 1 <= d <= MAX_HEAD_DIM:
        raise ValueError(f"head_dim must be in [1, {MAX_HEAD_DIM}], got {d}")
    _like(k, q, (b, kv, n, d), "k")
    _like(v, q, (b, kv, n, d), "v")
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    elif not _LEAST <= scale <= _MOST:
        raise ValueError(f"scale must be positive and finite in fp32, got {scale}")
    if lengths is not None:
        if lengths.dtype != torch.int32 or lengths.shape != (b,) or lengths.device != q.device:
            raise ValueError(f"lengths must be int32 [{b}] on {q.device}")
        lengths = lengths.contiguous()
    return code, lengths, scale


def _new_heads(b: int, h: int, n: int, d: int, ref: torch.Tensor) -> torch.Tensor:
    """``[b, h, n, d]`` over memory of ``[b, n, h, d]``: a position's heads beside each other,
    as the projections around attention read and write them."""
    return torch.empty_strided((b, h, n, d), (n * h * d, d, h * d, 1), dtype=ref.dtype,
                               device=ref.device)


def attention_forward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
                      causal: bool = True, lengths: torch.Tensor | None = None,
                      scale: float | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Softmax attention of each sequence over its own keys: ``q [b, h, n, d]``, ``k`` and ``v
    [b, kv, n, d]`` with ``h`` a multiple of ``kv`` (consecutive query heads share a key head),
    any strides (a tensor whose positions do not start on 16-byte borders is copied first, and so
    is one whose ``d`` is no multiple of 8), ``d`` up to 128; ``scale`` is ``1/√d`` unless given.
    ``causal``: position i sees the positions up to i. ``lengths`` (int32 ``[b]``): positions
    from a sequence's length on are neither read nor seen; their outputs are zero.

    Returns ``(out [b, h, n, d], lse fp32 [b, h, n])``, ``lse`` the logarithm of each row's sum
    of exponentials (−inf for a row that sees nothing), which the backward pass takes. ``out`` lies
    in memory as ``[b, n, h, d]``."""
    code, lengths, scale = _attention_args(q, k, v, lengths, scale)
    _on_gpu(q)
    b, h, n, own = q.shape
    d = (own + 7) & ~7
    out = _new_heads(b, h, n, d, q)
    lse = torch.empty(b, h, n, dtype=torch.float32, device=q.device)

    def pack(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> bytes:
        return _packed(_ATTENTION, *_heads(q), *_heads(k), *_heads(v), *_heads(out), *_NO_HEADS,
                       *_NO_HEADS, *_NO_HEADS, *_NO_HEADS, lse.data_ptr(),
                       0 if lengths is None else lengths.data_ptr(), b, h, k.shape[1], n, d, code,
                       causal, scale)

    _call_attention("attention_forward", (q, k, v), d, pack)
    return out if d == own else out[..., :own], lse


def attention_backward(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                       out: torch.Tensor, lse: torch.Tensor, *, causal: bool = True,
                       lengths: torch.Tensor | None = None, scale: float | None = None
                       ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(dq, dk, dv)`` of :func:`attention_forward` at ``(q, k, v)`` with its ``out`` and
    ``lse``, in the inputs' type, lying in memory as ``[b, n, heads, d]``. The probabilities are
    recomputed; ``dk`` and ``dv`` are summed in fp32 over the query heads that share them."""
    code, lengths, scale = _attention_args(q, k, v, lengths, scale)
    b, h, n, own = q.shape
    kv = k.shape[1]
    _like(dout, q, q.shape, "dout")
    _like(out, q, q.shape, "out")
    lse = _floats(lse, q.device, (b, h, n), "lse")
    _on_gpu(q)
    d = (own + 7) & ~7
    dq = _new_heads(b, h, n, d, q)
    dk = _new_heads(b, kv, n, d, q)
    dv = _new_heads(b, kv, n, d, q)

    def pack(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
             dout: torch.Tensor) -> bytes:
        return _packed(_ATTENTION, *_heads(q), *_heads(k), *_heads(v), *_heads(out),
                       *_heads(dout), *_heads(dq), *_heads(dk), *_heads(dv), lse.data_ptr(),
                       0 if lengths is None else lengths.data_ptr(), b, h, kv, n, d, code, causal,
                       scale)

    _call_attention("attention_backward", (q, k, v, out, dout), d, pack)
    if d != own:
        return dq[..., :own], dk[..., :own], dv[..., :own]
    return dq, dk, dv


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, causal, lengths, scale):
        out, lse = attention_forward(q, k, v, causal=causal, lengths=lengths, scale=scale)
        ctx.save_for_backward(q, k, v, out, lse, lengths)
        ctx.causal, ctx.scale = causal, scale
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        q, k, v, out, lse, lengths = ctx.saved_tensors
        dq, dk, dv = attention_backward(g, q, k, v, out, lse, causal=ctx.causal,
                                        lengths=lengths, scale=ctx.scale)
        return dq, dk, dv, None, None, None


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, causal: bool = True,
              lengths: torch.Tensor | None = None, scale: float | None = None) -> torch.Tensor:
    """:func:`attention_forward`'s output, differentiable in ``q``, ``k`` and ``v``."""
    return _Attention.apply(q, k, v, causal, lengths, scale)


# ---- the loss over a vocabulary -------------------------------------------------------------

def _matrix(t: torch.Tensor) -> torch.Tensor:
    """Rows of consecutive values, each row its own."""
    return t if t.stride(1) == 1 and t.stride(0) >= t.shape[1] else t.contiguous()


def _loss_args(x: torch.Tensor, w: torch.Tensor, targets: torch.Tensor
               ) -> tuple[int, torch.Tensor]:
    if x.dim() != 2 or w.dim() != 2:
        raise ValueError("x must be [rows, dim] and w [vocab, dim]")
    code = _dtype(x, "x")
    if w.shape[0] < 1 or w.shape[1] < 1:
        raise ValueError("w must hold at least one row of at least one value")
    _like(x, w, (x.shape[0], w.shape[1]), "x")
    targets = _indices(targets, x.device, "targets")
    if targets.shape != (x.shape[0],):
        raise ValueError(f"targets must be [{x.shape[0]}], one for each row of x")
    _on_gpu(x)
    return code, targets


def vocab_loss_forward(x: torch.Tensor, w: torch.Tensor, targets: torch.Tensor
                       ) -> tuple[torch.Tensor, torch.Tensor]:
    """Softmax cross entropy of the rows of ``x [rows, dim]`` against a vocabulary matrix
    ``w [vocab, dim]`` of the same type, without its logits: ``(loss, lse)``, fp32 ``[rows]``,
    ``loss_r = lse_r − x_r·w_{t_r}``. A negative target is a row without a loss (0); one past the
    vocabulary gives NaN."""
    code, targets = _loss_args(x, w, targets)
    rows, dim = x.shape
    x, w = _matrix(x), _matrix(w)
    loss = torch.empty(rows, dtype=torch.float32, device=x.device)
    lse = torch.empty(rows, dtype=torch.float32, device=x.device)
    args = _packed(_LOSS, x.data_ptr(), w.data_ptr(), targets.data_ptr(), loss.data_ptr(),
                   lse.data_ptr(), 0, 0, 0, x.stride(0), w.stride(0), 0, 0, rows, dim, w.shape[0],
                   code)
    native.get().operator("vocab_loss_forward", args, x.device)
    return loss, lse


def vocab_loss_backward(weights: torch.Tensor, x: torch.Tensor, w: torch.Tensor,
                        targets: torch.Tensor, lse: torch.Tensor
                        ) -> tuple[torch.Tensor, torch.Tensor]:
    """``(dx, dw)`` of ``Σ_r weights_r · loss_r`` (``weights`` fp32 ``[rows]``) in the inputs'
    type. Rows of weight zero and rows without a target are left out of the products."""
    code, targets = _loss_args(x, w, targets)
    rows, dim = x.shape
    weights = _floats(weights, x.device, (rows,), "weights")
    lse = _floats(lse, x.device, (rows,), "lse")
    x, w = _matrix(x), _matrix(w)
    dx = torch.empty(rows, dim, dtype=x.dtype, device=x.device)
    dw = torch.empty(w.shape[0], dim, dtype=x.dtype, device=x.device)
    args = _packed(_LOSS, x.data_ptr(), w.data_ptr(), targets.data_ptr(), 0, lse.data_ptr(),
                   weights.data_ptr(), dx.data_ptr(), dw.data_ptr(), x.stride(0), w.stride(0),
                   dim, dim, rows, dim, w.shape[0], code)
    native.get().operator("vocab_loss_backward", args, x.device)
    return dx, dw


def _sum(t: torch.Tensor) -> torch.Tensor:
    """The sum of a vector. torch's sum of many values clears its counters by a memset, which has no
    place in a captured graph (recorded at 2^20 values, not at 2^16): such a vector is summed by
    rows of 4096 first."""
    if t.numel() > 1 << 16:
        t = torch.nn.functional.pad(t, (0, -t.numel() % 4096)).view(-1, 4096).sum(1)
    return t.sum()


class _VocabLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, targets, weights):
        loss, lse = vocab_loss_forward(x, w, targets)
        ctx.save_for_backward(x, w, targets, weights, lse,
                              loss if ctx.needs_input_grad[3] else None)
        return _sum(torch.where(weights != 0, loss * weights, 0.0))

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        x, w, targets, weights, lse, loss = ctx.saved_tensors
        dx = dw = dweights = None
        if ctx.needs_input_grad[0] or ctx.needs_input_grad[1]:
            dx, dw = vocab_loss_backward(weights * g, x, w, targets, lse)
        if ctx.needs_input_grad[3]:
            dweights = torch.where((weights != 0) | loss.isfinite(), loss * g, 0.0)
        return dx, dw, None, dweights


def vocab_loss(x: torch.Tensor, w: torch.Tensor, targets: torch.Tensor,
               weights: torch.Tensor) -> torch.Tensor:
    """``Σ_r weights_r · loss_r`` of :func:`vocab_loss_forward`'s losses, fp32, differentiable
    in ``x``, ``w`` and ``weights``; rows of weight zero count for nothing, whatever their loss (the
    gradient of such a weight is the row's loss, or zero where that is not finite)."""
    if x.dim() != 2:
        raise ValueError("x must be [rows, dim]")
    weights = _floats(weights, x.device, (x.shape[0],), "weights")
    return _VocabLoss.apply(x, w, targets, weights)


# ---- the embedding --------------------------------------------------------------------------

def _check_scale(scale: float) -> None:
    if not -_MOST <= scale <= _MOST:
        raise ValueError(f"scale must be finite in fp32, got {scale}")


def embedding_forward(ids: torch.Tensor, table: torch.Tensor, *, scale: float = 1.0
                      ) -> torch.Tensor:
    """``scale · table[ids]``: rows of ``table [vocab, dim]`` for ids of any shape, in the
    table's type; an id outside the table gives a row of NaN."""
    if table.dim() != 2 or table.shape[0] < 1 or table.shape[1] < 1:
        raise ValueError("table must be [vocab, dim], neither of them 0")
    code = _dtype(table, "table")
    _check_scale(scale)
    ids = _indices(ids, table.device, "ids")
    _on_gpu(table)
    table = _matrix(table)
    out = torch.empty(*ids.shape, table.shape[1], dtype=table.dtype, device=table.device)
    args = _packed(_EMBEDDING, ids.data_ptr(), table.data_ptr(), out.data_ptr(),
                   table.stride(0), table.shape[1], ids.numel(), table.shape[1], table.shape[0],
                   code, 0, scale)
    native.get().operator("embedding_forward", args, table.device)
    return out


def embedding_backward(ids: torch.Tensor, dout: torch.Tensor, vocab: int, *,
                       scale: float = 1.0, add_to: torch.Tensor | None = None) -> torch.Tensor:
    """The table's gradient ``[vocab, dim]``: row v is ``scale`` times the sum in fp32 of
    ``dout``'s rows whose id is v, added up in runs of consecutive positions and the runs in order
    (whose length is the call's: a dense and an added gradient of the same tokens may differ in their
    last bits). With ``add_to`` (a gradient the table already has) it is added there, touching only
    the rows that occur, and that tensor is returned. Ids outside the table add to nothing."""
    code = _dtype(dout, "dout")
    _check_scale(scale)
    ids = _indices(ids, dout.device, "ids")
    dim = dout.shape[-1] if dout.dim() else 0
    if dim < 1 or dout.shape[:-1] != ids.shape:
        raise ValueError(f"dout must be {tuple(ids.shape)} rows, got {tuple(dout.shape)}")
    if not 1 <= vocab <= 1 << 30:
        raise ValueError(f"vocab must be in [1, 2^30], got {vocab}")
    if add_to is not None:
        _like(add_to, dout, (vocab, dim), "add_to")
        if dim > 1 and add_to.stride(1) != 1 or vocab > 1 and add_to.stride(0) < dim:
            raise ValueError("add_to must have rows of consecutive values, each its own")
    _on_gpu(dout)
    rows = _matrix(dout.reshape(-1, dim))
    table = add_to
    if table is None:
        table = torch.empty(vocab, dim, dtype=dout.dtype, device=dout.device)
    args = _packed(_EMBEDDING, ids.data_ptr(), table.data_ptr(), rows.data_ptr(),
                   table.stride(0), rows.stride(0), ids.numel(), dim, vocab, code,
                   add_to is not None, scale)
    native.get().operator("embedding_backward", args, dout.device)
    return table


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, table, scale):
        ctx.save_for_backward(ids)
        ctx.vocab, ctx.scale = table.shape[0], scale
        return embedding_forward(ids, table, scale=scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        ids, = ctx.saved_tensors
        return None, embedding_backward(ids, g, ctx.vocab, scale=ctx.scale), None


def embedding(ids: torch.Tensor, table: torch.Tensor, *, scale: float = 1.0) -> torch.Tensor:
    """:func:`embedding_forward`, differentiable in ``table``."""
    return _Embedding.apply(ids, table, scale)
