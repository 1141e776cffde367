"""The operators of a training step that nobody audits: attention, the loss over a vocabulary
and the embedding, each with its gradient; what lies between a layer's products (norms, rotary
positions, the gated activation); and the clipped update.

A captured step (``verification.prover``) keeps every product of the inventory, the attention
probabilities and the logits among them, because a verifier will ask for them. A step that
leaves no transcript (a warm-up, a held-out loss, the steps between audits) need not write
either to memory. These calls run such a pass on the same model, with the kernels of
``libpots_mi355x`` (``pots_attention_*``, ``pots_vocab_loss_*``, ``pots_embedding_*``,
``pots_rms_norm_*``, ``pots_rotary_turn``, ``pots_gated_silu_*``, ``pots_gradient_norm``,
``pots_clip_gradients``, ``pots_sgd_step``):

- :func:`attention`, :func:`vocab_loss`, :func:`embedding`, :func:`rms_norm`, :func:`rotary` and
  :func:`gated_silu` are differentiable;
- the ``*_forward`` and ``*_backward`` functions under them are the kernels' own calls, for
  programs that keep their own tape or only evaluate;
- :func:`rms_norm_quantized` gives a norm's output in 8 bits;
- :func:`gradient_norm`, :func:`clip_gradients` and :func:`sgd_step` take a model's whole gradient.

Tensors are on the GPU, in fp32 or bf16; sums, softmax statistics and losses are fp32. Calls
enqueue on the current stream and never wait for the GPU; outputs and scratch come from torch's
allocator on that stream, so a tensor made on another stream needs the usual
``wait_stream``. Results are the same bits on every run. Wrong shapes, types, sizes and devices raise
``ValueError``; ids and targets are not read on the host, so those outside the vocabulary show
in the result instead (NaN; a negative target is a row without a loss).
``verification.computation.instances.decoder.DecoderComputation.uncaptured_loss`` and
``verification.prover.step.uncaptured_step`` run them.

A differentiable call saves its inputs by reference. A backward pass that is captured into a
graph wants leaves that no other live tape has used on another stream, as with any torch
function.
"""

from __future__ import annotations

import itertools
import math
import operator
import struct
from collections.abc import Sequence

import torch

from verification.commitment import native

__all__ = ["attention", "attention_forward", "attention_backward", "vocab_loss",
           "vocab_loss_forward", "vocab_loss_backward", "embedding", "embedding_forward",
           "embedding_backward", "rms_norm", "rms_norm_forward", "rms_norm_backward",
           "rms_norm_quantized", "rotary", "rotary_forward", "rotary_backward",
           "rotary_frequencies", "gated_silu", "gated_silu_forward", "gated_silu_backward",
           "gradient_norm", "clip_gradients", "sgd_step", "MAX_HEAD_DIM", "MAX_NORM_DIM",
           "MAX_ROTARY_DIM"]

MAX_HEAD_DIM = 128
MAX_NORM_DIM = 1 << 14
MAX_ROTARY_DIM = 1024

_DTYPES = {torch.float32: 0, torch.bfloat16: 1}
_EIGHT_BITS = {torch.float8_e4m3fn: 2, torch.int8: 3}
_F64 = 4
# the argument blocks of include/pots_mi355x.h
_ATTENTION = struct.Struct("<32q2q7If")
_LOSS = struct.Struct("<12q4I")
_EMBEDDING = struct.Struct("<5q5If")
_NORM = struct.Struct("<17q7If")
_ROTARY = struct.Struct("<21q16I")
_GATED = struct.Struct("<9q3I4x")
_GRADIENTS = struct.Struct("<q2f2I")
_GRADIENT = struct.Struct("<3qQ2I")
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


# ---- the norm -------------------------------------------------------------------------------

def _rows(t: torch.Tensor) -> tuple[torch.Tensor, int]:
    """``[..., d]`` as rows of consecutive values, and how far apart they start."""
    if t.is_contiguous():
        return t, t.shape[-1]
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    if t.shape[1] > 1 and t.stride(1) != 1:
        t = t.contiguous()
    return t, t.stride(0)


# (torch.empty takes twice the host time of these)
def _new_like(t: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """A contiguous tensor of ``t``'s shape."""
    if t.is_contiguous():
        return torch.empty_like(t, dtype=dtype)
    return torch.empty(t.shape, dtype=dtype, device=t.device)


def _new_floats(shape: Sequence[int], *near: torch.Tensor | None) -> torch.Tensor:
    """An fp32 tensor on the device of ``near``."""
    for t in near:
        if t is not None and t.dtype == torch.float32:
            return t.new_empty(shape)
    return torch.empty(shape, dtype=torch.float32, device=near[0].device)


def _norm_args(x: torch.Tensor, weight: torch.Tensor, eps: float, what: str) -> int:
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_NORM_DIM:
        raise ValueError(f"{what} must be [..., dim] with dim in [1, {MAX_NORM_DIM}], got "
                         f"{tuple(x.shape)}")
    if weight.shape != x.shape[-1:] or weight.device != x.device:
        raise ValueError(f"weight must be [{x.shape[-1]}] on {x.device}")
    if not 2.0**-126 <= eps <= _MOST:
        raise ValueError(f"eps must be a normal positive number of fp32, got {eps}")
    return _dtype(weight, "weight")


def _summands(x: torch.Tensor, residual: torch.Tensor | None) -> None:
    _dtype(x, "x")
    if residual is None:
        return
    if residual.shape != x.shape or residual.device != x.device:
        raise ValueError(f"residual must be {tuple(x.shape)} on {x.device}")
    _dtype(residual, "residual")


def _run_norm(name: str, x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None,
              y: torch.Tensor, y_type: int, rstd: torch.Tensor | None,
              scales: torch.Tensor | None, block: int, eps: float) -> torch.Tensor:
    """The forward calls; the sum that was normed."""
    total, to, other, other_ptr, other_row = x, 0, None, 0, 0
    if residual is not None:
        total = _new_like(residual, residual.dtype)
        other, other_row = _rows(residual)
        to, other_ptr = total.data_ptr(), other.data_ptr()
    rows, row = _rows(x)
    own, dim = weight.contiguous(), x.shape[-1]
    args = _packed(_NORM, rows.data_ptr(), other_ptr, own.data_ptr(), to, y.data_ptr(),
                   0 if rstd is None else rstd.data_ptr(),
                   0 if scales is None else scales.data_ptr(), 0, 0, 0, 0, 0, row, other_row, 0, 0, 0,
                   x.numel() // dim, dim, block, _DTYPES[x.dtype], _DTYPES[total.dtype],
                   _DTYPES[weight.dtype], y_type, eps)
    native.get().operator(name, args, x.device)
    return total


def rms_norm_forward(x: torch.Tensor, weight: torch.Tensor, *, eps: float = 1e-6,
                     residual: torch.Tensor | None = None, out_dtype: torch.dtype | None = None
                     ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``y = t · s · weight`` over rows ``[..., dim]`` with ``t = x + residual`` and
    ``s = 1/√(mean t² + eps)``: ``(y, t, s)``. Each tensor has its own type, fp32 or bf16: ``t``
    the residual's (rounded to it once, and that is what is normed), ``y`` ``out_dtype``
    (``x``'s unless given), ``s`` fp32 ``[...]``. Without a residual ``t`` is ``x`` itself. Squares
    are added in fp32: a row whose 2-norm is 1.8e19 or more has an infinite sum, and comes out as zeros."""
    _norm_args(x, weight, eps, "x")
    _summands(x, residual)
    out_dtype = x.dtype if out_dtype is None else out_dtype
    if out_dtype not in _DTYPES:
        raise ValueError(f"out_dtype must be float32 or bfloat16, not {out_dtype}")
    _on_gpu(x)
    y = _new_like(x, out_dtype)
    rstd = _new_floats(x.shape[:-1], weight, residual)
    total = _run_norm("rms_norm_forward", x, weight, residual, y, _DTYPES[out_dtype], rstd, None, 0,
                      eps)
    return y, total, rstd


def rms_norm_quantized(x: torch.Tensor, weight: torch.Tensor, *, eps: float = 1e-6,
                       residual: torch.Tensor | None = None,
                       dtype: torch.dtype = torch.float8_e4m3fn, block: int | None = None
                       ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """:func:`rms_norm_forward`'s ``y`` in 8 bits, ``float8_e4m3fn`` or ``int8``: ``(q, scales,
    t)`` with ``y ≈ q · scale``, rounded to nearest from fp32. A scale (fp32 ``[..., blocks]``) is
    the largest size of a row (``block`` None), or of each ``block`` columns (32, 64, 128 or 256;
    the last may be fewer), over 448 or 127, and at least 2^-126. A block that holds a NaN has the
    scale NaN, and one that holds an infinity an infinite scale: there what is finite is 0. A ``y / scale``
    that is NaN (all of the first, the infinities of the second) is NaN in e4m3 and −128 in int8, whose
    numbers else are −127 to 127."""
    _norm_args(x, weight, eps, "x")
    _summands(x, residual)
    if dtype not in _EIGHT_BITS:
        raise ValueError(f"dtype must be float8_e4m3fn or int8, not {dtype}")
    if block not in (None, 32, 64, 128, 256):
        raise ValueError(f"block must be 32, 64, 128 or 256, or None for a row, not {block}")
    blocks = 1 if block is None else -(-x.shape[-1] // block)
    _on_gpu(x)
    q = _new_like(x, dtype)
    scales = _new_floats((*x.shape[:-1], blocks), weight, residual)
    total = _run_norm("rms_norm_quantized", x, weight, residual, q, _EIGHT_BITS[dtype], None,
                      scales, block or 0, eps)
    return q, scales, total


def rms_norm_backward(dy: torch.Tensor, total: torch.Tensor, weight: torch.Tensor,
                      rstd: torch.Tensor, *, dtotal: torch.Tensor | None = None,
                      x_dtype: torch.dtype | None = None
                      ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(dx, dresidual, dweight)`` of :func:`rms_norm_forward` with its ``t`` and ``s``, for the
    gradients ``dy`` of ``y`` and ``dtotal`` (of ``t``'s type, or None) of ``t``. ``x`` and the
    residual have the same gradient: ``dresidual`` in ``t``'s type, ``dx`` in ``x_dtype`` (``t``'s
    unless given; the same tensor where they are one type). ``dweight`` is summed in fp32 over all
    rows, in ``weight``'s type."""
    return _norm_backward(dy, total, weight, rstd, dtotal, x_dtype, True)


def _norm_backward(dy: torch.Tensor, total: torch.Tensor, weight: torch.Tensor, rstd: torch.Tensor,
                   dtotal: torch.Tensor | None, x_dtype: torch.dtype | None, of_weight: bool
                   ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
    """:func:`rms_norm_backward`, without ``dweight`` (None) unless ``of_weight``."""
    code = _norm_args(total, weight, 1.0, "total")
    _dtype(total, "total")
    if dy.shape != total.shape or dy.device != total.device:
        raise ValueError(f"dy must be {tuple(total.shape)} on {total.device}")
    dy_type = _dtype(dy, "dy")
    if dtotal is not None:
        _like(dtotal, total, total.shape, "dtotal")
    rstd = _floats(rstd, total.device, total.shape[:-1], "rstd")
    x_dtype = total.dtype if x_dtype is None else x_dtype
    if x_dtype not in _DTYPES:
        raise ValueError(f"x_dtype must be float32 or bfloat16, not {x_dtype}")
    _on_gpu(total)
    dresidual = dx = _new_like(total, total.dtype)
    if x_dtype != total.dtype:
        dx = _new_like(total, x_dtype)
    dweight = _new_like(weight, weight.dtype) if of_weight else None
    (g, g_row), (t, t_row), own = _rows(dy), _rows(total), weight.contiguous()
    other, other_ptr, other_row = None, 0, 0
    if dtotal is not None:
        other, other_row = _rows(dtotal)
        other_ptr = other.data_ptr()
    dim = total.shape[-1]
    args = _packed(_NORM, 0, 0, own.data_ptr(), t.data_ptr(), 0, rstd.data_ptr(), 0, g.data_ptr(),
                   other_ptr, 0 if dx is dresidual else dx.data_ptr(), dresidual.data_ptr(),
                   0 if dweight is None else dweight.data_ptr(), 0, 0, t_row, g_row, other_row, total.numel() // dim, dim, 0,
                   _DTYPES[x_dtype], _DTYPES[total.dtype], code, dy_type, 1.0)
    native.get().operator("rms_norm_backward", args, total.device)
    return dx, dresidual, dweight


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps, out_dtype):
        y, total, rstd = rms_norm_forward(x, weight, eps=eps, residual=residual,
                                          out_dtype=out_dtype)
        ctx.save_for_backward(total, weight, rstd)
        ctx.x_dtype, ctx.added = x.dtype, residual is not None
        ctx.set_materialize_grads(False)
        return (y, total) if ctx.added else y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dtotal=None):
        total, weight, rstd = ctx.saved_tensors
        if dy is None and dtotal is None:
            return None, None, None, None, None
        if dy is None:  # nobody read the norm
            return dtotal.to(ctx.x_dtype), None, dtotal, None, None
        dx, dresidual, dweight = _norm_backward(dy, total, weight, rstd, dtotal, ctx.x_dtype,
                                                ctx.needs_input_grad[1])
        return dx, dweight, dresidual if ctx.added else None, None, None


def rms_norm(x: torch.Tensor, weight: torch.Tensor, *, eps: float = 1e-6,
             residual: torch.Tensor | None = None, out_dtype: torch.dtype | None = None
             ) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """:func:`rms_norm_forward`'s ``y``, and with a residual ``(y, t)``, differentiable in ``x``,
    ``weight`` and ``residual``."""
    return _RmsNorm.apply(x, weight, residual, eps, out_dtype)


# ---- rotary positions -----------------------------------------------------------------------

def rotary_frequencies(width: int, *, base: float = 10000.0,
                       device: torch.device | str = "cuda") -> torch.Tensor:
    """``base^(−2i/width)`` for the ``width/2`` pairs i of a head, fp64."""
    if width < 2 or width % 2:
        raise ValueError(f"width must be even and positive, got {width}")
    i = torch.arange(0, width, 2, dtype=torch.float64)
    return (base ** (-i / width)).to(device)


def _turned(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor,
            frequencies: torch.Tensor, sections: Sequence[int] | None, adjacent: bool,
            inverse: bool) -> tuple[torch.Tensor, torch.Tensor]:
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError("q and k must be [batch, heads, n, head_dim]")
    b, h, n, d = q.shape
    kv = k.shape[1]
    code = _dtype(q, "q")
    if not 1 <= d <= MAX_ROTARY_DIM or h < 1 or kv < 1:
        raise ValueError(f"head_dim must be in [1, {MAX_ROTARY_DIM}] and there must be heads, got "
                         f"{tuple(q.shape)}")
    _like(k, q, (b, kv, n, d), "k")
    pairs = frequencies.numel()
    if (frequencies.dtype not in (torch.float32, torch.float64) or frequencies.dim() != 1
            or frequencies.device != q.device or not 2 <= 2 * pairs <= d):
        raise ValueError(f"frequencies must be float32 or float64 [pairs] on {q.device}, one for "
                         f"each pair of a head of {d}")
    counts = ends = (pairs,)
    if sections is not None:
        counts = tuple(sections)
        if not 1 <= len(counts) <= 4 or min(counts) < 0 or sum(counts) != pairs:
            raise ValueError(f"sections must be up to 4 counts whose sum is {pairs}, got {counts}")
        ends = tuple(itertools.accumulate(counts))
    axes, at = len(counts), positions
    if at.dtype not in (torch.int64, torch.int32) or at.device != q.device:
        raise ValueError(f"positions must be int64 or int32 on {q.device}")
    # (strides as they are: views of small tensors cost more than the launch)
    shape, strides = at.shape, at.stride()
    if sections is None:
        shape, strides = (1, *shape), (0, *strides)
    if len(shape) == 2:
        shape, strides = (shape[0], 1, shape[1]), (strides[0], 0, strides[1])
    if len(shape) != 3 or shape[0] != axes or shape[1] not in (1, b) or shape[2] != n:
        raise ValueError(f"positions must be {'' if sections is None else f'{axes} times '}"
                         f"[{n}] or [{b}, {n}], got {tuple(positions.shape)}")
    if shape[1] == 1:
        strides = (strides[0], 0, strides[2])
    _on_gpu(q)
    if q.stride(3) != 1:
        q = q.contiguous()
    if k.stride(3) != 1:
        k = k.contiguous()
    frequencies = frequencies.contiguous()
    of_q, of_k = (n * h * d, d, h * d), (n * kv * d, d, kv * d)  # as _new_heads has them
    to_q, to_k = q.new_empty_strided(q.shape, (*of_q, 1)), q.new_empty_strided(k.shape, (*of_k, 1))
    args = _packed(_ROTARY, q.data_ptr(), *q.stride()[:3], k.data_ptr(), *k.stride()[:3],
                   to_q.data_ptr(), *of_q, to_k.data_ptr(), *of_k, at.data_ptr(),
                   frequencies.data_ptr(), *strides, b, h, kv, n, d, pairs, axes, *ends,
                   *(pairs,) * (4 - axes), code, 0 if frequencies.dtype == torch.float32 else _F64,
                   64 if at.dtype == torch.int64 else 32, adjacent, inverse)
    native.get().operator("rotary_turn", args, q.device)
    return to_q, to_k


def rotary_forward(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor,
                   frequencies: torch.Tensor, *, sections: Sequence[int] | None = None,
                   adjacent: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """``q [b, h, n, d]`` and ``k [b, kv, n, d]`` with their pairs turned by the angles
    ``position · frequency``, any strides, fp32 or bf16, ``d`` up to 1024. ``frequencies`` (fp32
    or fp64 ``[pairs]``, :func:`rotary_frequencies`): pair i is the columns ``(i, i + pairs)``, or
    ``(2i, 2i + 1)`` with ``adjacent``; columns from ``2 · pairs`` on are copied. ``positions``
    (int64 or int32) are ``[n]`` or ``[b, n]``. With ``sections``, counts of consecutive pairs for
    each of up to 4 axes (time, height, width), they are ``[axes, n]`` or ``[axes, b, n]``. Angles
    are taken in 64 bits. The results lie in memory as ``[b, n, heads, d]``."""
    return _turned(q, k, positions, frequencies, sections, adjacent, False)


def rotary_backward(dq: torch.Tensor, dk: torch.Tensor, positions: torch.Tensor,
                    frequencies: torch.Tensor, *, sections: Sequence[int] | None = None,
                    adjacent: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """The gradients of :func:`rotary_forward`'s ``q`` and ``k`` from those of its results: the
    turns back."""
    return _turned(dq, dk, positions, frequencies, sections, adjacent, True)


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, frequencies, sections, adjacent):
        ctx.save_for_backward(positions, frequencies)
        ctx.kw = {"sections": sections, "adjacent": adjacent}
        return rotary_forward(q, k, positions, frequencies, **ctx.kw)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq, dk):
        return *rotary_backward(dq, dk, *ctx.saved_tensors, **ctx.kw), None, None, None, None


def rotary(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, frequencies: torch.Tensor,
           *, sections: Sequence[int] | None = None, adjacent: bool = False
           ) -> tuple[torch.Tensor, torch.Tensor]:
    """:func:`rotary_forward`, differentiable in ``q`` and ``k``."""
    return _Rotary.apply(q, k, positions, frequencies, sections, adjacent)


# ---- the gated activation -------------------------------------------------------------------

def _gated_args(gate: torch.Tensor, up: torch.Tensor) -> int:
    code = _dtype(gate, "gate")
    if gate.dim() < 1:
        raise ValueError("gate must be [..., columns]")
    _like(up, gate, gate.shape, "up")
    return code


def gated_silu_forward(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """``silu(gate) · up``, ``silu(g) = g / (1 + e^−g)``, of two tensors ``[..., columns]`` of one
    shape and type, each anywhere (the halves of one product, for instance): up to 2^32 − 1 rows
    of up to 2^32 − 1 values, and 2^40 values in all."""
    code = _gated_args(gate, up)
    _on_gpu(gate)
    out = _new_like(gate, gate.dtype)
    if out.numel():
        (g, g_row), (u, u_row), columns = _rows(gate), _rows(up), gate.shape[-1]
        args = _packed(_GATED, g.data_ptr(), u.data_ptr(), 0, out.data_ptr(), 0, 0, g_row, u_row, 0,
                       out.numel() // columns, columns, code)
        native.get().operator("gated_silu_forward", args, gate.device)
    return out


def gated_silu_backward(dout: torch.Tensor, gate: torch.Tensor, up: torch.Tensor
                        ) -> tuple[torch.Tensor, torch.Tensor]:
    """``(dgate, dup)`` of :func:`gated_silu_forward`."""
    code = _gated_args(gate, up)
    _like(dout, gate, gate.shape, "dout")
    _on_gpu(gate)
    dgate, dup = _new_like(gate, gate.dtype), _new_like(gate, gate.dtype)
    if dgate.numel():
        (g, g_row), (u, u_row), (d, d_row) = _rows(gate), _rows(up), _rows(dout)
        columns = gate.shape[-1]
        args = _packed(_GATED, g.data_ptr(), u.data_ptr(), d.data_ptr(), 0, dgate.data_ptr(),
                       dup.data_ptr(), g_row, u_row, d_row, dgate.numel() // columns, columns, code)
        native.get().operator("gated_silu_backward", args, gate.device)
    return dgate, dup


class _GatedSilu(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, up):
        ctx.save_for_backward(gate, up)
        return gated_silu_forward(gate, up)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        return gated_silu_backward(g, *ctx.saved_tensors)


def gated_silu(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """:func:`gated_silu_forward`, differentiable in ``gate`` and ``up``."""
    return _GatedSilu.apply(gate, up)


# ---- the whole gradient ---------------------------------------------------------------------

# what a list's checks read of every tensor, as functions that map() calls without a frame
_TYPE_OF, _SHAPE_OF = operator.attrgetter("dtype"), operator.attrgetter("shape")
_DEVICE_OF, _POINTER, _COUNT = torch.Tensor.get_device, torch.Tensor.data_ptr, torch.Tensor.numel
_CONTIGUOUS = torch.Tensor.is_contiguous


class _List:
    """Tensors of one device: their types, and whether all are contiguous."""

    def __init__(self, of: Sequence[torch.Tensor], what: str) -> None:
        self.tensors, self.what = list(of), what
        if not self.tensors:
            raise ValueError(f"{what} must be tensors, at least one")
        try:
            self.devices = set(map(_DEVICE_OF, self.tensors))
            self.types = list(map(_DTYPES.get, map(_TYPE_OF, self.tensors)))
            self.whole = all(map(_CONTIGUOUS, self.tensors))
        except TypeError:
            raise ValueError(f"{what} must be tensors, at least one") from None
        if None in self.types or not self.whole and any(
                [t.layout is not torch.strided for t in self.tensors]):
            raise ValueError(f"{what} must be dense, float32 or bfloat16")
        if len(self.devices) > 1:
            raise ValueError(f"{what} must be on one device")

    def like(self, other: "_List", types: bool) -> None:
        if self.devices != other.devices:
            raise ValueError(f"{self.what} and {other.what} must be on one device")
        if list(map(_SHAPE_OF, self.tensors)) != list(map(_SHAPE_OF, other.tensors)):
            raise ValueError(f"{self.what} and {other.what} must have the same shapes")
        if types and self.types != other.types:
            raise ValueError(f"{self.what} and {other.what} must have the same types")

    def read(self) -> list[torch.Tensor]:
        return self.tensors if self.whole else [t.contiguous() for t in self.tensors]


def _written(out: Sequence[torch.Tensor] | None, of: _List) -> _List:
    """Where the results go that stand for ``of``: there, unless there is an ``out``."""
    to = of
    if out is not None:
        to = _List(out, "out")
        to.like(of, types=True)
    if not to.whole:
        raise ValueError(f"{to.what} must be contiguous, since they are written")
    return to


def _change(name: str, gradients: _List, weights: _List | None, out: _List | None,
            max_norm: float, eta: float) -> torch.Tensor:
    """The calls over lists; the norm."""
    first = gradients.tensors[0]
    _on_gpu(first)
    norm = _new_floats((), first)
    g = gradients.read()
    pointers = list(map(_POINTER, g))
    zeros = [0] * len(g)
    w_pointers, w_types, to = zeros, zeros, pointers
    if weights is not None:
        w = weights.read()
        to = w_pointers = list(map(_POINTER, w))
        w_types = weights.types
    if out is not None and out is not gradients and out is not weights:
        to = list(map(_POINTER, out.tensors))
    entries = map(_GRADIENT.pack, pointers, w_pointers, to, map(_COUNT, g), gradients.types, w_types)
    args = _packed(_GRADIENTS, norm.data_ptr(), max_norm, eta, len(g), 0) + b"".join(entries)
    native.get().operator(name, args, first.device)
    if out is not None:  # autograd is told, as it is of any write (it counts none of inference's)
        try:
            torch.autograd.graph.increment_version(out.tensors)
        except RuntimeError:
            torch.autograd.graph.increment_version([t for t in out.tensors if not t.is_inference()])
    return norm


def _max_norm(max_norm: float) -> float:
    if not max_norm >= _LEAST:
        raise ValueError(f"max_norm must be positive in fp32, got {max_norm}")
    return max_norm if max_norm <= _MOST else math.inf


def gradient_norm(gradients: Sequence[torch.Tensor]) -> torch.Tensor:
    """The 2-norm of the values of all ``gradients`` (fp32 or bf16, of any shapes) together, fp32
    ``[]``. Squares are added in fp64, so nothing overflows on the way."""
    return _change("gradient_norm", _List(gradients, "gradients"), None, None, 0.0, 0.0)


def clip_gradients(gradients: Sequence[torch.Tensor], max_norm: float, *,
                   out: Sequence[torch.Tensor] | None = None) -> torch.Tensor:
    """Scale ``gradients`` by ``min(1, max_norm / norm)``, in place or into ``out``; returns their
    :func:`gradient_norm`. A norm that is NaN makes every value NaN, and an infinite one zero but
    for the infinities (NaN); with an infinite ``max_norm`` nothing is scaled, whatever the norm. What
    is written must be contiguous, and overlap nothing but the gradient that it replaces."""
    g = _List(gradients, "gradients")
    return _change("clip_gradients", g, None, _written(out, g), _max_norm(max_norm), 0.0)


def sgd_step(weights: Sequence[torch.Tensor], gradients: Sequence[torch.Tensor], eta: float, *,
             max_norm: float = math.inf, out: Sequence[torch.Tensor] | None = None
             ) -> torch.Tensor:
    """``W ← W − eta · min(1, max_norm / norm) · G`` over a model's weights and their gradients, in
    place or into ``out``, the gradients left as they are; returns their :func:`gradient_norm`.
    Weights and gradients are fp32 or bf16 each; the update is one fp32 multiplication and addition,
    rounded once. Without a bound (``max_norm`` infinite) it is ``W − eta · G`` value by value; norms that
    are not finite otherwise, and what is written: :func:`clip_gradients`."""
    g, w = _List(gradients, "gradients"), _List(weights, "weights")
    w.like(g, types=False)
    if not -_MOST <= eta <= _MOST:
        raise ValueError(f"eta must be finite in fp32, got {eta}")
    return _change("sgd_step", g, w, _written(out, w), _max_norm(max_norm), eta)
