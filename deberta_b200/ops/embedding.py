"""Embedding lookup with an optional second (delta) table, and its gradient scatter.

Covers the plain word-embedding gather and the gradient-disentangled form ``base[ids] + delta[ids]`` of the
reference (``modeling/rtd.py:157-226``) in one kernel; the backward adds the output gradient rows straight into the
fp32 ``main_grad`` buffers of the trainable tables (no dense ``[vocab, hidden]`` gradient tensor, no sort). Without a
GPU, without ``main_grad`` buffers, or for other dtypes it is ``F.embedding``.

Those additions are atomic, so rows that several tokens share are summed in an order that varies from run to run. Under
``torch.use_deterministic_algorithms(True)`` the buffers get their rows from ``csrc/embed_sorted.cu`` instead, which sorts the
tokens and adds in a fixed order; :func:`scaled_embedding` always does.
"""

from __future__ import annotations

import ctypes
import functools

import torch
import torch.nn.functional as F

from . import _lib
from .dropout import DTYPE_CODES, on_device, rows_view

__all__ = ["embedding_lookup", "scaled_embedding"]


def _usable(table: torch.Tensor | None) -> bool:
    return table is None or (table.is_cuda and table.dtype == torch.bfloat16 and table.is_contiguous()
                             and table.shape[1] % 8 == 0)


def _grad_ready(table: torch.Tensor | None) -> bool:
    """Frozen tables need nothing; trainable ones need the engine's fp32 gradient buffer."""
    if table is None or not table.requires_grad:
        return True
    g = getattr(table, "main_grad", None)
    return g is not None and g.dtype == torch.float32 and g.is_contiguous()


def embed_forward(ids, table, delta):
    """``table[ids] (+ delta[ids])``: one kernel on bf16 CUDA tables, ``F.embedding`` otherwise."""
    if table.is_cuda and table.dtype == torch.bfloat16:
        flat = ids.reshape(-1).to(torch.int64).contiguous()
        vocab, hidden = table.shape
        out = torch.empty((flat.numel(), hidden), dtype=table.dtype, device=table.device)
        _lib.call("db200_embed_fwd", _lib.ptr(flat), _lib.ptr(table), _lib.ptr(delta), _lib.ptr(out),
                  ctypes.c_longlong(flat.numel()), ctypes.c_int(hidden), ctypes.c_longlong(vocab), _lib.stream_ptr())
        return out.view(*ids.shape, hidden)
    out = F.embedding(ids, table)
    return out if delta is None else out + F.embedding(ids, delta)


def embed_backward(dout, ids, vocab: int, padding_idx: int, grads) -> None:
    """Add the rows of ``dout`` to row ``ids[t]`` of every fp32 buffer in ``grads`` (``None`` entries skipped)."""
    d2 = dout.reshape(-1, dout.shape[-1])
    flat = ids.reshape(-1).to(torch.int64).contiguous()
    if d2.is_cuda and d2.dtype == torch.bfloat16:
        if d2.stride(-1) != 1 or d2.stride(0) % 8 or d2.data_ptr() % 16:
            d2 = d2.contiguous()
        grads = [g for g in grads if g is not None]
        if torch.are_deterministic_algorithms_enabled() and grads and flat.numel():
            d2, ld = rows_view(d2)
            _sorted_backward(d2, ld, flat, d2.shape[1], vocab, int(padding_idx), 1.0, None, grads)
            return
        for g in grads:
            if g is not None:
                _lib.call("db200_embed_bwd", _lib.ptr(flat), _lib.ptr(d2), ctypes.c_longlong(d2.stride(0)), _lib.ptr(g),
                          ctypes.c_longlong(flat.numel()), ctypes.c_int(d2.shape[1]), ctypes.c_longlong(vocab),
                          ctypes.c_longlong(int(padding_idx)), _lib.stream_ptr())
        return
    rows = d2.float()
    if padding_idx >= 0:
        rows = rows * flat.ne(padding_idx).unsqueeze(-1).to(rows.dtype)
    for g in grads:
        if g is not None:
            g.index_add_(0, flat, rows.to(g.dtype))


class _Embed(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, table, delta, padding_idx):
        ctx.ids, ctx.tables, ctx.padding_idx = ids, (table, delta), padding_idx
        return embed_forward(ids, table, delta)

    @staticmethod
    def backward(ctx, dout):
        pad = -1 if ctx.padding_idx is None else int(ctx.padding_idx)
        grads = [t.main_grad if (t is not None and t.requires_grad) else None for t in ctx.tables]
        embed_backward(dout, ctx.ids, ctx.tables[0].shape[0], pad, grads)
        return None, None, None, None


def embedding_lookup(ids: torch.Tensor, table: torch.Tensor, delta: torch.Tensor | None = None,
                     padding_idx: int | None = None) -> torch.Tensor:
    """``table[ids] (+ delta[ids])``; gradients of trainable tables go to their ``main_grad`` on the kernel path."""
    # Under a compiler the lookup is F.embedding (the kernel path scatters into the engine's gradient buffers, and ops that
    # mutate views of the flat gradient storage do not go into a compiled graph: see ops/linear.py:linear).
    if _usable(table) and _usable(delta) and table.is_cuda and _grad_ready(table) and _grad_ready(delta) and \
            (delta is None or delta.shape == table.shape) and not torch.compiler.is_compiling():
        if torch.is_grad_enabled() and (table.requires_grad or (delta is not None and delta.requires_grad)):
            return _Embed.apply(ids, table, delta, padding_idx)
        return embed_forward(ids, table, delta)
    out = F.embedding(ids, table, padding_idx=padding_idx)
    if delta is not None:
        out = out + F.embedding(ids, delta, padding_idx=padding_idx)
    return out


# ---- scaled lookup with a gradient by sorted tokens ----------------------------------------------------------------------
_P, _LL, _I, _F = _lib.c_void_p, _lib.c_ll, _lib.c_int, _lib.c_float
_gather = _lib.bind("db200_embed_scaled", _P, _P, _P, _LL, _I, _LL, _F, _I, _P)
_sorted_sums = _lib.bind("db200_embed_sorted_bwd", _P, _P, _LL, _LL, _I, _LL, _LL, _F, _I, _P, _P, _P, _P, _P)


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(tokens: int, cols: int, vocab: int) -> int:
    fn = _lib.lib().db200_embed_sorted_workspace
    fn.restype = _LL
    return int(fn(_LL(tokens), _I(cols), _LL(vocab)))


def _sorted_backward(d2, ld: int, flat, cols: int, vocab: int, padding_idx: int, scale: float, grad, buffers) -> None:
    """``scale`` times the rows of ``d2`` summed by id: written to ``grad`` (dense, every row) or added to one or two fp32
    ``buffers``, in an order that the ids alone decide."""
    n = flat.numel()
    size = _workspace_bytes(n, cols, vocab)
    work = torch.empty(size, dtype=torch.uint8, device=d2.device) if size else None
    acc = [*(b.data_ptr() for b in buffers), None, None]
    _sorted_sums(flat.data_ptr(), d2.data_ptr(), ld, n, cols, vocab, padding_idx, scale, DTYPE_CODES[d2.dtype],
                 None if grad is None else grad.data_ptr(), acc[0], acc[1],
                 None if work is None else work.data_ptr(), _lib.raw_stream())


class _ScaledEmbed(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, table, scale, padding_idx):
        vocab, cols = table.shape
        with on_device(table):
            flat = ids.to(torch.int64).contiguous()
            out = torch.empty((*ids.shape, cols), dtype=table.dtype, device=table.device)
            _gather(flat.data_ptr(), table.data_ptr(), out.data_ptr(), flat.numel(), cols, vocab, scale,
                    DTYPE_CODES[table.dtype], _lib.raw_stream())
        ctx.save_for_backward(flat)
        ctx.table = table  # (its shape and gradient buffer)
        ctx.meta = (scale, padding_idx)
        return out

    @staticmethod
    def backward(ctx, dout):
        if torch.is_grad_enabled():  # (a second derivative is refused when it is asked for)
            return _scaled_embed_backward_once(ctx, dout)
        return _scaled_embed_backward(ctx, dout)


def _scaled_embed_backward(ctx, dout):
    (flat,) = ctx.saved_tensors
    table, (scale, padding_idx) = ctx.table, ctx.meta
    buffer = getattr(table, "main_grad", None)
    vocab, cols = table.shape
    with on_device(table):
        d2, ld = rows_view(dout)
        grad = torch.empty_like(table) if buffer is None else None
        _sorted_backward(d2, ld, flat, cols, vocab, padding_idx, scale, grad, () if buffer is None else (buffer,))
    return None, grad, None, None


_scaled_embed_backward_once = torch.autograd.function.once_differentiable(_scaled_embed_backward)


def scaled_embedding(ids: torch.Tensor, table: torch.Tensor, scale: float = 1.0,
                     padding_idx: int | None = None) -> torch.Tensor:
    """``scale * table[ids]`` with a reproducible gradient.

    ``ids``: integers of any shape on the device of ``table`` (``[vocab, hidden]``). Tokens with id ``padding_idx`` are looked up
    but have no gradient. The gradient is summed in fp32 by sorted tokens, the same bits in every run: dense in the table's type,
    or added to the table's ``main_grad`` where it has one. On contiguous bf16, fp16 and fp32 CUDA tables this is
    ``csrc/embed_sorted.cu``, which reads ids out of range as the nearest row and leaves them out of the gradient; elsewhere it
    is ``F.embedding``."""
    if table.dim() != 2 or not table.is_floating_point():
        raise ValueError(f"table must be a floating [vocab, hidden] tensor, got {table.dtype} of shape {tuple(table.shape)}.")
    if ids.dtype not in (torch.int64, torch.int32) or ids.device != table.device:
        raise ValueError(f"ids must be int64 or int32 on {table.device}, got {ids.dtype} on {ids.device}.")
    vocab = table.shape[0]
    if padding_idx is not None:
        if not -vocab <= padding_idx < vocab:
            raise ValueError(f"padding_idx {padding_idx} is outside the table's {vocab} rows.")
        padding_idx = int(padding_idx) % vocab
    buffer = getattr(table, "main_grad", None) if table.requires_grad else None
    if (table.is_cuda and table.dtype in DTYPE_CODES and table.is_contiguous() and table.numel() and ids.numel()
            and (buffer is None or (buffer.dtype == torch.float32 and buffer.is_contiguous()))
            and not torch.compiler.is_compiling()):
        return _ScaledEmbed.apply(ids, table, float(scale), -1 if padding_idx is None else padding_idx)
    return F.embedding(ids, table, padding_idx=padding_idx) * float(scale)
