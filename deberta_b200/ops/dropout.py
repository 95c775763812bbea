"""Dropout whose mask is a function of a seed and of the place, and is never stored.

Column ``c`` of row ``r`` (the last dimension; all leading dimensions counted as one) is dropped where 16 of the 128 bits
that Philox4x32-7 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011) gives at counter
``(c // 8, r mod 2^32, r // 2^32, 0)`` under the 64-bit seed are below ``round(p * 65536)``. The probability is therefore
a multiple of 2^-16 (0.1 becomes 6554/65536), the kept values are scaled by its exact complement, and ``p`` below 2^-17
drops nothing. The backward pass draws the same bits again, on any layout, device or stream and in a replayed graph; so does
a recomputed forward pass. Where a value is dropped its infinities and NaN are dropped with it.

The seed is an ``int`` (its low 64 bits) or an int64 tensor with one element on the device of the data, which is read when
the kernel runs: a captured graph draws new masks when the tensor changes between replays. Two calls with one seed and one
width draw the same bits; :func:`draw_seed` gives a fresh seed from torch's generator without a synchronisation.

On bf16, fp16 and fp32 CUDA tensors the operators run ``csrc/dropout.cu`` (under a compiler as custom ops); elsewhere they are
the PyTorch statement of the same map (:func:`dropout_keep_mask`).
"""

from __future__ import annotations

import contextlib
import ctypes

import torch

from . import _lib

__all__ = ["dropout", "dropout_add", "dropout_keep_mask", "dropout_threshold", "draw_seed"]

DTYPE_CODES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_LOW = 0xFFFFFFFF


def dropout_threshold(p: float) -> int:
    """``round(p * 65536)``; ``p`` has to leave something: 0 <= p < 1 after rounding."""
    p = float(p)
    if not 0.0 <= p < 1.0 or int(p * 65536.0 + 0.5) > 65535:
        raise ValueError(f"dropout probability must be in [0, 1 - 2^-17), got {p}.")
    return int(p * 65536.0 + 0.5)


def inverse_keep(threshold: int) -> float:
    """What kept values are multiplied by."""
    return 65536.0 / (65536 - threshold)


def draw_seed(device: torch.device | str | None = None) -> torch.Tensor:
    """A fresh seed (int64, one element) from torch's generator of ``device``: follows ``torch.manual_seed``, is repeated by
    activation checkpointing, and a captured graph draws a new one at every replay."""
    return torch.randint(0, 1 << 62, (1,), dtype=torch.int64, device=device)


def check_seed(seed, device: torch.device) -> None:
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1:
            raise ValueError(f"a seed tensor must be int64 with one element, got {seed.dtype} with {seed.numel()}.")
        if seed.device != device:
            raise ValueError(f"the seed is on {seed.device}, the data on {device}.")
    elif isinstance(seed, bool) or not isinstance(seed, int):
        raise TypeError(f"seed must be an int or an int64 tensor with one element, got {type(seed).__name__}.")


def seed_args(seed) -> tuple[int | None, int]:
    """(device address or ``None``, value) as the launchers take them."""
    if isinstance(seed, torch.Tensor):
        return seed.data_ptr(), 0
    return None, seed & 0xFFFFFFFFFFFFFFFF


_HERE = contextlib.nullcontext()


def on_device(t: torch.Tensor):
    """Makes the device of ``t`` the current one: launches go to its streams."""
    return _HERE if t.get_device() == torch.cuda.current_device() else torch.cuda.device(t.device)


def seed_tensor(seed, device) -> torch.Tensor:
    """The seed as the custom ops take it."""
    if isinstance(seed, torch.Tensor):
        return seed
    return torch.full((1,), ((int(seed) + (1 << 63)) & ((1 << 64) - 1)) - (1 << 63), dtype=torch.int64, device=device)


def dropout_keep_mask(shape, p: float, seed, device: torch.device | str | None = None) -> torch.Tensor:
    """bool tensor of ``shape``: the places that dropout with this seed keeps (the PyTorch statement of the map)."""
    t = dropout_threshold(p)
    shape = tuple(int(s) for s in shape)
    device = seed.device if isinstance(seed, torch.Tensor) and device is None else device
    cols = shape[-1] if shape else 1
    rows = 1
    for s in shape[:-1]:
        rows *= s
    if torch.compiler.is_compiling():  # (a compiler that narrows index arithmetic to 32 bits must not see the products)
        from . import library

        return library.dropout_keep(seed_tensor(seed, device).to(device), rows, cols, t).view(shape)
    return _keep_rows(rows, cols, t, seed, device).reshape(shape)


def _keep_rows(rows: int, cols: int, threshold: int, seed, device) -> torch.Tensor:
    if isinstance(seed, torch.Tensor):
        wide = seed.to(device).reshape(())
        k0, k1 = wide & _LOW, (wide >> 32) & _LOW
    else:
        k0, k1 = int(seed) & _LOW, (int(seed) >> 32) & _LOW
    row = torch.arange(rows, device=device)[:, None]
    c0 = torch.arange((cols + 7) // 8, device=device)[None, :]
    c1, c2, c3 = row & _LOW, row >> 32, torch.zeros_like(row)
    for _ in range(7):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # products modulo 2^64; the shifts below mask the sign away
        c0, c1, c2, c3 = ((b >> 32) & _LOW) ^ c1 ^ k0, b & _LOW, ((a >> 32) & _LOW) ^ c3 ^ k1, a & _LOW
        k0, k1 = (k0 + 0x9E3779B9) & _LOW, (k1 + 0xBB67AE85) & _LOW
    words = torch.stack(torch.broadcast_tensors(c0, c1, c2, c3), dim=-1)
    halves = torch.stack((words & 0xFFFF, words >> 16), dim=-1).reshape(rows, (cols + 7) // 8 * 8)[:, :cols]
    return halves >= threshold


def dropout_reference(x: torch.Tensor, residual: torch.Tensor | None, threshold: int, seed) -> torch.Tensor:
    """The PyTorch statement: fp32 (fp64 for fp64 inputs), rounded once."""
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    keep = dropout_keep_mask(x.shape, threshold / 65536.0, seed, x.device)
    out = torch.where(keep, x.to(wide) * inverse_keep(threshold), torch.zeros((), dtype=wide, device=x.device))
    return (out if residual is None else out + residual.to(wide)).to(x.dtype)


def rows_view(x: torch.Tensor) -> tuple[torch.Tensor, int]:
    """(tensor, row stride) of ``x`` as rows of its last dimension with unit inner stride: ``x`` itself where it is contiguous,
    a two-dimensional view where its layout has one, else a copy."""
    if x.is_contiguous():
        return x, (x.shape[-1] if x.dim() else 1)
    x2 = x.reshape(-1, x.shape[-1])
    rows, cols = x2.shape
    if (cols > 1 and x2.stride(1) != 1) or (rows > 1 and x2.stride(0) < cols):
        x2 = x2.contiguous()
    return x2, (x2.stride(0) if rows > 1 else cols)


_MAX_COLS = (1 << 31) - 16  # the kernels count a row's columns in 32 bits


def kernel_ok(x: torch.Tensor) -> bool:
    return x.is_cuda and x.dtype in DTYPE_CODES and x.numel() > 0 and (x.dim() == 0 or x.shape[-1] <= _MAX_COLS)


_P, _LL, _I, _F = _lib.c_void_p, _lib.c_ll, _lib.c_int, _lib.c_float
SEED_TYPES = (_P, ctypes.c_ulonglong, ctypes.c_uint, _F)  # address, value, threshold, scale
_dropout_kernel = _lib.bind("db200_dropout", _P, _LL, _P, _LL, _P, _LL, _I, _I, *SEED_TYPES, _P)


def _launch(x, residual, threshold: int, seed) -> torch.Tensor:
    with on_device(x):
        x2, ldx = rows_view(x)
        r2, ldr = (None, 0) if residual is None else rows_view(residual)
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
        cols = x.shape[-1] if x.dim() else 1
        address, value = seed_args(seed)
        _dropout_kernel(x2.data_ptr(), ldx, None if r2 is None else r2.data_ptr(), ldr, out.data_ptr(), x.numel() // cols,
                        cols, DTYPE_CODES[x.dtype], address, value, threshold, inverse_keep(threshold), _lib.raw_stream())
    return out


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, threshold, seed):
        held = isinstance(seed, torch.Tensor)
        if held:
            ctx.save_for_backward(seed)  # (a seed that is overwritten before the backward pass is an error)
        ctx.meta = (threshold, None if held else seed)
        return _launch(x, residual, threshold, seed)

    @staticmethod
    def backward(ctx, dy):
        threshold, seed = ctx.meta
        if seed is None:
            (seed,) = ctx.saved_tensors
        dx = None
        if ctx.needs_input_grad[0]:  # the same operator again, which is differentiable in turn
            dx = (_Dropout.apply if torch.is_grad_enabled() else _launch)(dy, None, threshold, seed)
        return dx, (dy if ctx.needs_input_grad[1] else None), None, None


def _run(x, residual, threshold: int, seed) -> torch.Tensor:
    if kernel_ok(x):
        if torch.compiler.is_compiling():
            from . import library

            return library.dropout(x, residual, seed_tensor(seed, x.device), threshold)
        return _Dropout.apply(x, residual, threshold, seed)
    return dropout_reference(x, residual, threshold, seed)


def check_pair(x: torch.Tensor, residual: torch.Tensor) -> None:
    if x.shape != residual.shape or x.dtype != residual.dtype or x.device != residual.device:
        raise ValueError(f"x and residual must agree: {tuple(x.shape)} {x.dtype} {x.device} and "
                         f"{tuple(residual.shape)} {residual.dtype} {residual.device}.")


def dropout(x: torch.Tensor, p: float, seed, *, training: bool = True) -> torch.Tensor:
    """``x`` with each value dropped with probability ``p`` and the others divided by ``1 - p``; ``x`` itself out of training.

    ``x``: floating, any shape and strides; the result is contiguous."""
    threshold = dropout_threshold(p)
    check_seed(seed, x.device)
    if not x.is_floating_point():
        raise TypeError(f"dropout needs a floating tensor, got {x.dtype}.")
    return _run(x, None, threshold, seed) if training and threshold else x


def dropout_add(x: torch.Tensor, residual: torch.Tensor, p: float, seed, *, training: bool = True) -> torch.Tensor:
    """``residual + dropout(x)``, summed in fp32 and rounded once. Both have one shape, type and device."""
    threshold = dropout_threshold(p)
    check_seed(seed, x.device)
    check_pair(x, residual)
    if not x.is_floating_point():
        raise TypeError(f"dropout needs a floating tensor, got {x.dtype}.")
    return _run(x, residual, threshold, seed) if training and threshold else residual + x
