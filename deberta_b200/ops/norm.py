"""LayerNorm and RMSNorm with fp32 statistics (``csrc/norm.cu`` on bf16 CUDA tensors), and the same norms of a residual
sum with dropout on the branch (``add_layer_norm``, ``add_rms_norm``: ``csrc/add_norm.cu``)."""

from __future__ import annotations

import ctypes
import functools

import torch
import torch.nn.functional as F

from . import _lib
from .dropout import (DTYPE_CODES, SEED_TYPES, check_pair, check_seed, dropout_keep_mask, dropout_threshold, inverse_keep,
                      kernel_ok, on_device, rows_view, seed_args, seed_tensor)

__all__ = ["layer_norm", "rms_norm", "add_layer_norm", "add_rms_norm", "layer_norm_reference", "rms_norm_reference",
           "add_norm_reference"]


def layer_norm_reference(x, weight, bias, eps, row_keep=None):
    y = F.layer_norm(x.float(), (x.shape[-1],), weight.float(), None if bias is None else bias.float(), eps)
    if row_keep is not None:
        y = y * row_keep.unsqueeze(-1).to(y.dtype)
    return y.to(x.dtype)


def rms_norm_reference(x, weight, eps, row_keep=None):
    xf = x.float()
    y = xf * torch.rsqrt(xf.pow(2).mean(dim=-1, keepdim=True) + eps) * weight.float()
    if row_keep is not None:
        y = y * row_keep.unsqueeze(-1).to(y.dtype)
    return y.to(x.dtype)


def _kernel_ok(x: torch.Tensor, weight: torch.Tensor) -> bool:
    return (
        x.is_cuda
        and x.dtype == torch.bfloat16
        and weight.dtype == torch.bfloat16
        and x.shape[-1] % 8 == 0
        and x.shape[-1] <= 2048
    )


def norm_forward(x, weight, bias, row_keep, eps: float, rms: bool):
    """(y, mean, rstd) of ``x`` [rows, H]; ``mean`` is empty for RMSNorm. Kernel on bf16 CUDA, PyTorch otherwise."""
    rows, H = x.shape
    if _kernel_ok(x, weight):
        y = torch.empty_like(x)
        mean = torch.empty(0 if rms else rows, dtype=torch.float32, device=x.device)
        rstd = torch.empty(rows, dtype=torch.float32, device=x.device)
        keep = None if row_keep is None else row_keep.to(torch.uint8).contiguous()
        _lib.call(
            "db200_norm_fwd", _lib.ptr(x), _lib.ptr(weight), _lib.ptr(bias), _lib.ptr(keep), _lib.ptr(y),
            _lib.ptr(None if rms else mean), _lib.ptr(rstd), ctypes.c_int(rows), ctypes.c_int(H), ctypes.c_float(eps),
            ctypes.c_int(int(rms)), _lib.stream_ptr(),
        )
        return y, mean, rstd
    xf = x.float()
    if rms:
        mean = torch.empty(0, dtype=torch.float32, device=x.device)
        rstd = torch.rsqrt(xf.pow(2).mean(dim=-1) + eps)
        y = xf * rstd[:, None] * weight.float()
    else:
        mean = xf.mean(dim=-1)
        rstd = torch.rsqrt(xf.var(dim=-1, unbiased=False) + eps)
        y = (xf - mean[:, None]) * rstd[:, None] * weight.float()
        if bias is not None:
            y = y + bias.float()
    if row_keep is not None:
        y = y * row_keep.reshape(-1, 1).to(y.dtype)
    return y.to(x.dtype), mean, rstd


def norm_backward(dy, x, weight, mean, rstd, row_keep, rms: bool, has_bias: bool, w_grad, b_grad):
    """(dx, dgamma, dbeta): a parameter gradient that was added to its fp32 buffer (``w_grad`` / ``b_grad``) is ``None``."""
    rows, H = x.shape
    dy = dy.contiguous()
    if _kernel_ok(x, weight):
        dx = torch.empty_like(x)
        dg = w_grad if w_grad is not None else torch.zeros(H, dtype=torch.float32, device=x.device)
        db = None
        if has_bias:
            db = b_grad if b_grad is not None else torch.zeros(H, dtype=torch.float32, device=x.device)
        keep = None if row_keep is None else row_keep.to(torch.uint8).contiguous()
        _lib.call(
            "db200_norm_bwd", _lib.ptr(dy), _lib.ptr(x), _lib.ptr(weight), _lib.ptr(None if rms else mean), _lib.ptr(rstd),
            _lib.ptr(keep), _lib.ptr(dx), _lib.ptr(dg), _lib.ptr(db), ctypes.c_int(rows), ctypes.c_int(H),
            ctypes.c_int(int(rms)), _lib.stream_ptr(),
        )
        return (dx, None if w_grad is not None else dg.to(weight.dtype),
                None if (db is None or b_grad is not None) else db.to(weight.dtype))
    dyf, xf, g = dy.float(), x.float(), weight.float()
    if row_keep is not None:
        dyf = dyf * row_keep.reshape(-1, 1).to(dyf.dtype)
    xhat = xf * rstd[:, None] if rms else (xf - mean[:, None]) * rstd[:, None]
    dgamma = (dyf * xhat).sum(0)
    dbeta = dyf.sum(0) if has_bias else None
    dxhat = dyf * g
    if rms:
        dx = rstd[:, None] * (dxhat - xhat * (dxhat * xhat).mean(dim=-1, keepdim=True))
    else:
        dx = rstd[:, None] * (dxhat - dxhat.mean(dim=-1, keepdim=True) - xhat * (dxhat * xhat).mean(dim=-1, keepdim=True))
    if w_grad is not None:
        w_grad.add_(dgamma)
        dgamma = None
    if dbeta is not None and b_grad is not None:
        b_grad.add_(dbeta)
        dbeta = None
    return (dx.to(x.dtype), None if dgamma is None else dgamma.to(weight.dtype),
            None if dbeta is None else dbeta.to(weight.dtype))


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, rms, row_keep):
        keep = None if row_keep is None else row_keep.to(torch.uint8).contiguous()
        y, mean, rstd = norm_forward(x, weight, bias, keep, eps, rms)
        ctx.save_for_backward(x, mean, rstd, keep)
        ctx.refs = (weight, bias)
        ctx.rms = rms
        return y

    @staticmethod
    def backward(ctx, dy):
        x, mean, rstd, keep = ctx.saved_tensors
        weight, bias = ctx.refs
        has_bias = bias is not None and bias.requires_grad
        w_grad = getattr(weight, "main_grad", None) if weight.requires_grad else None
        b_grad = getattr(bias, "main_grad", None) if has_bias else None
        dx, gw, gb = norm_backward(dy, x, weight, mean, rstd, keep, ctx.rms, has_bias, w_grad, b_grad)
        return dx, (gw if weight.requires_grad else None), gb, None, None, None


def _norm_apply(x2, weight, bias, eps: float, rms: bool, rk):
    if torch.compiler.is_compiling():
        from . import library

        # (no gradient buffers under a compiler: see ops/linear.py:linear)
        return library.norm(x2, weight, bias, rk, float(eps), rms, None, None)[0]
    return _Norm.apply(x2, weight, bias, float(eps), rms, rk)


def layer_norm(x, weight, bias, eps: float, row_keep: torch.Tensor | None = None):
    """LayerNorm over the last dim; ``row_keep`` (bool per row) zeroes whole output rows."""
    if not _kernel_ok(x, weight):
        return layer_norm_reference(x, weight, bias, eps, row_keep)
    lead = x.shape[:-1]
    x2 = x.reshape(-1, x.shape[-1]).contiguous()
    rk = None if row_keep is None else row_keep.reshape(-1)
    return _norm_apply(x2, weight, bias, eps, False, rk).view(*lead, x.shape[-1])


def rms_norm(x, weight, eps: float, row_keep: torch.Tensor | None = None):
    """RMSNorm ``x * rsqrt(mean(x^2) + eps) * weight`` with fp32 reduction."""
    if not _kernel_ok(x, weight):
        return rms_norm_reference(x, weight, eps, row_keep)
    lead = x.shape[:-1]
    x2 = x.reshape(-1, x.shape[-1]).contiguous()
    rk = None if row_keep is None else row_keep.reshape(-1)
    return _norm_apply(x2, weight, None, eps, True, rk).view(*lead, x.shape[-1])


# ---- norm of a residual sum, with dropout on the branch ----------------------------------------------------------------
ADD_NORM_MAX_COLS = 8192  # a row lives in the registers of one block


def add_norm_reference(x, residual, weight, bias, eps: float, rms: bool, threshold: int, seed):
    """The PyTorch statement of ``add_layer_norm`` / ``add_rms_norm``: (norm of the sum, sum), in fp32 (fp64 for fp64
    inputs), each rounded once."""
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    branch = x.to(wide)
    if threshold:
        keep = dropout_keep_mask(x.shape, threshold / 65536.0, seed, x.device)
        branch = torch.where(keep, branch * inverse_keep(threshold), torch.zeros((), dtype=wide, device=x.device))
    total = residual.to(wide) + branch
    if rms:
        y = total * torch.rsqrt(total.pow(2).mean(dim=-1, keepdim=True) + eps) * weight.to(wide)
    else:
        y = F.layer_norm(total, (x.shape[-1],), weight.to(wide), None if bias is None else bias.to(wide), eps)
    return y.to(x.dtype), total.to(x.dtype)


_P, _LL, _I, _F = _lib.c_void_p, _lib.c_ll, _lib.c_int, _lib.c_float
_add_norm_fwd = _lib.bind("db200_add_norm_fwd", _P, _LL, _P, _LL, _P, _P, _P, _P, _P, _P, _LL, _I, _F, _I, *SEED_TYPES, _P)
_add_norm_bwd = _lib.bind("db200_add_norm_bwd", _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _I, _LL, _I, _I,
                          *SEED_TYPES, _P)


@functools.lru_cache(maxsize=1024)
def _parts(rows: int, cols: int) -> int:
    return int(_lib.lib().db200_add_norm_parts(_LL(rows), _I(cols)))


_address = lambda t: None if t is None else t.data_ptr()  # noqa: E731


def add_norm_forward(x, residual, weight, bias, eps: float, rms: bool, threshold: int, seed):
    """(y, total, stats): fp32 ``stats`` are the rows' reciprocal deviations and, for LayerNorm, their means behind them."""
    cols = x.shape[-1]
    rows = x.numel() // cols
    if not kernel_ok(x):
        y, total = add_norm_reference(x, residual, weight, bias, eps, rms, threshold, seed)
        t = total.float().reshape(rows, cols)
        if rms:
            return y, total, torch.rsqrt(t.pow(2).mean(-1) + eps)
        return y, total, torch.cat((torch.rsqrt(t.var(-1, unbiased=False) + eps), t.mean(-1)))
    with on_device(x):
        x2, ldx = rows_view(x)
        r2, ldr = rows_view(residual)
        w, b = weight.contiguous(), (None if bias is None else bias.contiguous())
        total = torch.empty_like(x, memory_format=torch.contiguous_format)
        y = torch.empty_like(total)
        stats = torch.empty((1 if rms else 2) * rows, dtype=torch.float32, device=x.device)
        rstd = stats.data_ptr()
        address, value = seed_args(seed)
        _add_norm_fwd(x2.data_ptr(), ldx, r2.data_ptr(), ldr, w.data_ptr(), _address(b), total.data_ptr(), y.data_ptr(),
                      None if rms else rstd + 4 * rows, rstd, rows, cols, eps, DTYPE_CODES[x.dtype], address, value,
                      threshold, inverse_keep(threshold), _lib.raw_stream())
    return y, total, stats


def add_norm_backward(dy, dtotal, total, w, stats, rms: bool, threshold: int, seed, has_bias: bool, w_grad, b_grad):
    """(dx, dresidual, dweight, dbias): ``dresidual`` is ``None`` where it equals ``dx`` (no dropout), a parameter gradient where
    it went into its fp32 buffer. ``dtotal`` may be ``None``."""
    cols = total.shape[-1]
    rows, dev, dtype = total.numel() // cols, total.device, total.dtype
    if not kernel_ok(total):
        t, g = total.float().reshape(rows, cols), dy.float().reshape(rows, cols)
        rstd = stats[:rows, None]
        xh = (t if rms else t - stats[rows:, None]) * rstd
        gw = g * w.float()
        d = rstd * (gw - (0 if rms else gw.mean(-1, keepdim=True)) - xh * (gw * xh).mean(-1, keepdim=True))
        d = d.view(total.shape) if dtotal is None else d.view(total.shape) + dtotal.float()
        dw, db = (g * xh).sum(0).to(w.dtype), g.sum(0).to(w.dtype) if has_bias else None
        if not threshold:
            return d.to(dtype), None, dw, db
        keep = dropout_keep_mask(total.shape, threshold / 65536.0, seed, dev)
        return (d * keep * inverse_keep(threshold)).to(dtype), d.to(dtype), dw, db
    with on_device(total):
        dy = dy.contiguous()
        dtotal = None if dtotal is None else dtotal.contiguous()
        dx = torch.empty_like(total)
        dres = torch.empty_like(total) if threshold else None
        parts = torch.empty((2 if has_bias else 1) * _parts(rows, cols) * cols, dtype=torch.float32, device=dev)
        dw = torch.empty_like(w) if w_grad is None else None
        db = torch.empty(cols, dtype=dtype, device=dev) if has_bias and b_grad is None else None
        rstd = stats.data_ptr()
        address, value = seed_args(seed)
        _add_norm_bwd(dy.data_ptr(), total.data_ptr(), _address(dtotal), w.data_ptr(), None if rms else rstd + 4 * rows, rstd,
                      dx.data_ptr(), _address(dres), parts.data_ptr(), _address(dw), _address(w_grad), _address(db),
                      _address(b_grad), int(has_bias), rows, cols, DTYPE_CODES[dtype], address, value, threshold,
                      inverse_keep(threshold), _lib.raw_stream())
    return dx, dres, dw, db


class _AddNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps, rms, threshold, seed):
        held = isinstance(seed, torch.Tensor)
        y, total, stats = add_norm_forward(x, residual, weight, bias, eps, rms, threshold, seed)
        ctx.save_for_backward(total, weight.contiguous(), stats, seed if held else None)
        ctx.refs = (weight, bias)  # (their gradient buffers)
        ctx.meta = (rms, threshold, None if held else seed)
        ctx.set_materialize_grads(False)
        return y, total

    @staticmethod
    def backward(ctx, dy, dtotal):
        if torch.is_grad_enabled():  # (a second derivative is refused when it is asked for)
            return _add_norm_backward_once(ctx, dy, dtotal)
        return _add_norm_backward(ctx, dy, dtotal)


def _add_norm_backward(ctx, dy, dtotal):
    if dy is None and dtotal is None:
        return (None,) * 8
    total, w, stats, seed = ctx.saved_tensors
    weight, bias = ctx.refs
    rms, threshold, value = ctx.meta
    has_bias = bias is not None and bias.requires_grad
    w_grad = getattr(weight, "main_grad", None) if weight.requires_grad else None
    b_grad = getattr(bias, "main_grad", None) if has_bias else None
    dx, dres, dw, db = add_norm_backward(torch.zeros_like(total) if dy is None else dy, dtotal, total, w, stats, rms, threshold,
                                         value if seed is None else seed, has_bias, w_grad, b_grad)
    return dx, (dx if dres is None else dres), (dw if weight.requires_grad else None), db, None, None, None, None


_add_norm_backward_once = torch.autograd.function.once_differentiable(_add_norm_backward)


def _buffer_ok(param) -> bool:
    g = None if param is None or not param.requires_grad else getattr(param, "main_grad", None)
    return g is None or (g.dtype == torch.float32 and g.is_contiguous())


def _add_norm(x, residual, weight, bias, eps: float, rms: bool, dropout_p: float, seed, training: bool):
    check_pair(x, residual)
    if x.dim() < 1 or not x.is_floating_point():
        raise ValueError(f"the norm needs a floating tensor with at least one dimension, got {x.dtype} of shape {tuple(x.shape)}.")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and (t.shape != x.shape[-1:] or t.device != x.device):
            raise ValueError(f"{name} must have shape ({x.shape[-1]},) on {x.device}, got {tuple(t.shape)} on {t.device}.")
    threshold = dropout_threshold(dropout_p) if training else 0
    if threshold:
        if seed is None:
            raise ValueError("dropout_p > 0 needs a seed (ops.dropout.draw_seed).")
        check_seed(seed, x.device)
    else:
        seed = 0
    if (kernel_ok(x) and x.shape[-1] <= ADD_NORM_MAX_COLS and weight.dtype == x.dtype
            and (bias is None or bias.dtype == x.dtype) and _buffer_ok(weight) and _buffer_ok(bias)):
        if torch.compiler.is_compiling():  # (no gradient buffers under a compiler: see ops/linear.py:linear)
            from . import library

            seed = seed_tensor(seed, x.device) if threshold else None
            return library.add_norm(x, residual, weight, bias, seed, threshold, float(eps), rms)[:2]
        return _AddNorm.apply(x, residual, weight, bias, float(eps), rms, threshold, seed)
    return add_norm_reference(x, residual, weight, bias, float(eps), rms, threshold, seed)


def add_layer_norm(x, residual, weight, bias, eps: float, *, dropout_p: float = 0.0, seed=None, training: bool = True):
    """``(y, total)`` with ``total = residual + dropout(x)`` and ``y = LayerNorm(total)`` over the last dim, in one pass.

    ``x`` and ``residual`` have one shape, type and device; ``bias`` may be ``None``. The statistics are fp32 and those of the
    unrounded sum. ``dropout_p`` and ``seed`` as in :func:`deberta_b200.ops.dropout.dropout`; without dropout no seed is
    needed. bf16, fp16 and fp32 CUDA tensors whose parameters have their type run the kernels, up to 8192 columns; the
    parameter gradients are summed in a fixed order, into ``main_grad`` where the parameter has one."""
    return _add_norm(x, residual, weight, bias, eps, False, dropout_p, seed, training)


def add_rms_norm(x, residual, weight, eps: float, *, dropout_p: float = 0.0, seed=None, training: bool = True):
    """``(y, total)`` with ``total = residual + dropout(x)`` and ``y = RMSNorm(total)``; see :func:`add_layer_norm`."""
    return _add_norm(x, residual, weight, None, eps, True, dropout_p, seed, training)
