"""Dropout of the backbones: torch's generator, or counter-based masks inside the kernels (``dropout_generator`` of a config)."""

from __future__ import annotations

from typing import Any

import torch
import torch.nn.functional as F

from deberta_b200.ops.dropout import draw_seed, dropout
from deberta_b200.ops.norm import add_layer_norm, add_rms_norm

__all__ = ["counter_based", "drop", "attention_seed", "drop_add_layer_norm", "drop_add_rms_norm"]


def counter_based(config: Any) -> bool:
    """Whether the model draws its masks from the counter-based generator (``ops/dropout.py``)."""
    name = str(getattr(config, "dropout_generator", None) or "torch")
    if name not in ("torch", "counter"):
        raise ValueError(f"dropout_generator must be one of: torch|counter, got {name!r}.")
    return name == "counter"


def drop(x: torch.Tensor, p: float, training: bool, counter: bool) -> torch.Tensor:
    """Dropout of ``x``; each counter-based call draws a seed from torch's generator of the device."""
    if not (training and p > 0.0):
        return x
    return dropout(x, p, draw_seed(x.device)) if counter else F.dropout(x, p, True)


def attention_seed(x: torch.Tensor, p: float, training: bool, counter: bool) -> torch.Tensor | None:
    """Seed for the attention operators' probabilities, or ``None``: torch's generator or no dropout."""
    return draw_seed(x.device) if counter and training and p > 0.0 else None


def drop_add_layer_norm(branch, residual, norm, p: float, training: bool, counter: bool) -> torch.Tensor:
    """``LayerNorm(dropout(branch) + residual)``: one kernel where the masks are counter-based."""
    if counter and training and p > 0.0 and branch.dtype == residual.dtype:
        return add_layer_norm(branch, residual, norm.weight, norm.bias, norm.eps, dropout_p=p, seed=draw_seed(branch.device))[0]
    from deberta_b200.ops.norm import layer_norm

    return layer_norm(drop(branch, p, training, counter) + residual, norm.weight, norm.bias, norm.eps)


def drop_add_rms_norm(branch, residual, norm, p: float, training: bool, counter: bool) -> torch.Tensor:
    """``RMSNorm(residual + dropout(branch))``: one kernel where the masks are counter-based."""
    if counter and training and p > 0.0 and branch.dtype == residual.dtype:
        return add_rms_norm(branch, residual, norm.weight, norm.eps, dropout_p=p, seed=draw_seed(branch.device))[0]
    return norm(residual + drop(branch, p, training, counter))
