"""Dropout whose mask comes from a counter and is never stored.

``y = keep * x / (1 - p) (+ residual)``: element ``e`` (of the tensor in logical,
row-major order) is kept by a rule on ``(seed, e)`` alone, the one the fused
group norm's dropout draws from (include/fp8ops.h, ``fp8_dropout``), so the
backward makes the mask again.  ``seed`` is an int64 device scalar, read when the
kernel runs: a captured CUDA graph draws a new mask on each replay if the caller
advances it.  The operator and its gradient are registered by csrc/torch_ops.cpp;
there is no second and no forward-mode derivative (both are refused).  Under
``torch.vmap`` every slice is a call of its own, whose elements are counted from 0:
with one seed all slices get one mask.
"""

from __future__ import annotations

import torch

from . import torch_ops

torch_ops.load(required=True)


def dropout_add(x: torch.Tensor, residual: torch.Tensor | None, p: float, seed: torch.Tensor) -> torch.Tensor:
    """``residual + dropout_p(x)`` (``dropout_p(x)`` without a residual), rounded once to ``x``'s dtype.

    ``x``: bfloat16, float16 or float32, ``residual`` of the same shape and dtype; ``0 <= p <= 1``; ``seed``: one
    int64 value on the device."""
    return torch.ops.fp8_b200.dropout_add(x, residual, p, seed)


def dropout(x: torch.Tensor, p: float, seed: torch.Tensor) -> torch.Tensor:
    """``x`` with each element dropped with probability ``p`` and the others scaled by ``1 / (1 - p)``."""
    return torch.ops.fp8_b200.dropout_add(x, None, p, seed)


__all__ = ["dropout", "dropout_add"]
