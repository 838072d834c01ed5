"""Dropout whose mask comes from a counter and is never stored.

``y = keep * x / (1 - p) (+ residual)``: element ``e`` (of the tensor in logical,
row-major order) is kept by a rule on ``(seed, e)`` alone, the one the fused
group norm's dropout draws from (include/fp8ops.h, ``fp8_dropout``), so the
backward makes the mask again.  ``seed`` is an int64 device scalar, read when the
kernel runs: a captured CUDA graph draws a new mask on each replay if the caller
advances it.
"""

from __future__ import annotations

import torch

from .ops import DTYPE_CODES, _call_on, _require_cuda


def _check(x: torch.Tensor, residual: torch.Tensor | None, p: float, seed: torch.Tensor) -> torch.device:
    dev = _require_cuda(x, seed) if residual is None else _require_cuda(x, seed, residual)
    if x.dtype not in DTYPE_CODES:
        raise RuntimeError(f"dropout: expected a bfloat16, float16 or float32 tensor, got {x.dtype}")
    if not 0.0 <= p <= 1.0:
        raise RuntimeError(f"dropout: p must be in [0, 1], got {p}")
    if seed.dtype != torch.int64 or seed.numel() != 1:
        raise RuntimeError(f"dropout: seed must be one int64 value, got {seed.numel()} of {seed.dtype}")
    if residual is not None and (residual.dtype != x.dtype or residual.shape != x.shape):
        raise RuntimeError(f"dropout: residual {tuple(residual.shape)} {residual.dtype} does not match "
                           f"{tuple(x.shape)} {x.dtype}")
    return dev


def _apply(x: torch.Tensor, residual: torch.Tensor | None, p: float, seed: torch.Tensor) -> torch.Tensor:
    dev = _check(x, residual, p, seed)
    x = x.contiguous()
    y = torch.empty_like(x)
    if residual is not None:
        residual = residual.contiguous()
    _call_on(dev, "fp8_dropout", x.data_ptr(), 0 if residual is None else residual.data_ptr(), y.data_ptr(),
             DTYPE_CODES[x.dtype], x.numel(), p, seed.data_ptr())
    return y


@torch.library.custom_op("fp8_b200::dropout", mutates_args=())
def dropout_op(x: torch.Tensor, residual: torch.Tensor | None, p: float, seed: torch.Tensor) -> torch.Tensor:
    """-> y, contiguous, in x's dtype."""
    return _apply(x, residual, p, seed)


@dropout_op.register_fake
def _(x, residual, p, seed):
    return torch.empty_like(x, memory_format=torch.contiguous_format)


def _run(x, residual, p, seed):
    return (dropout_op if torch.compiler.is_compiling() else _apply)(x, residual, p, seed)


class Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p: float, seed):
        ctx.save_for_backward(seed)
        ctx.p = p
        ctx.has_residual = residual is not None
        return _run(x, residual, p, seed)

    @staticmethod
    def backward(ctx, dy):
        (seed,) = ctx.saved_tensors
        dx = _run(dy, None, ctx.p, seed) if ctx.needs_input_grad[0] else None
        return dx, dy if ctx.has_residual else None, None, None


def dropout_add(x: torch.Tensor, residual: torch.Tensor | None, p: float, seed: torch.Tensor) -> torch.Tensor:
    """``residual + dropout_p(x)`` (``dropout_p(x)`` without a residual), rounded once to ``x``'s dtype."""
    if torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad)):
        return Dropout.apply(x, residual, float(p), seed)
    return _run(x, residual, float(p), seed)


def dropout(x: torch.Tensor, p: float, seed: torch.Tensor) -> torch.Tensor:
    """``x`` with each element dropped with probability ``p`` and the others scaled by ``1 / (1 - p)``."""
    return dropout_add(x, None, p, seed)


__all__ = ["dropout", "dropout_add", "dropout_op", "Dropout"]
