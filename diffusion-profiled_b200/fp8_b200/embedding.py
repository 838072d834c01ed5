"""Token embedding with scaling, and its gradient by sorted tokens.

``y_i = scale * W[id_i]``; the gradient ``dW_v = scale * sum of dy_i over the tokens
with id v`` is dense, summed in fp32 in an order that the ids alone fix (no float
atomics): the same call gives the same bits.
"""

from __future__ import annotations

import torch

from . import _lib
from .ops import DTYPE_CODES, _call_on, _require_cuda


def _check(ids: torch.Tensor, other: torch.Tensor, *dtypes: torch.dtype) -> torch.device:
    dev = _require_cuda(ids, other)
    if ids.dtype not in (torch.int64, torch.int32):
        raise RuntimeError(f"embedding: ids must be int64 or int32, got {ids.dtype}")
    for d in dtypes:
        if d not in DTYPE_CODES:
            raise RuntimeError(f"embedding: expected bfloat16, float16 or float32, got {d}")
    return dev


def _fwd(ids: torch.Tensor, weight: torch.Tensor, scale: float, dtype: torch.dtype) -> torch.Tensor:
    dev = _check(ids, weight, weight.dtype, dtype)
    if weight.dim() != 2 or weight.shape[0] == 0 or weight.shape[1] == 0:
        raise RuntimeError(f"embedding: weight must be [vocab, width], got {tuple(weight.shape)}")
    vocab, width = weight.shape
    if weight.stride(1) != 1 and width > 1:
        weight = weight.contiguous()
    ids = ids.contiguous()
    out = torch.empty(*ids.shape, width, device=dev, dtype=dtype)
    _call_on(dev, "fp8_embedding_fwd", ids.data_ptr(), ids.dtype == torch.int64, ids.numel(), weight.data_ptr(),
             DTYPE_CODES[weight.dtype], vocab, width, weight.stride(0), scale, out.data_ptr(), DTYPE_CODES[dtype])
    return out


def _bwd(ids: torch.Tensor, dout: torch.Tensor, vocab: int, scale: float, padding_idx: int,
         weight_dtype: torch.dtype) -> torch.Tensor:
    dev = _check(ids, dout, dout.dtype, weight_dtype)
    width = dout.shape[-1]
    if tuple(dout.shape[:-1]) != tuple(ids.shape):
        raise RuntimeError(f"embedding backward: dout {tuple(dout.shape)} does not match ids {tuple(ids.shape)}")
    ids, dout = ids.contiguous(), dout.contiguous()
    dw = torch.empty(vocab, width, device=dev, dtype=weight_dtype)
    n = ids.numel()
    ws_bytes = _lib.load().fp8_embedding_bwd_workspace_bytes(n, vocab, width)
    ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8)
    _call_on(dev, "fp8_embedding_bwd", ids.data_ptr(), ids.dtype == torch.int64, n, dout.data_ptr(),
             DTYPE_CODES[dout.dtype], dw.data_ptr(), DTYPE_CODES[weight_dtype], vocab, width, scale, padding_idx,
             ws.data_ptr(), ws_bytes)
    return dw


@torch.library.custom_op("fp8_b200::embedding_fwd", mutates_args=())
def embedding_fwd(ids: torch.Tensor, weight: torch.Tensor, scale: float, dtype: torch.dtype) -> torch.Tensor:
    """-> y [*ids.shape, width] in ``dtype``."""
    return _fwd(ids, weight, scale, dtype)


@embedding_fwd.register_fake
def _(ids, weight, scale, dtype):
    return weight.new_empty(*ids.shape, weight.shape[1], dtype=dtype)


@torch.library.custom_op("fp8_b200::embedding_bwd", mutates_args=())
def embedding_bwd(ids: torch.Tensor, dout: torch.Tensor, vocab: int, scale: float, padding_idx: int,
                  weight_dtype: torch.dtype) -> torch.Tensor:
    """-> dW [vocab, width] in ``weight_dtype`` (padding_idx < 0: none)."""
    return _bwd(ids, dout, vocab, scale, padding_idx, weight_dtype)


@embedding_bwd.register_fake
def _(ids, dout, vocab, scale, padding_idx, weight_dtype):
    return dout.new_empty(vocab, dout.shape[-1], dtype=weight_dtype)


class TokenEmbedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale: float, padding_idx: int, dtype):
        ctx.save_for_backward(ids)
        ctx.cfg = (weight.shape[0], scale, padding_idx, weight.dtype)
        return (embedding_fwd if torch.compiler.is_compiling() else _fwd)(ids, weight, scale, dtype)

    @staticmethod
    def backward(ctx, dout):
        (ids,) = ctx.saved_tensors
        bwd = embedding_bwd if torch.compiler.is_compiling() else _bwd
        return None, bwd(ids, dout, *ctx.cfg), None, None, None


def embed_tokens(ids: torch.Tensor, weight: torch.Tensor, scale: float = 1.0, padding_idx: int | None = None,
                 dtype: torch.dtype | None = None) -> torch.Tensor:
    """``scale * weight[ids]`` as ``dtype`` (the weight's own if None), shape ``[*ids.shape, width]``.

    ``ids``: int64 or int32.  The row of ``padding_idx`` is looked up like any other and gets no gradient
    (``nn.Embedding``); a negative one counts from the end of the vocabulary.  An id outside the vocabulary
    gives a row of zeros and sets the device error word (``_lib.device_error()`` returns 201)."""
    dtype = weight.dtype if dtype is None else dtype
    if padding_idx is None:
        pad = -1
    else:
        pad = padding_idx + weight.shape[0] if padding_idx < 0 else padding_idx
        if not 0 <= pad < weight.shape[0]:
            raise RuntimeError(f"embedding: padding_idx {padding_idx} outside a vocabulary of {weight.shape[0]}")
    if torch.is_grad_enabled() and weight.requires_grad:
        return TokenEmbedding.apply(ids, weight, float(scale), pad, dtype)
    return (embedding_fwd if torch.compiler.is_compiling() else _fwd)(ids, weight, float(scale), dtype)


__all__ = ["embed_tokens", "embedding_fwd", "embedding_bwd", "TokenEmbedding"]
