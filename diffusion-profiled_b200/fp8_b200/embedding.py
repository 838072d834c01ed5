"""Token embedding with scaling, and its gradient by sorted tokens.

``y_i = scale * W[id_i]``; the gradient ``dW_v = scale * sum of dy_i over the tokens
with id v`` is dense, summed in fp32 in an order that the ids alone fix (no float
atomics): the same call gives the same bits.  The operator and its gradient are
registered by csrc/torch_ops.cpp.
"""

from __future__ import annotations

import torch

from . import torch_ops

torch_ops.load(required=True)


def embed_tokens(ids: torch.Tensor, weight: torch.Tensor, scale: float = 1.0, padding_idx: int | None = None,
                 dtype: torch.dtype | None = None) -> torch.Tensor:
    """``scale * weight[ids]`` as ``dtype`` (the weight's own if None), shape ``[*ids.shape, width]``.

    ``ids``: int64 or int32.  The row of ``padding_idx`` is looked up like any other and gets no gradient
    (``nn.Embedding``); a negative one counts from the end of the vocabulary.  An id outside the vocabulary
    gives a row of zeros and sets the device error word (``_lib.device_error()`` returns 201)."""
    if padding_idx is None:
        pad = -1
    else:
        vocab = weight.shape[0]
        pad = padding_idx + vocab if padding_idx < 0 else padding_idx
        if not 0 <= pad < vocab:
            raise RuntimeError(f"embedding: padding_idx {padding_idx} outside a vocabulary of {vocab}")
    return torch.ops.fp8_b200.embed_tokens(ids, weight, scale, pad, weight.dtype if dtype is None else dtype)


def embedding_fwd(ids: torch.Tensor, weight: torch.Tensor, scale: float, dtype: torch.dtype) -> torch.Tensor:
    """-> y ``[*ids.shape, width]`` in ``dtype`` (no gradient)."""
    return torch.ops.fp8_b200.embedding_fwd(ids, weight, scale, dtype)


def embedding_bwd(ids: torch.Tensor, dout: torch.Tensor, vocab: int, scale: float, padding_idx: int,
                  weight_dtype: torch.dtype) -> torch.Tensor:
    """-> dW ``[vocab, width]`` in ``weight_dtype`` (padding_idx < 0: none)."""
    return torch.ops.fp8_b200.embedding_bwd(ids, dout, vocab, scale, padding_idx, weight_dtype)


__all__ = ["embed_tokens", "embedding_fwd", "embedding_bwd"]
