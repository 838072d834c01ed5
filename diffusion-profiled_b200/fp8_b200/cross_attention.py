"""Attention of a set of queries over an encoder's states of another length.

``o_i = sum_j softmax_j(scale q_i . k_j) v_j`` with the queries of an image (or one
new token) on one side and the keys and values projected from a prompt's states on
the other.  Forward and backward run on the kernels of ``csrc/cross_attention.cuh``
and ``csrc/cross_attention_bwd.cuh``; the scores are never stored.  The operators and
the gradient are registered by csrc/torch_ops.cpp.

Tensors are ``[batch, tokens, heads, head_dim]`` in bfloat16 or float16, as a
projection's output unflattens to (no head transposes); any strides are taken, those
the kernels cannot load from are copied once.  ``head_dim`` is a multiple of 8 up to
128.  Several query heads may share a key head (grouped heads).  ``key_lengths`` and
``key_mask`` say which keys each sequence has; a sequence left with none gets zeros,
and no gradient flows from it.
"""

from __future__ import annotations

import torch

from . import torch_ops

torch_ops.load(required=True)

MAX_HEAD_DIM = 128


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, key_lengths: torch.Tensor | None = None,
                    key_mask: torch.Tensor | None = None, scale: float | None = None) -> torch.Tensor:
    """Softmax attention of ``q [B, Lq, H, D]`` over ``k, v [B, Lk, Hkv, D]`` -> ``[B, Lq, H, D]``.

    ``key_lengths`` (int ``[B]``): sequence b has keys ``0 .. key_lengths[b] - 1``.  ``key_mask`` (bool
    ``[B, Lk]``): True where a key is kept.  Both may be given.  ``scale``: ``1 / sqrt(D)`` if None.  Query head
    h reads key head ``h // (H // Hkv)``."""
    return torch.ops.fp8_b200.cross_attention(q, k, v, key_lengths, key_mask, scale)


def cross_attention_packed(q: torch.Tensor, kv: torch.Tensor, key_lengths: torch.Tensor | None = None,
                           key_mask: torch.Tensor | None = None, scale: float | None = None) -> torch.Tensor:
    """:func:`cross_attention` with keys and values side by side, ``kv [B, Lk, 2, Hkv, D]`` (one projection of
    the encoder's states); the gradient of ``kv`` comes in one tensor, without a stack."""
    return torch.ops.fp8_b200.cross_attention(q, kv, None, key_lengths, key_mask, scale)


def cross_attention_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, key_lengths: torch.Tensor | None,
                        key_mask: torch.Tensor | None, scale: float) -> tuple[torch.Tensor, torch.Tensor]:
    """-> (o ``[B, Lq, H, D]``, lse ``[B, H, Lq]`` fp32), without a gradient."""
    return torch.ops.fp8_b200.cross_attention_fwd(q, k, v, key_lengths, key_mask, scale)


def cross_attention_bwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor, lse: torch.Tensor,
                        dout: torch.Tensor, key_lengths: torch.Tensor | None, key_mask: torch.Tensor | None,
                        scale: float) -> tuple[torch.Tensor, torch.Tensor]:
    """-> (dq ``[B, Lq, H, D]``, dkv ``[B, Lk, 2, Hkv, D]``) from the forward's o and lse."""
    return torch.ops.fp8_b200.cross_attention_bwd(q, k, v, o, lse, dout, key_lengths, key_mask, scale)


__all__ = ["cross_attention", "cross_attention_packed", "cross_attention_fwd", "cross_attention_bwd", "MAX_HEAD_DIM"]
