"""Conditioning the UNet on a prompt: its tokens' states, and the pixels' attention over them.

The reference's UNet is unconditional; these two modules are this library's own and
are built only where ``UNetConfig.prompt_vocab`` is set.  :class:`PromptEncoder` turns
token ids into states (:func:`fp8_b200.embedding.embed_tokens`, dropout, layer norm);
:class:`PromptAttention` reads them from a feature map's pixels
(:func:`fp8_b200.cross_attention.cross_attention_packed`) and adds what it found onto
the map with dropout (:func:`fp8_b200.dropout.dropout_add`).  They run on CUDA tensors
only.  The projections are ``nn.Linear``, which follows autocast, as in the UNet's own
attention blocks (its FP8 whitelist is of 3x3 convolutions); the sums with the position,
and with the map where there is no dropout, are torch's.
"""

from __future__ import annotations

import math

import torch
import torch.nn as nn

from .cross_attention import cross_attention_packed
from .dropout import dropout, dropout_add
from .embedding import embed_tokens
from .norm import fused_layer_norm_supported, layer_norm_bf16


class _Seeded(nn.Module):
    """A module whose dropout masks follow a device counter (a captured graph draws a new mask on each replay)."""

    def __init__(self, p_drop: float):
        super().__init__()
        self.p_drop = p_drop
        self.register_buffer("dropout_seed", torch.randint(0, 2**62, (), dtype=torch.int64), persistent=False)

    def _next_seed(self) -> torch.Tensor:
        seed = self.dropout_seed.clone()
        self.dropout_seed.add_(1)
        return seed


def _norm_bf16(x: torch.Tensor, norm: nn.LayerNorm) -> torch.Tensor:
    fused = x.numel() > 0 and fused_layer_norm_supported(x, norm)
    return layer_norm_bf16(x, norm) if fused else norm(x.float()).to(torch.bfloat16)


class PromptEncoder(_Seeded):
    """Token ids ``[B, L]`` (L up to ``max_tokens``) -> states ``[B, L, width]`` in bfloat16:
    ``LayerNorm(dropout(sqrt(width) * E[ids] + position))``.  ``padding_idx``: a token whose row gets no gradient."""

    def __init__(self, vocab: int, width: int, max_tokens: int, padding_idx: int | None = None, p_drop: float = 0.0):
        super().__init__(p_drop)
        self.padding_idx = padding_idx
        self.scale = math.sqrt(width)
        self.weight = nn.Parameter(torch.randn(vocab, width) / self.scale)
        self.position = nn.Parameter(0.02 * torch.randn(max_tokens, width))
        self.norm = nn.LayerNorm(width)

    def forward(self, ids: torch.Tensor) -> torch.Tensor:
        if ids.dim() != 2 or ids.shape[1] > self.position.shape[0]:
            raise RuntimeError(f"prompt: ids must be [batch, up to {self.position.shape[0]}], got {tuple(ids.shape)}")
        x = embed_tokens(ids, self.weight, self.scale, self.padding_idx, torch.bfloat16)
        x = x + self.position[: ids.shape[1]].to(torch.bfloat16)
        if self.training and self.p_drop > 0.0:
            x = dropout(x, self.p_drop, self._next_seed())
        return _norm_bf16(x, self.norm)


class PromptAttention(_Seeded):
    """``x + dropout(out(attention(q(LayerNorm(x)), kv(states))))`` over the pixels of ``x [B, C, H, W]``.

    ``states [B, L, width]``; ``lengths`` (int ``[B]``): how many of each sequence's states there are.  The output
    projection starts at zero: the map is unchanged until it is trained."""

    def __init__(self, channels: int, width: int, n_heads: int, p_drop: float = 0.0):
        super().__init__(p_drop)
        if channels % n_heads or (channels // n_heads) % 8 or channels // n_heads > 128:
            raise ValueError(f"prompt attention: {channels} channels do not make {n_heads} heads of a multiple of 8 up to 128")
        self.nh = n_heads
        self.norm = nn.LayerNorm(channels)
        self.q = nn.Linear(channels, channels, bias=False)
        self.kv = nn.Linear(width, 2 * channels, bias=False)
        self.out = nn.Linear(channels, channels, bias=False)
        nn.init.zeros_(self.out.weight)

    def forward(self, x: torch.Tensor, states: torch.Tensor, lengths: torch.Tensor | None = None) -> torch.Tensor:
        b, c, h, w = x.shape
        if states.dim() != 3 or states.shape[0] != b:
            raise RuntimeError(f"prompt attention: states must be [{b}, tokens, width], got {tuple(states.shape)}")
        d = c // self.nh
        tokens = x.flatten(2).transpose(1, 2).contiguous()  # [B, HW, C]: a view where x is channels-last
        linear_dtype = self.q.weight.dtype
        feed = lambda t: t if torch.is_autocast_enabled("cuda") else t.to(linear_dtype)  # noqa: E731
        q = self.q(feed(_norm_bf16(tokens, self.norm))).to(torch.bfloat16)
        kv = self.kv(feed(states)).to(torch.bfloat16)
        o = cross_attention_packed(q.view(b, h * w, self.nh, d), kv.view(b, states.shape[1], 2, self.nh, d), lengths)
        o = self.out(feed(o.flatten(2))).to(x.dtype)
        if self.training and self.p_drop > 0.0:
            y = dropout_add(o, tokens, self.p_drop, self._next_seed())
        else:
            y = tokens + o
        return y.transpose(1, 2).view(b, c, h, w)


__all__ = ["PromptEncoder", "PromptAttention"]
