"""Attention of a set of queries over an encoder's states of another length.

``o_i = sum_j softmax_j(scale q_i . k_j) v_j`` with the queries of an image (or one
new token) on one side and the keys and values projected from a prompt's states on
the other.  Forward and backward run on the kernels of ``csrc/cross_attention.cuh``;
the scores are never stored.

Tensors are ``[batch, tokens, heads, head_dim]`` in bfloat16 or float16, as a
projection's output unflattens to (no head transposes); any strides are taken, those
the kernels cannot load from are copied once.  ``head_dim`` is a multiple of 8 up to
128.  Several query heads may share a key head (grouped heads).  ``key_lengths`` and
``key_mask`` say which keys each sequence has; a sequence left with none gets zeros,
and no gradient flows from it.
"""

from __future__ import annotations

import math
from ctypes import byref

import torch

from . import _lib
from .ops import DTYPE_CODES, _call_on, _require_cuda

MAX_HEAD_DIM = 128


def _loadable(t: torch.Tensor) -> torch.Tensor:
    """``t``, or a copy of it in rows, if the kernels' loads cannot take its strides or address."""
    fits = t.data_ptr() % 16 == 0 and t.stride(3) == 1
    for n, s in zip(t.shape[:3], t.stride()[:3]):
        fits = fits and (n == 1 or (s % 8 == 0 and s > 0))
    return t if fits else t.clone(memory_format=torch.contiguous_format)


def _strides(t: torch.Tensor | None) -> tuple[int, int, int]:
    return (0, 0, 0) if t is None else t.stride()[:3]


def _check(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, key_lengths: torch.Tensor | None,
           key_mask: torch.Tensor | None) -> torch.device:
    dev = _require_cuda(q, k, v, *(t for t in (key_lengths, key_mask) if t is not None))
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
        raise RuntimeError(f"cross attention: q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} are not "
                           "[batch, tokens, heads, head_dim] of one batch and head size")
    if q.dtype not in (torch.bfloat16, torch.float16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise RuntimeError(f"cross attention: q, k and v must all be bfloat16 or all float16, got {q.dtype}, "
                           f"{k.dtype}, {v.dtype}")
    d, heads, kv_heads = q.shape[3], q.shape[2], k.shape[2]
    if d % 8 != 0 or not 8 <= d <= MAX_HEAD_DIM:
        raise RuntimeError(f"cross attention: head_dim must be a multiple of 8 up to {MAX_HEAD_DIM}, got {d}")
    if kv_heads == 0 or heads == 0 or heads % kv_heads != 0:
        raise RuntimeError(f"cross attention: {heads} heads are not a multiple of {kv_heads} key heads")
    if key_lengths is not None and (key_lengths.dtype not in (torch.int32, torch.int64)
                                    or tuple(key_lengths.shape) != (q.shape[0],)):
        raise RuntimeError(f"cross attention: key_lengths must be int32 or int64 [{q.shape[0]}], got "
                           f"{key_lengths.dtype} {tuple(key_lengths.shape)}")
    if key_mask is not None and (key_mask.dtype != torch.bool or tuple(key_mask.shape) != (q.shape[0], k.shape[1])):
        raise RuntimeError(f"cross attention: key_mask must be bool [{q.shape[0]}, {k.shape[1]}], got "
                           f"{key_mask.dtype} {tuple(key_mask.shape)}")
    return dev


def _args(q, k, v, o, lse, key_lengths, key_mask, scale, dout=None, dq=None, dk=None, dv=None):
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    tensors = (q, k, v, o, dout, dq, dk, dv)
    return _lib.CrossAttentionArgs(
        ptr(q), ptr(k), ptr(v), ptr(o), ptr(lse), ptr(dout), ptr(dq), ptr(dk), ptr(dv),
        *(_strides(t) for t in tensors), ptr(key_lengths), ptr(key_mask),
        0 if key_mask is None else key_mask.stride(0), q.shape[0], q.shape[1], k.shape[1], q.shape[2], k.shape[2],
        q.shape[3], DTYPE_CODES[q.dtype], scale)


def _masks(key_lengths, key_mask):
    if key_lengths is not None:
        key_lengths = key_lengths.to(torch.int32).contiguous()
    if key_mask is not None and key_mask.stride(1) != 1:
        key_mask = key_mask.contiguous()
    return key_lengths, key_mask


def _launch(dev: torch.device, name: str, args, backward: int) -> None:
    ws_bytes = _lib.load().fp8_cross_attention_workspace_bytes(byref(args), backward)
    ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8) if ws_bytes else None
    _call_on(dev, name, byref(args), 0 if ws is None else ws.data_ptr(), ws_bytes)


def _fwd(q, k, v, key_lengths, key_mask, scale: float, want_lse: bool):
    dev = _check(q, k, v, key_lengths, key_mask)
    b, lq, h, d = q.shape
    o = torch.empty(b, lq, h, d, device=dev, dtype=q.dtype)
    lse = torch.empty(b, h, lq, device=dev, dtype=torch.float32) if want_lse else None
    if o.numel() == 0 or k.shape[1] == 0:
        o.zero_()
        return o, lse if lse is None else lse.fill_(-math.inf)
    q, k, v = _loadable(q), _loadable(k), _loadable(v)
    key_lengths, key_mask = _masks(key_lengths, key_mask)
    _launch(dev, "fp8_cross_attention_fwd", _args(q, k, v, o, lse, key_lengths, key_mask, scale), 0)
    return o, lse


def _bwd(q, k, v, o, lse, dout, key_lengths, key_mask, scale: float, dk: torch.Tensor, dv: torch.Tensor):
    """dq; writes dk and dv."""
    dev = _check(q, k, v, key_lengths, key_mask)
    if dout.shape != o.shape or dout.dtype != q.dtype:
        raise RuntimeError(f"cross attention backward: dout {tuple(dout.shape)} {dout.dtype} does not match the "
                           f"output {tuple(o.shape)} {q.dtype}")
    dq = torch.empty(q.shape, device=dev, dtype=q.dtype)
    if q.numel() == 0 or k.shape[1] == 0:
        dk.zero_()
        dv.zero_()
        return dq.zero_()
    q, k, v, o, dout = (_loadable(t) for t in (q, k, v, o, dout))
    key_lengths, key_mask = _masks(key_lengths, key_mask)
    _launch(dev, "fp8_cross_attention_bwd",
            _args(q, k, v, o, lse, key_lengths, key_mask, scale, dout, dq, dk, dv), 1)
    return dq


@torch.library.custom_op("fp8_b200::cross_attention_fwd", mutates_args=())
def cross_attention_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, key_lengths: torch.Tensor | None,
                        key_mask: torch.Tensor | None, scale: float) -> tuple[torch.Tensor, torch.Tensor]:
    """-> (o [B, Lq, H, D], lse [B, H, Lq] fp32)."""
    return _fwd(q, k, v, key_lengths, key_mask, scale, True)


@cross_attention_fwd.register_fake
def _(q, k, v, key_lengths, key_mask, scale):
    b, lq, h, d = q.shape
    return q.new_empty(b, lq, h, d), q.new_empty(b, h, lq, dtype=torch.float32)


@torch.library.custom_op("fp8_b200::cross_attention_bwd", mutates_args=())
def cross_attention_bwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor, lse: torch.Tensor,
                        dout: torch.Tensor, key_lengths: torch.Tensor | None, key_mask: torch.Tensor | None,
                        scale: float) -> tuple[torch.Tensor, torch.Tensor]:
    """-> (dq [B, Lq, H, D], dkv [B, Lk, 2, Hkv, D])."""
    dkv = _empty_kv(k)
    return _bwd(q, k, v, o, lse, dout, key_lengths, key_mask, scale, dkv[:, :, 0], dkv[:, :, 1]), dkv


@cross_attention_bwd.register_fake
def _(q, k, v, o, lse, dout, key_lengths, key_mask, scale):
    return q.new_empty(q.shape), _empty_kv(k)


def _empty_kv(k: torch.Tensor) -> torch.Tensor:
    b, lk, hkv, d = k.shape
    return k.new_empty(b, lk, 2, hkv, d)


class CrossAttention(torch.autograd.Function):
    """``apply(q, k, v, ...)``, or ``apply(q, kv, None, ...)`` with keys and values packed ``[B, Lk, 2, Hkv, D]``."""

    @staticmethod
    def forward(ctx, q, k, v, key_lengths, key_mask, scale: float):
        kk, vv = k.unbind(2) if v is None else (k, v)
        if torch.compiler.is_compiling():
            o, lse = cross_attention_fwd(q, kk, vv, key_lengths, key_mask, scale)
        else:
            o, lse = _fwd(q, kk, vv, key_lengths, key_mask, scale, True)
        ctx.save_for_backward(q, k, v, o, lse, key_lengths, key_mask)
        ctx.scale = scale
        return o

    @staticmethod
    def backward(ctx, dout):
        q, k, v, o, lse, key_lengths, key_mask = ctx.saved_tensors
        kk, vv = k.unbind(2) if v is None else (k, v)
        if torch.compiler.is_compiling():
            dq, dkv = cross_attention_bwd(q, kk, vv, o, lse, dout, key_lengths, key_mask, ctx.scale)
        else:
            dkv = _empty_kv(kk)
            dq = _bwd(q, kk, vv, o, lse, dout, key_lengths, key_mask, ctx.scale, dkv[:, :, 0], dkv[:, :, 1])
        dk, dv = (dkv, None) if v is None else dkv.unbind(2)
        return dq, dk, dv, None, None, None


def _attend(q, k, v, key_lengths, key_mask, scale: float | None):
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else float(scale)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or (v is not None and v.requires_grad)):
        return CrossAttention.apply(q, k, v, key_lengths, key_mask, scale)
    kk, vv = k.unbind(2) if v is None else (k, v)
    if torch.compiler.is_compiling():
        return cross_attention_fwd(q, kk, vv, key_lengths, key_mask, scale)[0]
    return _fwd(q, kk, vv, key_lengths, key_mask, scale, False)[0]


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, key_lengths: torch.Tensor | None = None,
                    key_mask: torch.Tensor | None = None, scale: float | None = None) -> torch.Tensor:
    """Softmax attention of ``q [B, Lq, H, D]`` over ``k, v [B, Lk, Hkv, D]`` -> ``[B, Lq, H, D]``.

    ``key_lengths`` (int ``[B]``): sequence b has keys ``0 .. key_lengths[b] - 1``.  ``key_mask`` (bool
    ``[B, Lk]``): True where a key is kept.  Both may be given.  ``scale``: ``1 / sqrt(D)`` if None.  Query head
    h reads key head ``h // (H // Hkv)``."""
    return _attend(q, k, v, key_lengths, key_mask, scale)


def cross_attention_packed(q: torch.Tensor, kv: torch.Tensor, key_lengths: torch.Tensor | None = None,
                           key_mask: torch.Tensor | None = None, scale: float | None = None) -> torch.Tensor:
    """:func:`cross_attention` with keys and values side by side, ``kv [B, Lk, 2, Hkv, D]`` (one projection of
    the encoder's states); the gradient of ``kv`` comes in one tensor, without a stack."""
    if kv.dim() != 5 or kv.shape[2] != 2:
        raise RuntimeError(f"cross attention: kv must be [batch, tokens, 2, kv_heads, head_dim], got {tuple(kv.shape)}")
    return _attend(q, kv, None, key_lengths, key_mask, scale)


__all__ = ["cross_attention", "cross_attention_packed", "cross_attention_fwd", "cross_attention_bwd",
           "CrossAttention", "MAX_HEAD_DIM"]
