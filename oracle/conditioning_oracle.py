"""Plain 64-bit implementations of the text-conditioning operators (test infrastructure only).

Each returns the exact value of the operator on the given inputs and, for the
attention, how far a kernel with the stated roundings may be from it, element by
element:

* u is the unit roundoff of the tensors' type (2^-8 for bfloat16, 2^-11 for float16):
  every output is rounded once, |err| <= u |x|;
* the weights p_ij and the score gradients ds_ij are rounded once to the tensors'
  type for the tensor cores, so a sum over them is off by at most u times the same sum
  of absolute values; in float16 values below 2^-14 are rounded to a multiple of 2^-24
  instead;
* delta_i may be formed from the rounded output: |err| <= u sum_d |do_id o_id|;
* scores, exponentials and accumulations are 32-bit: each p_ij is off by a relative
  2^-12 at most here (|s| < 64 at 2^-22, lengths up to 2^12 at 2^-24 a step), which is
  added to u.
"""

from __future__ import annotations

import numpy as np
import torch

ROUNDOFF = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0**-24}
FP32_SLACK = 2.0**-12


def kept_keys(b: int, lk: int, key_lengths, key_mask) -> torch.Tensor:
    keep = torch.ones(b, lk, dtype=torch.bool)
    if key_lengths is not None:
        keep &= torch.arange(lk) < key_lengths.cpu()[:, None]
    if key_mask is not None:
        keep &= key_mask.cpu()
    return keep


def cross_attention(q, k, v, dout=None, key_lengths=None, key_mask=None, scale=None):
    """-> {name: (exact, bound)} for o and lse, and for dq, dk, dv if ``dout`` is given (CPU, float64)."""
    dtype = q.dtype
    u, tiny = ROUNDOFF.get(dtype, 0.0), TINY.get(dtype, 0.0)
    q, k, v = (x.detach().cpu().double() for x in (q, k, v))
    b, lq, h, d = q.shape
    lk, hkv = k.shape[1], k.shape[2]
    scale = d**-0.5 if scale is None else scale
    keep = kept_keys(b, lk, key_lengths, key_mask)
    live = keep[:, :, None, None]
    k, v = torch.where(live, k, 0.0), torch.where(live, v, 0.0)  # what is not kept is never used
    spread = lambda x: x.repeat_interleave(h // hkv, dim=2).transpose(1, 2)  # noqa: E731
    qh, kh, vh = q.transpose(1, 2), spread(k), spread(v)
    s = (qh @ kh.transpose(-1, -2) * scale).masked_fill(~keep[:, None, None, :], -torch.inf)
    lse = torch.logsumexp(s, dim=-1) if lk else torch.full((b, h, lq), -torch.inf, dtype=torch.float64)
    p = torch.where(torch.isinf(lse)[..., None], 0.0, torch.exp(s - torch.where(torch.isinf(lse), 0.0, lse)[..., None]))
    o = p @ vh
    w = u + FP32_SLACK
    fold = lambda x: x.transpose(1, 2).reshape(b, lk, hkv, h // hkv, d).sum(3)  # noqa: E731
    back = lambda x: x.transpose(1, 2)  # noqa: E731
    out = {
        "o": (back(o), back(u * o.abs() + w * (p @ vh.abs()) + tiny * (1 + vh.abs().sum(-2, keepdim=True)))),
        "lse": (lse, FP32_SLACK * (1 + torch.where(torch.isinf(lse), 0.0, lse).abs())),
    }
    if dout is None:
        return out
    g = dout.detach().cpu().double().transpose(1, 2)
    dp = g @ vh.transpose(-1, -2)
    delta = (p * dp).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    # rounding of ds itself, of p and delta inside it, and 32-bit products of |g| |v|
    ds_err = w * ds.abs() + p * (w * ((g * o).abs().sum(-1, keepdim=True)) + FP32_SLACK * (g.abs() @ vh.abs().transpose(-1, -2)))
    ds_err = ds_err + torch.where(keep[:, None, None, :], tiny, 0.0)
    p_err = w * p + torch.where(keep[:, None, None, :], tiny, 0.0)
    dq, dk, dv = ds @ kh * scale, ds.transpose(-1, -2) @ qh * scale, p.transpose(-1, -2) @ g
    one = lambda x, sums: u * x.abs() + sums + tiny  # noqa: E731
    out["dq"] = (back(dq), back(one(dq, ds_err @ kh.abs() * abs(scale))))
    dk, dv = fold(dk), fold(dv)
    out["dk"] = (dk, one(dk, fold(ds_err.transpose(-1, -2) @ qh.abs() * abs(scale))))
    out["dv"] = (dv, one(dv, fold(p_err.transpose(-1, -2) @ g.abs())))
    return out


def excess(got: torch.Tensor, exact: torch.Tensor, bound: torch.Tensor) -> float:
    """Largest |got - exact| over its bound (a value where both are equal counts 0)."""
    got = got.detach().cpu().double()
    off = (got - exact).abs()
    off = torch.where(got == exact, 0.0, off)
    worst = (off / bound.clamp_min(1e-30)).max().item() if off.numel() else 0.0
    return float("inf") if worst != worst else worst


def embedding_grad(ids: torch.Tensor, dout: torch.Tensor, vocab: int, scale: float, padding_idx: int | None):
    """-> (exact dW, sum of absolute values per element) in float64; ids outside the vocabulary add nothing."""
    ids, dout = ids.reshape(-1).cpu().long(), dout.detach().reshape(-1, dout.shape[-1]).cpu().double() * scale
    live = (ids >= 0) & (ids < vocab)
    if padding_idx is not None:
        live &= ids != padding_idx
    dw = torch.zeros(vocab, dout.shape[1], dtype=torch.float64)
    mag = torch.zeros_like(dw)
    dw.index_add_(0, ids[live], dout[live])
    mag.index_add_(0, ids[live], dout[live].abs())
    return dw, mag


def dropout_keep(seed: int, n: int, p: float) -> np.ndarray:
    """The keep rule, one 64-bit word for four elements."""
    keep = np.empty(n, dtype=bool)
    mask = (1 << 64) - 1
    for word in range((n + 3) // 4):
        z = ((seed & mask) ^ (word * 0xD1B54A32D192ED03 & mask)) + 0x9E3779B97F4A7C15 & mask
        z = (z ^ z >> 30) * 0xBF58476D1CE4E5B9 & mask
        z = (z ^ z >> 27) * 0x94D049BB133111EB & mask
        z ^= z >> 31
        for e in range(4 * word, min(n, 4 * word + 4)):
            keep[e] = (z >> (16 * (e % 4)) & 0xFFFF) >= round(p * 65536)
    return keep
