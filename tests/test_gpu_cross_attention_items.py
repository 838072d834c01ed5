"""GPU tests of the attention's kernels where every CTA works on several items in turn.

A B200 has 148 SMs; the forward keeps two CTAs on each, the backward one.  Here each launch
has several hundred items (row tiles, or key tiles), of sequences without keys, with one
key tile and with several, in changing order, so that the rings, sums, statistics and
barriers that go on from one item to the next are used again and again.  Values and bounds
are the oracle's, as in test_gpu_cross_attention.py.
"""

from __future__ import annotations

import pytest
import torch

import conditioning_oracle as oracle

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16

SIZES = [
    # b, lq, lk, h, hkv, d: row tiles x head groups x b items of the forward and dQ, key tiles x hkv x b of dK and dV
    (110, 130, 300, 4, 4, 64),  # 880, 1320
    (90, 129, 270, 6, 2, 40),   # 720 of 126 rows (three heads each), 540
    (70, 257, 261, 2, 2, 128),  # 420, 420
    (80, 140, 140, 5, 5, 96),   # 800, 800
    (110, 256, 77, 4, 4, 64),   # 880, 440: one key tile
    (90, 130, 128, 4, 2, 128),  # 540, 180: one key tile
    (800, 16, 40, 1, 1, 8),     # 800, 800: one key tile
    (800, 3, 150, 1, 1, 64),    # 800, 1600: few rows, but too many sequences to split
]


def _lengths(kind, b, lk, g):
    """How many keys each sequence has: all short (one key tile, or none), or any length."""
    short = torch.randint(1, min(lk, 128) + 1, (b,), generator=g, dtype=torch.int32)
    if kind == "short":
        return short
    any_length = torch.randint(0, lk + 1, (b,), generator=g, dtype=torch.int32)
    pick = torch.randint(0, 4, (b,), generator=g)
    return torch.where(pick == 0, 0, torch.where(pick == 1, short, torch.where(pick == 2, any_length, lk))).int()


def _bounds_hold(got, want):
    for name, x in got.items():
        exact, bound = want[name]
        assert torch.isfinite(x).all(), name
        worst = oracle.excess(x, exact, bound)
        assert worst <= 1.0, f"{name}: {worst:.3f} of its bound"


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("kind", ["short", "mixed", "mask"])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_many_items_a_cta(cuda, size, kind, dtype):
    from fp8_b200 import _lib
    from fp8_b200.cross_attention import cross_attention

    b, lq, lk, h, hkv, d = size
    g = torch.Generator().manual_seed(sum(size))
    new = lambda *s: torch.randn(*s, generator=g).to(dtype)  # noqa: E731
    q, k, v, dout = new(b, lq, h, d), new(b, lk, hkv, d), new(b, lk, hkv, d), new(b, lq, h, d)
    lengths, mask = _lengths(kind, b, lk, g), None
    if kind == "mask":
        mask = torch.rand(b, lk, generator=g) < torch.rand(b, 1, generator=g)
        mask[::7] = False
    want = oracle.cross_attention(q, k, v, dout, lengths, mask)
    inputs = [t.to(cuda).requires_grad_(True) for t in (q, k, v)]
    lengths, mask, dout = (None if t is None else t.to(cuda) for t in (lengths, mask, dout))
    first = None
    for _ in range(3):  # the same bits every time
        o = cross_attention(*inputs, lengths, mask)
        got = dict(zip(("o", "dq", "dk", "dv"), (o.detach(), *torch.autograd.grad(o, inputs, dout))))
        if first is None:
            first = got
        assert all(torch.equal(got[n], first[n]) for n in got)
    _bounds_hold(first, want)
    with torch.no_grad():
        assert torch.equal(cross_attention(*inputs, lengths, mask), first["o"])
    assert _lib.device_error() == 0
