"""GPU tests of how much of the attention's precision is left, on the norm of its outputs.

The bounds of test_gpu_cross_attention.py hold element by element and grant every rounding
its worst case; these compare the error of a whole output with what its own rounding costs.
"""

from __future__ import annotations

import pytest
import torch

import conditioning_oracle as oracle

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def _error(got, exact):
    return ((got.detach().cpu().double() - exact).norm() / exact.norm()).item()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("size", [(1, 1, 1024, 4, 4, 64), (32, 1, 2000, 8, 2, 128), (3, 16, 4097, 2, 2, 80),
                                  (400, 1, 300, 2, 2, 64)], ids=lambda s: "x".join(map(str, s)))
def test_few_queries_lose_only_the_outputs_rounding(cuda, size, dtype):
    """A weight is off by at most 2^-16 of itself (two values of the type, 32-bit exponentials), independently of the
    others; beside the output's rounding of about 1.6e-3 (bf16) or 2e-4 (fp16) that adds less than 1 %.  A weight
    rounded once to the type adds over 25 %."""
    from fp8_b200.cross_attention import cross_attention

    b, lq, lk, h, hkv, d = size
    g = torch.Generator().manual_seed(sum(size))
    q, k, v = (torch.randn(*s, generator=g).to(dtype) for s in ((b, lq, h, d), (b, lk, hkv, d), (b, lk, hkv, d)))
    lengths = torch.randint(lk // 2, lk + 1, (b,), generator=g, dtype=torch.int32)
    exact = oracle.cross_attention(q, k, v, None, lengths)["o"][0]
    got = cross_attention(q.to(cuda), k.to(cuda), v.to(cuda), lengths.to(cuda))
    assert _error(got, exact) <= 1.02 * _error(exact.to(dtype), exact)
