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


@pytest.mark.parametrize("lengths", ["all", "mixed"])
@pytest.mark.parametrize("size", [(2, 200, 2048, 4, 2, 64), (1, 130, 4096, 2, 2, 128), (2, 300, 1021, 4, 4, 80),
                                  (3, 260, 120, 4, 4, 64)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("std,values", [(2.0**-10, 1.0), (2.0**-14, 1.0), (1.0, 1.0), (2.0**9, 16.0)])
def test_float16_gradients_of_any_size(cuda, std, values, size, lengths):
    """Gradients of a mean loss, of one scaled against underflow, and of large values.  Beside the outputs' own rounding
    (to steps of 2^-24 where they are small) each score gradient is off by at most 2^-11 of itself for its rounding and
    as much for delta's, independently of the others: less than 2^-10 of a gradient's norm.  (A score gradient of
    2^-21 that is rounded to steps of 2^-24 is off by a thirtieth.)"""
    from fp8_b200.cross_attention import cross_attention

    b, lq, lk, h, hkv, d = size
    g = torch.Generator().manual_seed(sum(size))
    new = lambda std, *s: (torch.randn(*s, generator=g) * std).to(FP16)  # noqa: E731
    q, k, v, dout = new(1, b, lq, h, d), new(1, b, lk, hkv, d), new(values, b, lk, hkv, d), new(std, b, lq, h, d)
    dout[:, ::5] *= 2.0**-4  # rows of smaller gradients
    count = None
    if lengths == "mixed":
        count = torch.randint(lk // 2, lk + 1, (b,), generator=g, dtype=torch.int32)
        v[torch.arange(lk) >= count[:, None]] = torch.inf  # what is not kept does not set the scale
    want = oracle.cross_attention(q, k, v, dout, count)
    inputs = [t.to(cuda).requires_grad_(True) for t in (q, k, v)]
    o = cross_attention(*inputs, None if count is None else count.to(cuda))
    for name, got in zip(("dq", "dk", "dv"), torch.autograd.grad(o, inputs, dout.to(cuda))):
        exact = want[name][0]
        if exact.abs().max() > 65504:
            continue  # not a float16 value
        assert torch.isfinite(got).all(), name
        rounded = _error(exact.to(FP16), exact)
        assert _error(got, exact) <= rounded + 2.0**-10, (name, rounded)
