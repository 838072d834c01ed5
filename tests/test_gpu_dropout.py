"""GPU tests of the counter-based dropout (fp8_b200.dropout).

The mask is compared bit for bit with the rule written out in Python integers.  Values:
y = keep x / (1 - p) + r with the scale rounded to 32 bits, one product, one sum and
one rounding to the type: |err| <= u |y| + 2^-22 (|x / (1 - p)| + |r|).
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

import conditioning_oracle as oracle

pytestmark = pytest.mark.gpu
U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}


def _seed(cuda, value):
    return torch.tensor(value, dtype=torch.int64, device=cuda)


@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("n", [1, 3, 8, 9, 1000, 4099, 65537])
@pytest.mark.parametrize("p,seed", [(0.1, 7), (0.5, -3), (0.9, 2**62 + 5)])
def test_values_and_gradients(cuda, n, p, seed, dtype):
    from fp8_b200.dropout import dropout, dropout_add

    g = torch.Generator().manual_seed(n)
    x, r, dy = (torch.randn(n, generator=g).to(dtype) for _ in range(3))
    keep = torch.from_numpy(oracle.dropout_keep(seed, n, p))
    xd, rd = x.to(cuda).requires_grad_(True), r.to(cuda).requires_grad_(True)
    tiny = 2.0**-25 if dtype == torch.float16 else 0.0

    def close(got, exact, parts):
        assert got.dtype == dtype
        off = (got.detach().cpu().double() - exact).abs()
        assert (off <= U[dtype] * exact.abs() + 2.0**-22 * parts + tiny).all()

    scaled = torch.where(keep, x.double() / (1 - p), 0.0)
    y = dropout(xd, p, _seed(cuda, seed))
    close(y, scaled, scaled.abs())
    assert torch.equal(y.detach().cpu() != 0, keep & (x != 0))
    y.backward(dy.to(cuda))
    dscaled = torch.where(keep, dy.double() / (1 - p), 0.0)
    close(xd.grad, dscaled, dscaled.abs())
    xd.grad = None
    y = dropout_add(xd, rd, p, _seed(cuda, seed))
    close(y, scaled + r.double(), scaled.abs() + r.double().abs())
    y.backward(dy.to(cuda))
    close(xd.grad, dscaled, dscaled.abs())
    assert torch.equal(rd.grad.cpu(), dy)


def test_ends_of_the_range(cuda):
    from fp8_b200.dropout import dropout, dropout_add

    x = torch.randn(100, device=cuda)
    assert torch.equal(dropout(x, 0.0, _seed(cuda, 1)), x)
    x[3] = torch.nan
    x[4] = torch.inf
    assert torch.count_nonzero(dropout(x, 1.0, _seed(cuda, 1))) == 0  # dropped values are not multiplied
    assert torch.equal(dropout_add(x, torch.ones_like(x), 1.0, _seed(cuda, 1)), torch.ones_like(x))
    assert dropout(x[:0], 0.5, _seed(cuda, 1)).shape == (0,)


def test_logical_order_and_alignment(cuda):
    """The mask goes by the logical index whatever the strides, and views off 16 bytes get the same values."""
    from fp8_b200.dropout import dropout, dropout_add

    x = torch.randn(37, 53, device=cuda).to(torch.bfloat16)
    want = dropout(x, 0.3, _seed(cuda, 5))
    assert torch.equal(dropout(x.t().contiguous().t(), 0.3, _seed(cuda, 5)), want)
    off = torch.zeros(37 * 53 + 1, device=cuda, dtype=torch.bfloat16)[1:].view(37, 53)
    off.copy_(x)
    assert torch.equal(dropout(off, 0.3, _seed(cuda, 5)), want)
    assert torch.equal(dropout_add(x, off, 0.3, _seed(cuda, 5)), dropout_add(x, x, 0.3, _seed(cuda, 5)))
    wide = torch.randn(1, 53, device=cuda).to(torch.bfloat16)
    assert torch.equal(dropout(wide.expand(37, 53), 0.3, _seed(cuda, 5)),
                       dropout(wide.expand(37, 53).contiguous(), 0.3, _seed(cuda, 5)))


def test_rate_and_independence(cuda):
    """Over 2^24 elements the kept share is within 5 standard deviations of 1 - p; two seeds agree on (1-p)^2 + p^2."""
    from fp8_b200.dropout import dropout

    n, p = 1 << 24, 0.25
    ones = torch.ones(n, device=cuda)
    a, b = (dropout(ones, p, _seed(cuda, s)) != 0 for s in (11, 12))
    assert abs(a.double().mean().item() - (1 - p)) < 5 * (p * (1 - p) / n) ** 0.5
    same = (1 - p) ** 2 + p**2
    assert abs((a == b).double().mean().item() - same) < 5 * (same * (1 - same) / n) ** 0.5
    for lag in (1, 4, 1024):
        assert abs((a[lag:] == a[:-lag]).double().mean().item() - same) < 6 * (same * (1 - same) / n) ** 0.5


def test_index_past_32_bits(cuda):
    """The counter is 64-bit: the mask of the last elements of a tensor of more than 2^32 is its own."""
    from fp8_b200.dropout import dropout

    n = (1 << 32) + 4096
    x = torch.ones(n, device=cuda, dtype=torch.bfloat16)
    y = dropout(x, 0.5, _seed(cuda, 3))
    tail = (y[-4096:] != 0).cpu().numpy()
    first = (1 << 32) // 4
    mask = (1 << 64) - 1
    want = np.empty(4096, dtype=bool)
    for w in range(1024):
        z = (3 ^ ((first + w) * 0xD1B54A32D192ED03 & mask)) + 0x9E3779B97F4A7C15 & mask
        z = (z ^ z >> 30) * 0xBF58476D1CE4E5B9 & mask
        z = (z ^ z >> 27) * 0x94D049BB133111EB & mask
        z ^= z >> 31
        want[4 * w: 4 * w + 4] = [(z >> (16 * e) & 0xFFFF) >= 32768 for e in range(4)]
    assert np.array_equal(tail, want)


def test_graph_replays_draw_new_masks(cuda):
    from fp8_b200.dropout import dropout

    x, seed = torch.ones(4096, device=cuda), _seed(cuda, 1)
    dropout(x, 0.5, seed)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = dropout(x, 0.5, seed)
    graph.replay()
    first = y.clone()
    seed.add_(1)
    graph.replay()
    assert torch.equal(first, dropout(x, 0.5, _seed(cuda, 1))) and torch.equal(y, dropout(x, 0.5, _seed(cuda, 2)))


def test_refusals(cuda):
    from fp8_b200.dropout import dropout, dropout_add

    x, s = torch.zeros(8, device=cuda), _seed(cuda, 0)
    for bad in (lambda: dropout(x.cpu(), 0.1, s), lambda: dropout(x, 0.1, s.cpu()), lambda: dropout(x.double(), 0.1, s),
                lambda: dropout(x, -0.1, s), lambda: dropout(x, 1.1, s), lambda: dropout(x, 0.1, s.float()),
                lambda: dropout(x, 0.1, torch.zeros(2, dtype=torch.int64, device=cuda)),
                lambda: dropout_add(x, x[:7], 0.1, s), lambda: dropout_add(x, x.half(), 0.1, s)):
        with pytest.raises(RuntimeError):
            bad()
