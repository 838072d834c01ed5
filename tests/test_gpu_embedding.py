"""GPU tests of the token embedding (fp8_b200.embedding) against 64-bit references.

Forward: one fp32 product rounded once, so |err| <= (u + 2^-24) |x| with the output
type's u (2^-8 bf16, 2^-11 fp16, 2^-24 fp32).  Gradient: n fp32 additions and a product,
|err| <= u |x| + (n + 2) 2^-24 sum |terms|, n the number of tokens with the id.
"""

from __future__ import annotations

import pytest
import torch

import conditioning_oracle as oracle

pytestmark = pytest.mark.gpu
U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _case(n, vocab, width, wdtype, dtype, kind="zipf", seed=0):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(vocab, width, generator=g).to(wdtype)
    if kind == "zipf":
        ids = (float(vocab) ** torch.rand(n, generator=g, dtype=torch.float64)).long() - 1
    elif kind == "one":
        ids = torch.full((n,), vocab // 2)
    else:
        ids = torch.randint(0, vocab, (n,), generator=g)
    return ids.clamp_(0, vocab - 1), w, torch.randn(n, width, generator=g).to(dtype)


def _check_grad(dw, ids, dout, vocab, scale, pad):
    exact, mag = oracle.embedding_grad(ids, dout, vocab, scale, pad)
    live = ids.reshape(-1)[(ids.reshape(-1) >= 0) & (ids.reshape(-1) < vocab)].long()
    count = torch.bincount(live, minlength=vocab).double()[:, None]
    tiny = 2.0**-25 if dw.dtype == FP16 else 0.0
    bound = U[dw.dtype] * exact.abs() + (count + 2) * 2.0**-24 * mag + tiny
    got = dw.cpu().double()
    off = (got - exact).abs()
    assert (off <= bound).all(), (off - bound).max().item()
    assert torch.count_nonzero(got[(count == 0).squeeze(1)]) == 0


SIZES = [(1, 1, 1), (1, 5, 8), (77, 1000, 512), (33, 7, 250), (2048, 4096, 64), (5003, 300, 777), (9856, 32768, 256),
         (70001, 120001, 40), (4097, 3, 1024)]


@pytest.mark.parametrize("n,vocab,width", SIZES)
@pytest.mark.parametrize("wdtype,dtype", [(FP32, BF16), (BF16, BF16), (FP32, FP32), (FP16, FP32), (BF16, FP16)])
def test_lookup_and_gradient(cuda, n, vocab, width, wdtype, dtype):
    from fp8_b200.embedding import embed_tokens

    ids, w, dout = _case(n, vocab, width, wdtype, dtype, seed=n + width)
    pad = int(ids[0]) if n > 40 else None
    wd = w.to(cuda).requires_grad_(True)
    out = embed_tokens(ids.to(cuda), wd, scale=1.7, padding_idx=pad, dtype=dtype)
    exact = w.double()[ids] * float(torch.tensor(1.7))
    assert out.dtype == dtype and out.shape == exact.shape
    assert ((out.detach().cpu().double() - exact).abs() <= (U[dtype] + 2.0**-24) * exact.abs()
            + (2.0**-25 if dtype == FP16 else 0.0)).all()
    out.backward(dout.to(cuda))
    assert wd.grad.dtype == wdtype
    _check_grad(wd.grad, ids, dout, vocab, float(torch.tensor(1.7)), pad)
    if pad is not None:
        assert torch.count_nonzero(wd.grad[pad]) == 0


# one launch up to 1024 tokens (of rows that are not too wide), three beyond
@pytest.mark.parametrize("kind", ["one", "uniform", "zipf"])
@pytest.mark.parametrize("n,vocab,width", [(255, 65, 777), (257, 64, 72), (1023, 63, 264), (1024, 4001, 250),
                                           (1025, 4001, 250), (2049, 1, 64), (1024, 5, 16648)])
def test_gradient_at_the_choice_of_launches(cuda, kind, n, vocab, width):
    from fp8_b200.embedding import embedding_bwd

    ids, _, dout = _case(n, vocab, width, FP32, BF16, kind, seed=n)
    ids[n // 2] = vocab  # one id outside the vocabulary adds to nothing
    got = embedding_bwd(ids.to(cuda), dout.to(cuda), vocab, 0.5, vocab - 1, FP32)
    inside = ids < vocab
    _check_grad(got, ids[inside], dout[inside], vocab, 0.5, vocab - 1)
    assert torch.equal(got, embedding_bwd(ids.to(cuda).int(), dout.to(cuda), vocab, 0.5, vocab - 1, FP32))


@pytest.mark.parametrize("kind", ["one", "uniform", "zipf"])
@pytest.mark.parametrize("n", [31, 1024, 20000])
def test_gradient_is_the_same_every_time(cuda, kind, n):
    from fp8_b200.embedding import embedding_bwd

    ids, _, dout = _case(n, 512, 96, FP32, BF16, kind, seed=n)
    ids, dout = ids.to(cuda), dout.to(cuda)
    a = embedding_bwd(ids, dout, 512, 2.0, -1, FP32)
    _check_grad(a, ids.cpu(), dout.cpu(), 512, 2.0, None)
    for _ in range(3):
        assert torch.equal(a, embedding_bwd(ids, dout, 512, 2.0, -1, FP32))


def test_shapes_types_and_strides(cuda):
    from fp8_b200.embedding import embed_tokens

    ids, w, _ = _case(60, 50, 48, FP32, FP32)
    ids, w = ids.to(cuda), w.to(cuda)
    want = w[ids.view(5, 12)]
    assert torch.equal(embed_tokens(ids.view(5, 12), w), want)
    assert torch.equal(embed_tokens(ids.view(5, 12).int(), w), want)
    assert torch.equal(embed_tokens(ids.view(12, 5).t(), w), w[ids.view(12, 5).t()])
    wide = torch.zeros(50, 101, device=cuda)
    wide[:, 3:51] = w
    assert torch.equal(embed_tokens(ids, wide[:, 3:51]), w[ids])
    assert torch.equal(embed_tokens(ids, w.t().contiguous().t()), w[ids])
    assert embed_tokens(ids[:0], w).shape == (0, 48)
    wg = w.clone().requires_grad_(True)
    embed_tokens(ids[:0], wg).sum().backward()
    assert torch.count_nonzero(wg.grad) == 0 and wg.grad.shape == w.shape
    # a gradient that arrives broadcast, and as a transposed view
    wg = w.clone().requires_grad_(True)
    out = embed_tokens(ids, wg)
    out.sum().backward()
    assert torch.equal(wg.grad, torch.bincount(ids, minlength=50).float()[:, None].expand(50, 48))


def test_padding_index_from_the_end(cuda):
    from fp8_b200.embedding import embed_tokens

    w = torch.ones(4, 8, device=cuda, requires_grad=True)
    embed_tokens(torch.tensor([3, 3, 0], device=cuda), w, padding_idx=-1).sum().backward()
    assert torch.equal(w.grad[:, 0].cpu(), torch.tensor([1.0, 0, 0, 0]))


def test_ids_outside_the_vocabulary(cuda):
    from fp8_b200 import _lib
    from fp8_b200.embedding import embed_tokens, embedding_bwd

    _lib.device_error()
    w = torch.ones(6, 16, device=cuda)
    ids = torch.tensor([0, 6, -1, 5, 2**40, -(2**40)], device=cuda)
    out = embed_tokens(ids, w)
    assert torch.equal(out[:, 0].cpu(), torch.tensor([1.0, 0, 0, 1, 0, 0]))
    assert _lib.device_error() == 201
    dw = embedding_bwd(ids, torch.ones(6, 16, device=cuda), 6, 1.0, -1, FP32)
    assert torch.equal(dw[:, 0].cpu(), torch.tensor([1.0, 0, 0, 0, 0, 1]))
    assert _lib.device_error() in (0, 201)


def test_gradient_against_differences(cuda):
    """The map is linear: along a direction the difference of the 64-bit forward is the gradient's product."""
    from fp8_b200.embedding import embed_tokens

    ids, w, dout = _case(500, 60, 32, FP32, FP32, seed=3)
    wd = w.to(cuda).requires_grad_(True)
    embed_tokens(ids.to(cuda), wd, scale=0.5).backward(dout.to(cuda))
    d = torch.randn(60, 32, generator=torch.Generator().manual_seed(1), dtype=torch.float64)
    loss = lambda x: (0.5 * x[ids] * dout.double()).sum()  # noqa: E731
    difference = (loss(w.double() + d) - loss(w.double() - d)) / 2
    along = (wd.grad.cpu().double() * d).sum()
    _, mag = oracle.embedding_grad(ids, dout, 60, 0.5, None)
    assert abs(along - difference) <= (500 * 2.0**-24 * mag * d.abs()).sum()


def test_refusals(cuda):
    from fp8_b200.embedding import embed_tokens

    w = torch.zeros(4, 8, device=cuda)
    ids = torch.zeros(3, device=cuda, dtype=torch.int64)
    for bad in (lambda: embed_tokens(ids.cpu(), w), lambda: embed_tokens(ids.float(), w),
                lambda: embed_tokens(ids, w.double()), lambda: embed_tokens(ids, w, dtype=torch.int8),
                lambda: embed_tokens(ids, w[0]), lambda: embed_tokens(ids, w, padding_idx=4),
                lambda: embed_tokens(ids, w, padding_idx=-5), lambda: embed_tokens(ids, w[:0])):
        with pytest.raises(RuntimeError):
            bad()


def test_rows_whose_offsets_pass_32_bits(cuda):
    from fp8_b200.embedding import embed_tokens, embedding_bwd

    vocab, width = 70_000, 65_536  # 4.6e9 values
    w = torch.empty(vocab, width, dtype=BF16, device=cuda)
    ids = torch.tensor([69_999, 3, 69_999, 40_001], device=cuda)
    rows = torch.randn(4, width, device=cuda).to(BF16)
    w[ids] = rows
    assert torch.equal(embed_tokens(ids, w), w[ids])
    del w
    dout = torch.randn(4, width, device=cuda).to(BF16)
    dw = embedding_bwd(ids, dout, vocab, 1.0, -1, BF16)
    assert torch.equal(dw[3], dout[1]) and torch.equal(dw[40_001], dout[3])
    assert torch.equal(dw[69_999], (dout[0].float() + dout[2].float()).to(BF16))
    assert torch.count_nonzero(dw[69_998]) == 0 and torch.count_nonzero(dw[40_000]) == 0
