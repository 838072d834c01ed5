"""GPU tests of the attention over an encoder's states (fp8_b200.cross_attention).

The oracle (oracle/conditioning_oracle.py) gives each output's 64-bit value and how far
the kernels' roundings may take it, element by element; a result may be at its bound
and no further.  Sizes: one token to several tiles on both sides, one off a tile, head
sizes that fill a tile partly, grouped heads, key lengths and masks that leave keys, tiles
or whole sequences out, strides of several layouts.
"""

from __future__ import annotations

import pytest
import torch

import conditioning_oracle as oracle

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def _inputs(b, lq, lk, h, hkv, d, dtype, seed=0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    shapes = ((b, lq, h, d), (b, lk, hkv, d), (b, lk, hkv, d), (b, lq, h, d))
    return [(torch.randn(*s, generator=g) * std).to(dtype) for s in shapes]


def _masks(kind, b, lk, seed=0):
    g = torch.Generator().manual_seed(1000 + seed)
    lengths = mask = None
    if kind in ("lengths", "both"):
        lengths = torch.randint(0, lk + 1, (b,), generator=g, dtype=torch.int32)
        lengths[0] = lk
        if b > 1:
            lengths[-1] = 0
    if kind in ("mask", "both"):
        mask = torch.rand(b, lk, generator=g) < 0.6
        if b > 1:
            mask[b // 2] = False
        if lk > 300:
            mask[0, 130:260] = False  # a whole tile of 128 keys is out
    return lengths, mask


def _run(cuda, q, k, v, dout=None, lengths=None, mask=None, scale=None, packed=False):
    from fp8_b200.cross_attention import cross_attention, cross_attention_packed

    dev = lambda t: None if t is None else t.to(cuda)  # noqa: E731
    q, k, v, lengths, mask = (dev(t) for t in (q, k, v, lengths, mask))
    train = dout is not None
    q = q.requires_grad_(train)
    if packed:
        kv = torch.stack((k, v), 2).requires_grad_(train)
        o = cross_attention_packed(q, kv, lengths, mask, scale)
    else:
        k, v = k.requires_grad_(train), v.requires_grad_(train)
        o = cross_attention(q, k, v, lengths, mask, scale)
    if not train:
        return {"o": o}
    o.backward(dev(dout))
    dk, dv = kv.grad.unbind(2) if packed else (k.grad, v.grad)
    return {"o": o, "dq": q.grad, "dk": dk, "dv": dv}


def _check(got, want):
    for name, x in got.items():
        exact, bound = want[name]
        assert x.shape == exact.shape, name
        assert torch.isfinite(x).all(), name
        worst = oracle.excess(x, exact, bound)
        assert worst <= 1.0, f"{name}: {worst:.3f} of its bound"


SIZES = [
    # b, lq, lk, h, hkv, d
    (1, 1, 1, 1, 1, 8),
    (2, 1, 129, 4, 4, 64),
    (3, 5, 77, 4, 2, 64),
    (2, 16, 16, 4, 4, 64),
    (2, 128, 128, 2, 2, 64),
    (1, 129, 127, 3, 1, 40),
    (2, 256, 77, 4, 4, 64),
    (1, 300, 257, 2, 1, 80),
    (1, 257, 400, 2, 2, 128),
    (2, 64, 513, 4, 1, 96),
    (5, 333, 341, 4, 2, 72),
    (1, 2, 1030, 8, 2, 128),
]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("mask", ["none", "lengths", "mask", "both"])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_forward_and_gradients(cuda, size, mask, dtype):
    q, k, v, dout = _inputs(*size, dtype, seed=sum(size))
    lengths, keep = _masks(mask, size[0], size[2], seed=sum(size))
    want = oracle.cross_attention(q, k, v, dout, lengths, keep)
    _check(_run(cuda, q, k, v, dout, lengths, keep, packed=sum(size) % 2 == 0), want)
    _check(_run(cuda, q, k, v, None, lengths, keep), want)


@pytest.mark.parametrize("size", [(1, 1, 1024, 4, 4, 64), (3, 1, 2000, 8, 2, 128), (2, 1, 63, 4, 1, 40),
                                  (1, 3, 4097, 6, 2, 64), (130, 1, 300, 2, 2, 64), (1, 16, 3000, 2, 2, 128)],
                         ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("mask", ["none", "lengths", "mask"])
def test_few_queries_over_long_states(cuda, size, mask):
    """The single-token form: the keys of one query split over the GPU and joined."""
    q, k, v, _ = _inputs(*size, BF16, seed=sum(size))
    lengths, keep = _masks(mask, size[0], size[2], seed=sum(size))
    _check(_run(cuda, q, k, v, None, lengths, keep), oracle.cross_attention(q, k, v, None, lengths, keep))


@pytest.mark.parametrize("size", [(1, 1, 1024, 4, 4, 64), (40, 2, 1000, 8, 4, 80)], ids=["inside", "launch"])
def test_joined_splits_are_the_same_every_time(cuda, size):
    """One after another, and on two streams side by side (joined inside the launch, or by a second one)."""
    from fp8_b200.cross_attention import cross_attention

    q, k, v, _ = (None if x is None else x.to(cuda) for x in _inputs(*size, BF16, seed=1))
    lengths = torch.randint(0, size[2] + 1, (size[0],), generator=torch.Generator().manual_seed(4), dtype=torch.int32)
    lengths = lengths.to(cuda)
    first = cross_attention(q, k, v, lengths)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(cuda) for _ in range(2)]
    got = []
    for i in range(8):
        with torch.cuda.stream(streams[i % 2]):
            got.append(cross_attention(q, k, v, lengths))
    torch.cuda.synchronize()
    assert all(torch.equal(first, o) for o in got)


@pytest.mark.parametrize("d,dtype", [(64, BF16), (128, FP16)])
def test_what_is_not_kept_is_never_used(cuda, d, dtype):
    """Infinities and NaN behind the lengths and the mask change nothing; their gradients are zero."""
    q, k, v, dout = _inputs(3, 140, 270, 4, 2, d, dtype, seed=3)
    lengths, keep = _masks("both", 3, 270, seed=3)
    want = oracle.cross_attention(q, k, v, dout, lengths, keep)
    out = ~oracle.kept_keys(3, 270, lengths, keep)
    k[out] = torch.nan
    v[out] = torch.inf
    v[:, ::3][out[:, ::3]] = torch.nan
    got = _run(cuda, q, k, v, dout, lengths, keep)
    _check(got, want)
    assert torch.count_nonzero(got["dk"][out.to(cuda)]) == 0 and torch.count_nonzero(got["dv"][out.to(cuda)]) == 0
    _check(_run(cuda, q[:, :1].contiguous(), k, v, None, lengths, keep),
           {"o": tuple(x[:, :1] for x in want["o"])})


def test_rows_without_keys(cuda):
    from fp8_b200.cross_attention import cross_attention_fwd

    q, k, v, dout = _inputs(2, 40, 50, 2, 2, 64, BF16)
    lengths = torch.tensor([0, -7], dtype=torch.int64)  # below zero counts as zero
    got = _run(cuda, q, k, v, dout, lengths)
    assert all(torch.count_nonzero(x) == 0 for x in got.values())
    o, lse = cross_attention_fwd(q.to(cuda), k.to(cuda), v.to(cuda), lengths.to(cuda), None, 0.125)
    assert torch.count_nonzero(o) == 0 and torch.isneginf(lse).all()
    lengths = torch.tensor([1000, 50], dtype=torch.int32)  # above the states counts as all of them
    _check(_run(cuda, q, k, v, dout, lengths), oracle.cross_attention(q, k, v, dout))


@pytest.mark.parametrize("lq,lk", [(0, 5), (5, 0), (0, 0)])
def test_empty_sides(cuda, lq, lk):
    q, k, v, dout = _inputs(2, lq, lk, 2, 2, 64, BF16)
    got = _run(cuda, q, k, v, dout)
    assert got["o"].shape == (2, lq, 2, 64) and all(torch.count_nonzero(x) == 0 for x in got.values())


def test_log_sum_exp(cuda):
    from fp8_b200.cross_attention import cross_attention_fwd

    for size in ((2, 150, 200, 2, 2, 64), (2, 1, 700, 4, 2, 128)):
        q, k, v, _ = _inputs(*size, BF16, seed=9)
        lengths, _ = _masks("lengths", size[0], size[2])
        want = oracle.cross_attention(q, k, v, None, lengths)
        o, lse = cross_attention_fwd(q.to(cuda), k.to(cuda), v.to(cuda), lengths.to(cuda), None, size[-1] ** -0.5)
        assert oracle.excess(lse, *want["lse"]) <= 1.0
        assert oracle.excess(o, *want["o"]) <= 1.0


@pytest.mark.parametrize("std,scale", [(6.0, None), (1.0, 1.0), (1.0, -0.3), (1.0, 0.0)])
def test_sharp_and_flat_scores(cuda, std, scale):
    """Large scores (weights near one-hot, maxima that rise late), a negative and a zero scale."""
    q, k, v, dout = _inputs(1, 200, 300, 2, 2, 64, BF16, seed=5, std=std)
    v, dout = v / std, dout / std
    k = k * torch.linspace(0.2, 1.0, 300)[:, None, None]  # later keys score higher
    k = k.to(BF16)
    if std > 1:
        q, k = (q / 2).to(BF16), k
    v, dout = v.to(BF16), dout.to(BF16)
    s = 64**-0.5 if scale is None else scale
    _check(_run(cuda, q, k, v, dout, scale=s), oracle.cross_attention(q, k, v, dout, scale=s))


def test_strides_and_layouts(cuda):
    """Head-major tensors, slices of a projection, a broadcast batch, rows off 16 bytes, a reversed token order."""
    from fp8_b200.cross_attention import cross_attention

    q, k, v, dout = _inputs(2, 70, 90, 4, 4, 64, BF16, seed=8)
    want = oracle.cross_attention(q, k, v, dout)
    head_major = lambda t: t.transpose(1, 2).contiguous().to(cuda).transpose(1, 2)  # noqa: E731
    wide = torch.zeros(2, 90, 4, 200, dtype=BF16, device=cuda)
    wide[..., 8:72] = k.to(cuda)
    odd = torch.zeros(2 * 90 * 4 * 64 + 1, dtype=BF16, device=cuda)[1:].view(2, 90, 4, 64)
    odd.copy_(v)
    strided = torch.zeros(2, 90, 4, 128, dtype=BF16, device=cuda)[..., ::2]
    strided.copy_(k)
    for qq, kk, vv in ((head_major(q), head_major(k), head_major(v)), (q.to(cuda), wide[..., 8:72], odd),
                       (q.to(cuda), strided, v.to(cuda))):
        assert oracle.excess(cross_attention(qq, kk, vv), *want["o"]) <= 1.0
    got = {}
    qq, kk, vv = (head_major(t).detach().requires_grad_(True) for t in (q, k, v))
    o = cross_attention(qq, kk, vv)
    o.backward(head_major(dout))
    got = {"o": o, "dq": qq.grad, "dk": kk.grad, "dv": vv.grad}
    _check(got, want)
    # one sequence's states for every image: the gradient is the sum over the batch
    one = [t[:1].to(cuda).requires_grad_(True) for t in (k, v)]
    o = cross_attention(q.to(cuda), *(t.expand(2, -1, -1, -1) for t in one))
    o.backward(dout.to(cuda))
    kb, vb = (t[:1].expand(2, -1, -1, -1) for t in (k, v))
    want = oracle.cross_attention(q, kb, vb, dout)
    for t, name in zip(one, ("dk", "dv")):
        exact, bound = want[name]
        total = exact.sum(0, keepdim=True)
        assert oracle.excess(t.grad, total, bound.sum(0, keepdim=True) + 2 * oracle.ROUNDOFF[BF16] * total.abs()) <= 1.0


def test_gradients_against_differences(cuda):
    """The kernels' gradients against central differences of the 64-bit forward along random directions."""
    size = (2, 33, 45, 4, 2, 64)
    q, k, v, dout = _inputs(*size, FP16, seed=21)
    lengths, keep = _masks("both", 2, 45, seed=4)
    lengths[-1] = 30
    got = _run(cuda, q, k, v, dout, lengths, keep)
    base = oracle.cross_attention(q, k, v, dout, lengths, keep)
    g = torch.Generator().manual_seed(2)
    x = [t.double() for t in (q, k, v)]
    for at, name in enumerate(("dq", "dk", "dv")):
        d = torch.randn(x[at].shape, generator=g, dtype=torch.float64)
        eps = 1e-4
        loss = []
        for sign in (1, -1):
            y = list(x)
            y[at] = x[at] + sign * eps * d
            loss.append((oracle.cross_attention(*y, None, lengths, keep)["o"][0] * dout.double()).sum().item())
        difference = (loss[0] - loss[1]) / (2 * eps)
        along = (got[name].cpu().double() * d).sum().item()
        # the kernel's own bound along |d|, and the difference's error, eps^2 times a third derivative of order one
        slack = (base[name][1] * d.abs()).sum().item() + 1e-4 * abs(difference) + 1e-4
        assert abs(along - difference) <= slack, (name, along, difference, slack)


def test_same_call_same_bits(cuda):
    q, k, v, dout = _inputs(2, 300, 500, 4, 2, 64, BF16, seed=2)
    a, b = (_run(cuda, q, k, v, dout) for _ in range(2))
    assert all(torch.equal(a[n], b[n]) for n in a)
    a, b = (_run(cuda, q[:, :1].contiguous(), k, v) for _ in range(2))
    assert torch.equal(a["o"], b["o"])


def test_other_stream_and_graph(cuda):
    """The call runs on torch's current stream and can be captured; replays follow the inputs and the lengths."""
    from fp8_b200.cross_attention import cross_attention

    q, k, v, _ = (t.to(cuda) for t in _inputs(2, 1, 900, 4, 4, 64, BF16, seed=6))
    lengths = torch.tensor([900, 5], dtype=torch.int32, device=cuda)
    cross_attention(q, k, v, lengths)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        first = cross_attention(q, k, v, lengths)
    torch.cuda.current_stream().wait_stream(stream)
    want = oracle.cross_attention(q, k, v, None, lengths)
    assert oracle.excess(first, *want["o"]) <= 1.0
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = cross_attention(q, k, v, lengths)
    lengths.copy_(torch.tensor([37, 600], dtype=torch.int32))
    graph.replay()
    assert oracle.excess(o, *oracle.cross_attention(q, k, v, None, lengths)["o"]) <= 1.0


def test_refusals(cuda):
    from fp8_b200.cross_attention import cross_attention, cross_attention_packed

    q = torch.zeros(2, 8, 4, 64, dtype=BF16, device=cuda)
    k = torch.zeros(2, 9, 4, 64, dtype=BF16, device=cuda)
    for bad in (lambda: cross_attention(q.cpu(), k, k), lambda: cross_attention(q.float(), k.float(), k.float()),
                lambda: cross_attention(q, k.half(), k), lambda: cross_attention(q, k, k[:, :8]),
                lambda: cross_attention(q, k[:1], k[:1]), lambda: cross_attention(q, k[..., :32], k[..., :32]),
                lambda: cross_attention(q[..., :60], k[..., :60], k[..., :60]),
                lambda: cross_attention(q, k[:, :, :3], k[:, :, :3]),
                lambda: cross_attention(torch.cat([q] * 3, -1), torch.cat([k] * 3, -1), torch.cat([k] * 3, -1)),
                lambda: cross_attention(q, k, k, key_lengths=torch.ones(2, device=cuda)),
                lambda: cross_attention(q, k, k, key_lengths=torch.ones(3, device=cuda, dtype=torch.int32)),
                lambda: cross_attention(q, k, k, key_mask=torch.ones(2, 9, device=cuda)),
                lambda: cross_attention(q, k, k, key_mask=torch.ones(2, 8, device=cuda, dtype=torch.bool)),
                lambda: cross_attention(q, k, k, scale=float("nan")), lambda: cross_attention_packed(q, k)):
        with pytest.raises(RuntimeError):
            bad()


def test_states_whose_offsets_pass_32_bits(cuda):
    """Packed states of 4.6e9 values: only a few keys of each sequence are kept, the last one's far behind 2^32."""
    from fp8_b200.cross_attention import cross_attention_packed

    b, lk, hkv, d = 2, 1_130_000, 8, 128
    kv = torch.empty(b, lk, 2, hkv, d, dtype=BF16, device=cuda)  # what is not kept is whatever was there
    assert kv.numel() > 2**32
    g = torch.Generator(device=cuda).manual_seed(0)
    keep = torch.zeros(b, lk, dtype=torch.bool, device=cuda)
    at = [[5, 70_000, lk - 1], [0, 130, lk - 2]]
    few = torch.randn(b, 3, 2, hkv, d, device=cuda, generator=g).to(BF16)
    for i in range(b):
        keep[i, at[i]] = True
        kv[i, at[i]] = few[i]
    q = torch.randn(b, 3, hkv, d, device=cuda, generator=g).to(BF16).requires_grad_(True)
    dout = torch.randn(b, 3, hkv, d, device=cuda, generator=g).to(BF16)
    kv.requires_grad_(True)
    out = cross_attention_packed(q, kv, key_mask=keep)
    dq, dkv = torch.autograd.grad(out, (q, kv), dout)
    want = oracle.cross_attention(q.detach().cpu(), few[:, :, 0].cpu(), few[:, :, 1].cpu(), dout.cpu(), None, None)
    picked = torch.stack([dkv[i, at[i]] for i in range(b)])
    got = {"o": out, "dq": dq, "dk": picked[:, :, 0], "dv": picked[:, :, 1]}
    for name, x in got.items():
        exact, bound = want[name]
        worst = oracle.excess(x.detach().cpu(), exact, bound)
        assert worst <= 1.0, f"{name}: {worst:.3f} of its bound"
    for i in range(b):
        for near in (at[i][1] - 1, at[i][1] + 1, lk - 3):
            assert torch.count_nonzero(dkv[i, near]) == 0
