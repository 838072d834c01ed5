"""GPU tests of what the conditioning operators share between calls: nothing.

Where CTAs of a launch meet, they meet at a cluster's barrier or at a counter of the call's own
workspace, which the call zeroes: whatever the workspace held, whatever runs beside the call,
and however often a captured call is replayed, the results are the same.
"""

from __future__ import annotations

import ctypes

import pytest
import torch

import conditioning_oracle as oracle

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _single_queries(cuda, b, lk, h, hkv, d, seed=0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    new = lambda *s: torch.randn(*s, device=cuda, generator=g).to(BF16)  # noqa: E731
    return new(b, 1, h, d), new(b, lk, hkv, d), new(b, lk, hkv, d)


def _attention_args(q, k, v, o):
    from fp8_b200 import _lib

    a = _lib.CrossAttentionArgs(batch=q.shape[0], q_len=q.shape[1], k_len=k.shape[1], heads=q.shape[2], kv_heads=k.shape[2],
                                head_dim=q.shape[3], dtype=0, scale=q.shape[3] ** -0.5)
    for name, t in (("q", q), ("k", k), ("v", v), ("o", o)):
        setattr(a, name, t.data_ptr())
        setattr(a, name + "_stride", _lib.HeadStrides(*t.stride()[:3]))
    return a


@pytest.mark.parametrize("lk,splits", [(129, 2), (300, 4), (600, 8), (1000, 8), (1500, 12)])
@pytest.mark.parametrize("lengths", ["all", "short"])
def test_attention_needs_its_partial_results_alone(cuda, lk, splits, lengths):
    """Up to 8 splits of 128 keys meet in a cluster, more are joined by a second launch; none at a counter in memory."""
    from fp8_b200 import _lib

    lib = _lib.load()
    q, k, v = _single_queries(cuda, 3, lk, 4, 2, 64)
    o = torch.empty_like(q)
    a = _attention_args(q, k, v, o)
    count = None
    if lengths == "short":  # splits without keys, and a sequence without any
        count = torch.tensor([lk, 1, 0], dtype=torch.int32, device=cuda)
        a.key_lengths = count.data_ptr()
    need = lib.fp8_cross_attention_workspace_bytes(ctypes.byref(a), 0)
    assert need == 4 * splits * 3 * 4 * (64 + 1)
    ws = torch.empty(need, dtype=torch.uint8, device=cuda)
    stream = torch.cuda.current_stream(cuda).cuda_stream
    want = oracle.cross_attention(q, k, v, None, count)["o"]
    for fill in (0, 255, 1):
        ws.fill_(fill)
        o.fill_(torch.nan)
        assert lib.fp8_cross_attention_fwd(ctypes.byref(a), ws.data_ptr(), need, stream) == 0, _lib.last_error()
        assert oracle.excess(o, *want) <= 1.0
    assert lib.fp8_cross_attention_fwd(ctypes.byref(a), ws.data_ptr(), need - 4, stream) != 0
    assert _lib.device_error() == 0


def test_a_replayed_attention_beside_many_calls(cuda):
    """A captured call replayed on one stream while another stream issues 9,000 calls of 128 joins each."""
    from fp8_b200.cross_attention import cross_attention

    q, k, v = _single_queries(cuda, 32, 256, 4, 4, 64, seed=1)
    want = cross_attention(q, k, v)
    assert oracle.excess(want, *oracle.cross_attention(q, k, v)["o"]) <= 1.0
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = cross_attention(q, k, v)
    replays, eager = torch.cuda.Stream(cuda), torch.cuda.Stream(cuda)
    wrong = torch.zeros((), dtype=torch.int64, device=cuda)
    torch.cuda.synchronize()
    for i in range(9000):
        with torch.cuda.stream(eager):
            last = cross_attention(q, k, v)
        if i % 4 == 0:
            with torch.cuda.stream(replays):
                got.fill_(torch.nan)
                graph.replay()
                wrong += (got != want).any()
    torch.cuda.synchronize()
    assert wrong.item() == 0 and torch.equal(last, want)


def _tokens(cuda, n, vocab, width, seed=0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    ids = torch.randint(0, vocab, (n,), device=cuda, generator=g)
    return ids, torch.randn(n, width, device=cuda, generator=g).to(BF16)


def _embedding_bwd(ids, dout, dw, ws, need=None):
    from fp8_b200 import _lib

    return _lib.load().fp8_embedding_bwd(ids.data_ptr(), 1, ids.numel(), dout.data_ptr(), 0, dw.data_ptr(), 1, dw.shape[0],
                                         dw.shape[1], 1.0, -1, ws.data_ptr(), ws.numel() if need is None else need,
                                         torch.cuda.current_stream().cuda_stream)


def _gradient_error(dw, ids, dout):
    exact, mag = oracle.embedding_grad(ids, dout, dw.shape[0], 1.0, None)
    count = torch.bincount(ids.cpu(), minlength=dw.shape[0]).double()[:, None]
    return oracle.excess(dw, exact, 2.0**-24 * exact.abs() + (count + 2) * 2.0**-24 * mag)


def test_embedding_sort_meets_at_a_counter_of_its_workspace(cuda):
    from fp8_b200 import _lib

    ids, dout = _tokens(cuda, 20_000, 700, 72)
    need = _lib.load().fp8_embedding_bwd_workspace_bytes(20_000, 700, 72)
    ws, dw = torch.empty(need, dtype=torch.uint8, device=cuda), torch.empty(700, 72, device=cuda)
    for fill in (0, 255, 1):
        ws.fill_(fill)
        dw.fill_(torch.nan)
        assert _embedding_bwd(ids, dout, dw, ws) == 0, _lib.last_error()
        assert _gradient_error(dw, ids, dout) <= 1.0
    assert _embedding_bwd(ids, dout, dw, ws, need - 16) != 0
    assert _lib.device_error() == 0


def test_a_replayed_gradient_beside_many_calls(cuda):
    """4,500 calls beside the replays: counters shared in a ring (of 8,192, two a call) would come round."""
    from fp8_b200 import _lib
    from fp8_b200.embedding import embedding_bwd

    ids, dout = _tokens(cuda, 5000, 300, 40, seed=1)
    run = lambda: embedding_bwd(ids, dout, 300, 1.0, -1, torch.float32)  # noqa: E731
    want = run()
    assert _gradient_error(want, ids, dout) <= 1.0
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    replays, eager = torch.cuda.Stream(cuda), torch.cuda.Stream(cuda)
    wrong = torch.zeros((), dtype=torch.int64, device=cuda)
    torch.cuda.synchronize()
    for i in range(4500):
        with torch.cuda.stream(eager):
            last = run()
        if i % 4 == 0:
            with torch.cuda.stream(replays):
                got.fill_(torch.nan)
                graph.replay()
                wrong += (got != want).any()
    torch.cuda.synchronize()
    assert wrong.item() == 0 and torch.equal(last, want)
    assert _lib.device_error() == 0


@pytest.mark.parametrize("dtype,code", [(BF16, 0), (torch.float32, 1), (torch.float16, 2)])
@pytest.mark.parametrize("n,offset", [(1 << 20, 0), (3_000_001, 0), (70_001, 1)])
def test_dropout_in_place(cuda, n, offset, dtype, code):
    """Over its input, and over its residual: the values of the call that writes elsewhere."""
    from fp8_b200 import _lib
    from fp8_b200.dropout import dropout, dropout_add

    g = torch.Generator(device=cuda).manual_seed(n)
    x, r = (torch.randn(n + offset, device=cuda, generator=g).to(dtype)[offset:] for _ in range(2))
    seed = torch.tensor(5, device=cuda)
    stream = torch.cuda.current_stream(cuda).cuda_stream
    run = lambda x, r, y: _lib.load().fp8_dropout(x.data_ptr(), None if r is None else r.data_ptr(), y.data_ptr(),  # noqa: E731
                                                  code, n, 0.3, seed.data_ptr(), stream)
    alone, joined = dropout(x, 0.3, seed), dropout_add(x, r, 0.3, seed)
    storage = torch.empty(n + offset, dtype=dtype, device=cuda)
    y = storage[offset:]
    for r_in, want in ((None, alone), (r, joined)):
        y.copy_(x)
        assert run(y, r_in, y) == 0 and torch.equal(y, want)
    y.copy_(r)
    assert run(x, y, y) == 0 and torch.equal(y, joined)


def test_a_sort_that_gives_up_reads_nothing_and_leaves_nothing_behind(cuda):
    from fp8_b200 import _lib

    lib = _lib.load()
    assert _lib.device_error() == 0
    ids, dout = _tokens(cuda, 20_000, 700, 72, seed=2)
    need = lib.fp8_embedding_bwd_workspace_bytes(20_000, 700, 72)
    ws, dw = torch.empty(need, dtype=torch.uint8, device=cuda), torch.empty(700, 72, device=cuda)
    assert lib.fp8_selftest_sort_timeout(10**9 + 1) != 0
    try:
        assert lib.fp8_selftest_sort_timeout(20_000_000) == 0
        ws.fill_(255)
        dw.fill_(torch.nan)
        assert _embedding_bwd(ids, dout, dw, ws) == 0, _lib.last_error()
        assert _lib.device_error(torch.cuda.current_stream().cuda_stream) == 202
        assert torch.count_nonzero(dw) == 0
    finally:
        assert lib.fp8_selftest_sort_timeout(0) == 0
    for _ in range(2):  # in the same workspace as it was left
        assert _embedding_bwd(ids, dout, dw, ws) == 0, _lib.last_error()
        assert _gradient_error(dw, ids, dout) <= 1.0
    assert _lib.device_error() == 0


def test_an_id_outside_the_vocabulary_does_not_hide_a_time_out(cuda):
    from fp8_b200 import _lib
    from fp8_b200.embedding import embed_tokens, embedding_bwd

    lib = _lib.load()
    assert _lib.device_error() == 0
    ids, dout = _tokens(cuda, 5000, 300, 40, seed=3)
    stray = lambda: embed_tokens(torch.full((2,), 300, device=cuda), torch.zeros(300, 8, device=cuda))  # noqa: E731
    stray()
    try:
        assert lib.fp8_selftest_sort_timeout(20_000_000) == 0
        embedding_bwd(ids, dout, 300, 1.0, -1, torch.float32)
    finally:
        assert lib.fp8_selftest_sort_timeout(0) == 0
    stray()  # and does not take its place
    assert _lib.device_error() == 202
    stray()
    assert _lib.device_error() == 201 and _lib.device_error() == 0


@pytest.mark.parametrize("dtype", [BF16, torch.float16])
@pytest.mark.parametrize("mode", [1, 2])
def test_programmatic_launches_give_the_same(cuda, mode, dtype):
    """Kernels that begin while the one before ends (fp8_set_pdl) wait for what it wrote, zeroed words included."""
    from fp8_b200 import _lib
    from fp8_b200.cross_attention import cross_attention
    from fp8_b200.dropout import dropout_add
    from fp8_b200.embedding import embed_tokens

    g = torch.Generator(device=cuda).manual_seed(mode)
    new = lambda *s: torch.randn(*s, device=cuda, generator=g).to(dtype)  # noqa: E731
    q, k, v, w, r = (new(*s).requires_grad_(True) for s in ((3, 200, 4, 64), (3, 700, 2, 64), (3, 700, 2, 64), (500, 256),
                                                           (3, 200, 256)))
    ids = torch.randint(0, 500, (3, 1000), device=cuda, generator=g)
    seed, dy, dx = torch.tensor(2, device=cuda), new(3, 200, 256), new(3, 1000, 256)

    def step():
        y = dropout_add(cross_attention(q, k, v).flatten(2), r, 0.2, seed)
        x = embed_tokens(ids, w)
        one = cross_attention(q[:, :1], k, v)
        return (y.detach(), x.detach(), one.detach(), *torch.autograd.grad((y, x), (q, k, v, w, r), (dy, dx)))

    want = step()
    try:
        _lib.set_pdl(mode)
        for _ in range(20):
            assert all(torch.equal(a, b) for a, b in zip(step(), want))
    finally:
        _lib.set_pdl(0)
    assert _lib.device_error() == 0
