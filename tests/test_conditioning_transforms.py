"""The conditioning operators under torch's transforms: what has no derivative says so; compiled code calls the same kernels."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from fp8_b200.cross_attention import cross_attention, cross_attention_packed
from fp8_b200.dropout import dropout, dropout_add
from fp8_b200.embedding import embed_tokens

BF16 = torch.bfloat16


def _meta(*shape, dtype=BF16):
    return torch.empty(shape, dtype=dtype, device="meta")


Q, K, KV, X, W = _meta(2, 5, 4, 64), _meta(2, 6, 4, 64), _meta(2, 6, 2, 4, 64), _meta(4, 8), _meta(50, 16)
IDS, SEED = _meta(3, 7, dtype=torch.int64), _meta(dtype=torch.int64)
OPERATORS = {
    "attention's queries": (lambda t: cross_attention(t, K, K), Q),
    "attention's keys": (lambda t: cross_attention(Q, t, K), K),
    "attention's values": (lambda t: cross_attention(Q, K, t), K),
    "packed states": (lambda t: cross_attention_packed(Q, t), KV),
    "embedding's weight": (lambda t: embed_tokens(IDS, t), W),
    "dropout": (lambda t: dropout(t, 0.1, SEED), X),
    "residual": (lambda t: dropout_add(X, t, 0.1, SEED), X),
}


@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("name", OPERATORS)
def test_forward_mode_is_refused(name, requires_grad):
    f, t = OPERATORS[name]
    assert f(t).device.type == "meta"
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(t.detach().requires_grad_(requires_grad), torch.empty_like(t))
        with pytest.raises(RuntimeError, match="forward-mode"):
            f(dual)
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(f, (t,), (torch.empty_like(t),))


@pytest.mark.parametrize("name", OPERATORS)
def test_a_second_derivative_is_refused(name):
    f, t = OPERATORS[name]
    t = t.detach().requires_grad_(True)
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(f(t).float().sum(), t, create_graph=True)


@pytest.mark.gpu
def test_compiled_code_calls_the_same_kernels(cuda):
    g = torch.Generator(device=cuda).manual_seed(0)
    new = lambda *s: torch.randn(*s, device=cuda, generator=g).to(BF16).requires_grad_(True)  # noqa: E731
    q, kv, w, r = new(2, 40, 4, 64), new(2, 150, 2, 2, 64), new(60, 256), new(2, 40, 256)
    ids = torch.randint(0, 60, (2, 40), device=cuda, generator=g)
    seed, lengths = torch.tensor(9, device=cuda), torch.tensor([150, 70], dtype=torch.int32, device=cuda)

    def step(q, kv, w, r):
        x = embed_tokens(ids, w, 2.0).view(2, 40, 4, 64)
        o = cross_attention_packed(q + x, kv, lengths).flatten(2)
        return dropout_add(o, r, 0.25, seed)

    dy = torch.randn(2, 40, 256, device=cuda, generator=g).to(BF16)
    results = []
    for f in (step, torch.compile(step, backend="aot_eager", fullgraph=True)):
        y = f(q, kv, w, r)
        results.append((y.detach(), *torch.autograd.grad(y, (q, kv, w, r), dy)))
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.gpu
def test_dropout_in_a_batch_of_calls_is_each_call(cuda):
    x = torch.randn(3, 7, 40, device=cuda)
    seed = torch.tensor(4, device=cuda)
    want = torch.stack([dropout(t, 0.5, seed) for t in x])
    assert torch.equal(torch.func.vmap(lambda t: dropout(t, 0.5, seed))(x), want)
