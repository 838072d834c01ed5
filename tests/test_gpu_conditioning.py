"""The prompt encoder and the attention over its states, as the UNet uses them, against the formulas in 64 bits.

Tolerance, on the norm of a tensor: every value on a path is rounded to bfloat16 at most ten times forward and ten
times backward (norm, projections, attention, output), each by at most 2^-9 of it; the roundings are independent, and
the layers between neither shrink nor grow a relative error by more than two: 2 * sqrt(20) * 2^-9 = 0.0175.
"""

from __future__ import annotations

import copy

import pytest
import torch
import torch.nn.functional as F

TOL = 0.0175

pytestmark = pytest.mark.gpu


def _near(got, want):
    assert got.shape == want.shape and torch.isfinite(got).all()
    err = (got.detach().cpu().double() - want.detach()).norm() / want.detach().norm()
    assert err <= TOL, err.item()


def _encoder_formula(m, ids):
    e = F.embedding(ids, m.weight, padding_idx=m.padding_idx) * m.scale + m.position[: ids.shape[1]]
    return F.layer_norm(e, e.shape[-1:], m.norm.weight, m.norm.bias, m.norm.eps)


def _attention_formula(m, x, states, lengths):
    b, c, h, w = x.shape
    tokens = x.flatten(2).transpose(1, 2)
    heads = lambda z: z.unflatten(-1, (m.nh, c // m.nh)).transpose(1, 2)  # noqa: E731
    q = heads(m.q(F.layer_norm(tokens, (c,), m.norm.weight, m.norm.bias, m.norm.eps)))
    k, v = (heads(z) for z in m.kv(states).chunk(2, dim=-1))
    s = q @ k.transpose(-1, -2) / (c // m.nh) ** 0.5
    s = s.masked_fill(torch.arange(states.shape[1]) >= lengths[:, None, None, None], float("-inf"))
    p = torch.nan_to_num(torch.softmax(s, dim=-1))  # a prompt of no tokens: nothing
    y = tokens + m.out((p @ v).transpose(1, 2).flatten(2))
    return y.transpose(1, 2).reshape(b, c, h, w)


@pytest.mark.parametrize("autocast", [True, False])
@pytest.mark.parametrize("channels,heads,width,length,size", [(64, 2, 48, 7, 3), (256, 4, 512, 77, 16), (80, 1, 64, 1, 5)])
def test_encoder_and_attention(cuda, channels, heads, width, length, size, autocast):
    from fp8_b200.conditioning import PromptAttention, PromptEncoder

    torch.manual_seed(length)
    enc = PromptEncoder(300, width, 80, padding_idx=0)
    att = PromptAttention(channels, width, heads)
    torch.nn.init.normal_(att.out.weight, std=channels**-0.5)
    b = 3
    ids = torch.randint(1, 300, (b, length))
    ids[:, length // 2 + 1:] = 0
    lengths = torch.tensor([length, max(1, length // 2), 0], dtype=torch.int32)
    x, dy = torch.randn(b, channels, size, size), torch.randn(b, channels, size, size)

    enc64, att64, x64 = copy.deepcopy(enc).double(), copy.deepcopy(att).double(), x.double().requires_grad_(True)
    want = _attention_formula(att64, x64, _encoder_formula(enc64, ids), lengths)
    want.backward(dy.double())

    enc, att = enc.to(cuda), att.to(cuda)
    xg = x.to(cuda).to(memory_format=torch.channels_last).requires_grad_(True)
    with torch.autocast("cuda", torch.bfloat16, enabled=autocast):
        got = att(xg, enc(ids.to(cuda)), lengths.to(cuda))
    got.backward(dy.to(cuda))
    _near(got, want)
    _near(xg.grad, x64.grad)
    for mine, other in ((enc, enc64), (att, att64)):
        for (name, p), q in zip(mine.named_parameters(), other.parameters()):
            if length == 1 and name in ("q.weight", "norm.weight", "norm.bias") and mine is att:
                continue  # one state: the scores have no gradient
            _near(p.grad, q.grad)
    assert torch.count_nonzero(enc.weight.grad[0]) == 0  # padding
    assert torch.equal(got[2], xg[2].to(got.dtype))  # an empty prompt adds nothing


def test_dropout_draws_another_mask_each_time_and_none_in_eval(cuda):
    from fp8_b200.conditioning import PromptAttention, PromptEncoder

    torch.manual_seed(0)
    enc, att = PromptEncoder(50, 64, 9, p_drop=0.5).to(cuda), PromptAttention(64, 64, 1, p_drop=0.5).to(cuda)
    torch.nn.init.normal_(att.out.weight)
    ids, x = torch.randint(0, 50, (2, 9), device=cuda), torch.randn(2, 64, 4, 4, device=cuda)
    run = lambda: att(x, enc(ids))  # noqa: E731
    a, b = run(), run()
    assert not torch.equal(a, b)
    assert (a == x).float().mean() > 0.4  # what was dropped is the residual alone
    enc.eval(), att.eval()
    assert torch.equal(run(), run())


def _unet(cuda, prompt_vocab, **more):
    from fp8_b200.unet import UNet, UNetConfig

    torch.manual_seed(1)
    model = UNet(UNetConfig(p_drop=0.0, prompt_vocab=prompt_vocab, prompt_width=64, **more))
    return model.to(memory_format=torch.channels_last).to(cuda)


def test_an_untrained_prompt_changes_nothing(cuda):
    plain, conditioned = _unet(cuda, 0), _unet(cuda, 500)
    g = torch.Generator(device=cuda).manual_seed(2)
    with torch.no_grad():
        for m in plain.modules():  # the zero-initialised layers: show what reaches them
            for p in m.parameters(recurse=False):
                if torch.count_nonzero(p) == 0 and p.dim() > 1:
                    p.normal_(std=0.02, generator=g)
    conditioned.load_state_dict(plain.state_dict(), strict=False)
    x = torch.randn(2, 3, 32, 32, device=cuda).to(memory_format=torch.channels_last)
    t = torch.tensor([3, 700], device=cuda)
    ids = torch.randint(0, 500, (2, 77), device=cuda)
    with torch.no_grad(), torch.autocast("cuda", torch.bfloat16):
        want = plain(x, t)
        got = conditioned(x, t, ids, torch.tensor([77, 4], dtype=torch.int32, device=cuda))
        assert torch.count_nonzero(want) > 0
        assert (got - want).abs().max() <= 0.02 * want.abs().max()
    for m in conditioned.modules():  # a trained one does
        if type(m).__name__ == "PromptAttention":
            torch.nn.init.normal_(m.out.weight, std=0.1)
    with torch.no_grad(), torch.autocast("cuda", torch.bfloat16):  # (autocast keeps casts of weights until it ends)
        assert (conditioned(x, t, ids) - want).abs().max() > 0.05 * want.abs().max()


@pytest.mark.parametrize("graph", [False, True])
def test_training_step_with_prompts(cuda, graph):
    from fp8_b200.train import GraphedTrainStep, TrainConfig

    model = _unet(cuda, 500)
    step = GraphedTrainStep(model, TrainConfig(batch_size=2, lr=1e-3), cuda, use_graph=graph, external_noise=True)
    g = torch.Generator(device=cuda).manual_seed(3)
    images = torch.randn(2, 3, 32, 32, device=cuda, generator=g)
    ids = torch.randint(1, 500, (2, 77), device=cuda, generator=g)
    t, eps = torch.tensor([10, 500], device=cuda), torch.randn(2, 3, 32, 32, device=cuda, generator=g)
    step.prepare()
    losses = []
    for _ in range(6):
        step.loss_acc.zero_()
        step.step(images, t, eps, prompt_ids=ids, prompt_lengths=torch.tensor([77, 30], dtype=torch.int32))
        losses.append(step.loss_acc.item())
    assert all(0.0 < v < 2.0 for v in losses) and losses[-1] < losses[0]
    grad = model.prompt.weight.grad
    used = torch.zeros(500, dtype=torch.bool, device=cuda)
    used[ids.unique()] = True
    assert torch.count_nonzero(grad[~used]) == 0
    assert torch.count_nonzero(grad[ids[0]]) > 0
    # the second prompt's tokens past its length reach no output
    late = used.clone()
    late[ids[0]] = False
    late[ids[1, :30]] = False
    assert torch.count_nonzero(grad[late]) == 0
    step.release()


def test_operators_in_a_captured_graph(cuda):
    """The forms that meet across CTAs (split keys, sorted gradient) leave their counters as a replay needs them."""
    from fp8_b200.cross_attention import cross_attention
    from fp8_b200.dropout import dropout
    from fp8_b200.embedding import embedding_bwd

    g = torch.Generator(device=cuda).manual_seed(5)
    new = lambda *s: torch.randn(*s, device=cuda, generator=g).to(torch.bfloat16)  # noqa: E731
    q, k, v, dout = new(2, 1, 4, 64), new(2, 1500, 4, 64), new(2, 1500, 4, 64), new(5000, 72)
    ids = torch.randint(0, 300, (5000,), device=cuda, generator=g)
    seed = torch.tensor(7, device=cuda)

    def run():
        out = cross_attention(q, k, v), embedding_bwd(ids, dout, 300, 1.0, -1, torch.float32), dropout(dout, 0.5, seed)
        seed.add_(1)
        return out

    side = torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.stream(side):
        want = [x.clone() for x in run()]
    torch.cuda.current_stream(cuda).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    masks = []
    for _ in range(3):
        q.neg_(), q.neg_()
        graph.replay()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        masks.append(got[2] != 0)
    assert not torch.equal(masks[0], masks[1]) and not torch.equal(masks[1], masks[2])
    # other inputs at the same addresses
    q.neg_()
    graph.replay()
    assert torch.equal(got[0], cross_attention(q, k, v)) and not torch.equal(got[0], want[0])
