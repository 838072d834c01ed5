"""Prompts at the edge of what the UNet's conditioning takes: of another batch than the images, of no tokens at all, and
lengths without prompts."""

from __future__ import annotations

import pytest
import torch

from fp8_b200.conditioning import PromptAttention, PromptEncoder
from fp8_b200.unet import UNet, UNetConfig


@pytest.mark.parametrize("shape", [(2, 10, 32), (1, 10, 32), (10, 32), (4, 1, 10, 32)])
def test_states_of_another_batch_are_refused(shape):
    """Four images: two prompts of ten states are not four of five."""
    attention, x = PromptAttention(64, 32, 1), torch.zeros(4, 64, 2, 2)
    with pytest.raises(RuntimeError, match=r"states must be \[4, tokens, width\]"):
        attention(x, torch.zeros(shape))


def test_lengths_without_prompts_are_refused():
    x, t = torch.zeros(1, 3, 32, 32), torch.zeros(1, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="prompt_vocab"):
        UNet(UNetConfig())(x, t, prompt_lengths=torch.tensor([3]))


@pytest.mark.gpu
@pytest.mark.parametrize("autocast", [True, False])
def test_prompts_without_tokens(cuda, autocast):
    torch.manual_seed(0)
    enc, att = PromptEncoder(20, 48, 9, padding_idx=0, p_drop=0.5).to(cuda), PromptAttention(64, 48, 2).to(cuda)
    torch.nn.init.normal_(att.out.weight)
    x = torch.randn(3, 64, 4, 4, device=cuda).to(memory_format=torch.channels_last).requires_grad_(True)
    with torch.autocast("cuda", torch.bfloat16, enabled=autocast):
        states = enc(torch.zeros(3, 0, dtype=torch.int64, device=cuda))
        y = att(x, states)
    assert states.shape == (3, 0, 48) and torch.equal(y, x)
    y.backward(torch.ones_like(y))
    assert torch.equal(x.grad, torch.ones_like(x))
    assert torch.count_nonzero(enc.weight.grad) == 0 and torch.count_nonzero(att.kv.weight.grad) == 0
