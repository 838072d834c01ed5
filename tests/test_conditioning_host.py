"""Host side of the UNet's conditioning on prompts: what its option adds, and what is refused."""

from __future__ import annotations

import pytest
import torch

from fp8_b200.conditioning import PromptAttention, PromptEncoder
from fp8_b200.unet import UNet, UNetConfig


def test_the_option_only_adds_parameters():
    torch.manual_seed(0)
    plain = UNet(UNetConfig())
    with_prompt = UNet(UNetConfig(prompt_vocab=1000, prompt_width=64))
    base = {k: v.shape for k, v in plain.state_dict().items()}
    more = {k: v.shape for k, v in with_prompt.state_dict().items()}
    added = set(more) - set(base)
    assert all(more[k] == s for k, s in base.items())
    assert added and all(k.startswith("prompt.") or ".prompt_attns." in k for k in added)
    assert more["prompt.weight"] == (1000, 64) and more["prompt.position"] == (77, 64)
    assert not any("dropout_seed" in k for k in added)  # seeds are not part of a checkpoint
    # one beside each attention block
    blocks = sum(type(m).__name__ == "CHWAttention" for m in with_prompt.modules())
    assert sum(isinstance(m, PromptAttention) for m in with_prompt.modules()) == blocks
    assert all(torch.count_nonzero(m.out.weight) == 0 for m in with_prompt.modules() if isinstance(m, PromptAttention))


def test_prompts_and_the_model_go_together():
    x, t, ids = torch.zeros(1, 3, 32, 32), torch.zeros(1, dtype=torch.int64), torch.zeros(1, 5, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="prompt"):
        UNet(UNetConfig())(x, t, ids)
    with pytest.raises(RuntimeError, match="prompt"):
        UNet(UNetConfig(prompt_vocab=10))(x, t)
    with pytest.raises(RuntimeError, match="up to 4"):
        PromptEncoder(10, 16, 4)(ids)
    with pytest.raises(RuntimeError, match="up to 4"):
        PromptEncoder(10, 16, 4)(ids[0])
    for channels, heads in ((130, 4), (64, 16), (512, 2)):
        with pytest.raises(ValueError, match="heads"):
            PromptAttention(channels, 16, heads)


def test_there_is_no_kernel_on_the_cpu():
    with pytest.raises((RuntimeError, NotImplementedError)):
        PromptEncoder(10, 16, 4)(torch.zeros(1, 3, dtype=torch.int64))


def test_shapes_without_data():
    """The operators' meta kernels, which tracing asks for shapes and types."""
    from fp8_b200.cross_attention import cross_attention, cross_attention_packed
    from fp8_b200.dropout import dropout_add
    from fp8_b200.embedding import embed_tokens, embedding_bwd

    meta = lambda *s, dtype=torch.bfloat16: torch.empty(s, dtype=dtype, device="meta")  # noqa: E731
    q, kv = meta(2, 9, 8, 40), meta(2, 5, 2, 4, 40)
    for o in (cross_attention_packed(q, kv), cross_attention(q, kv[:, :, 0], kv[:, :, 1])):
        assert o.shape == q.shape and o.dtype == q.dtype and o.device.type == "meta"
    ids, w = meta(3, 7, dtype=torch.int64), meta(50, 16, dtype=torch.float32)
    assert embed_tokens(ids, w, dtype=torch.float16).shape == (3, 7, 16)
    assert embedding_bwd(ids, meta(3, 7, 16), 50, 1.0, -1, torch.float32).shape == (50, 16)
    x = meta(3, 4)
    assert dropout_add(x, x, 0.1, meta(dtype=torch.int64)).shape == (3, 4)
