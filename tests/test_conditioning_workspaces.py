"""CPU tests of the conditioning operators' sizes: what lies in the embedding gradient's workspace, the counter its sort's
CTAs meet at included, and sizes whose tiles would pass 32 bits."""

from __future__ import annotations

import ctypes

import pytest

from fp8_b200 import _lib


@pytest.mark.parametrize("tokens,vocab,width", [(5000, 300, 72), (20_000, 32_768, 512), (262_147, 131_072, 1024)])
def test_the_sort_meets_at_a_counter_of_its_workspace(tokens, vocab, width):
    word = lambda n: -(-4 * n // 16) * 16  # noqa: E731  (n 32-bit values, in whole 16 bytes)
    need = vocab.bit_length()  # keys are 0 .. vocab
    passes = -(-need // 9)
    ctas = min(96, -(-tokens // 1024))
    chunks = -(-tokens // max(16, -(-tokens // 2048)))
    parts = [word(tokens)] * 4 + [word(ctas << -(-need // passes)), word(vocab // 32 + 1)] + [word(chunks * width)] * 2
    live = counter = word(1)
    assert _lib.load().fp8_embedding_bwd_workspace_bytes(tokens, vocab, width) == sum(parts) + live + counter


@pytest.mark.parametrize("name", ["q_len", "k_len"])
@pytest.mark.parametrize("length", [2**31 - 1, 2**31 - 127])
def test_lengths_whose_tiles_pass_32_bits_are_refused(name, length):
    lib, p = _lib.load(), 1 << 20  # a pointer that is never followed
    a = _lib.CrossAttentionArgs(batch=1, q_len=1, k_len=1, heads=1, kv_heads=1, head_dim=8, dtype=0, scale=1.0)
    for n in ("q", "k", "v", "o", "lse", "dout", "dq", "dk", "dv"):
        setattr(a, n, p)
        if n != "lse":
            setattr(a, n + "_stride", _lib.HeadStrides(8, 8, 8))
    setattr(a, name, length)
    for status in (lib.fp8_cross_attention_fwd(ctypes.byref(a), None, 0, None),
                   lib.fp8_cross_attention_bwd(ctypes.byref(a), None, 0, None)):
        assert status != _lib.FP8_OK and "too long" in _lib.last_error()[1]


def test_widths_that_pass_32_bits_are_refused():
    lib, p, width = _lib.load(), 1 << 20, 2**31 - 1
    assert lib.fp8_embedding_fwd(p, 1, 1, p, 0, 1, width, width, 1.0, p, 0, None) != _lib.FP8_OK
    assert "too wide" in _lib.last_error()[1]
    assert lib.fp8_embedding_bwd(p, 1, 1, p, 0, p, 0, 1, width, 1.0, -1, None, 0, None) != _lib.FP8_OK
    assert "too wide" in _lib.last_error()[1]
