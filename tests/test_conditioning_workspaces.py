"""CPU test of the embedding gradient's workspace: what lies in it, the counter its sort's CTAs meet at included."""

from __future__ import annotations

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
