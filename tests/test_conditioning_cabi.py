"""CPU tests of the conditioning operators' C entries: what they refuse before any CUDA call, and the message."""

from __future__ import annotations

import ctypes

import pytest

from fp8_b200 import _lib

BF16, FP32, FP16 = 0, 1, 2
P = 1 << 20  # a pointer that is never followed


def _args(**change):
    a = _lib.CrossAttentionArgs(batch=2, q_len=5, k_len=7, heads=4, kv_heads=2, head_dim=64, dtype=BF16, scale=0.125)
    for n in ("q", "k", "v", "o", "lse", "dout", "dq", "dk", "dv"):
        setattr(a, n, P)
    for n in ("q", "o", "dout", "dq"):
        setattr(a, n + "_stride", _lib.HeadStrides(5 * 256, 256, 64))
    for n in ("k", "v", "dk", "dv"):
        setattr(a, n + "_stride", _lib.HeadStrides(7 * 128, 128, 64))
    for n, v in change.items():
        setattr(a, n, v)
    return a


def _refused(status, word):
    code, message = _lib.last_error()
    assert status != _lib.FP8_OK and code == status and word in message, message


BAD = [({"batch": 0}, "positive"), ({"q_len": 0}, "positive"), ({"k_len": -1}, "positive"), ({"kv_heads": 3}, "multiple"),
       ({"head_dim": 136}, "head_dim"), ({"head_dim": 12}, "head_dim"), ({"dtype": FP32}, "dtype"),
       ({"scale": float("nan")}, "scale"), ({"scale": float("inf")}, "scale"), ({"q": None}, "aligned"),
       ({"v": P + 8}, "aligned"), ({"key_lengths": P + 2}, "aligned"),
       ({"q_stride": _lib.HeadStrides(5 * 256, 252, 64)}, "strides"),
       ({"k_stride": _lib.HeadStrides(7 * 128, -128, 64)}, "strides")]
BAD_BACKWARD = [({"lse": None}, "lse"), ({"dk": None}, "dk"), ({"dv": P + 4}, "aligned"),
                ({"dout_stride": _lib.HeadStrides(5 * 256, 256, 60)}, "strides")]


@pytest.mark.parametrize("change,word", BAD)
def test_attention_refuses(change, word):
    lib, a = _lib.load(), _args(**change)
    _refused(lib.fp8_cross_attention_fwd(ctypes.byref(a), None, 0, None), word)
    _refused(lib.fp8_cross_attention_bwd(ctypes.byref(a), None, 0, None), word)


@pytest.mark.parametrize("change,word", BAD_BACKWARD)
def test_attention_backward_refuses(change, word):
    a = _args(**change)
    _refused(_lib.load().fp8_cross_attention_bwd(ctypes.byref(a), None, 0, None), word)


def test_attention_refuses_no_arguments():
    _refused(_lib.load().fp8_cross_attention_fwd(None, None, 0, None), "NULL")


def test_embedding_refuses():
    lib = _lib.load()
    good = [P, 1, 10, P, FP32, 100, 64, 64, 1.0, P, BF16, None]
    for at, value, word in ((2, -1, "sizes"), (5, 0, "sizes"), (6, 0, "sizes"), (4, 3, "dtype"), (10, 7, "dtype"),
                            (3, None, "NULL"), (9, P + 1, "aligned")):
        bad = list(good)
        bad[at] = value
        _refused(lib.fp8_embedding_fwd(*bad), word)
    good = [P, 1, 10, P, BF16, P, FP32, 100, 64, 1.0, -1, None, 0, None]
    for at, value, word in ((2, -1, "sizes"), (7, 0, "sizes"), (4, -1, "dtype"), (6, 3, "dtype"), (5, None, "NULL"),
                            (3, P + 1, "aligned"), (2, 1 << 31, "many")):
        bad = list(good)
        bad[at] = value
        _refused(lib.fp8_embedding_bwd(*bad), word)
    assert lib.fp8_embedding_bwd_workspace_bytes(-1, 100, 64) == 0
    assert lib.fp8_embedding_bwd_workspace_bytes(77, 32768, 512) == 0  # one launch
    # keys, positions and counts of a sort, and partial sums
    assert lib.fp8_embedding_bwd_workspace_bytes(5000, 32768, 512) >= 4 * 4 * 5000


def test_dropout_refuses():
    lib = _lib.load()
    good = [P, P, P, BF16, 100, 0.5, P, None]
    for at, value, word in ((4, -1, "size"), (3, 3, "dtype"), (5, 1.5, "p must"), (5, float("nan"), "p must"),
                            (0, None, "NULL"), (6, None, "NULL"), (2, P + 1, "misaligned"), (6, P + 4, "misaligned")):
        bad = list(good)
        bad[at] = value
        _refused(lib.fp8_dropout(*bad), word)
    assert lib.fp8_dropout(None, None, None, BF16, 0, 0.5, None, None) == _lib.FP8_OK  # nothing to do
