"""Refusals of the operators of many sequences, before any HIP call: the C ABI and the Python wrappers."""

from __future__ import annotations

import ctypes

import pytest

ONE = ctypes.c_void_p(256)
ODD = ctypes.c_void_p(260)


def refused(status, text):
    from asdsl import _hip

    assert status == _hip.ASDSL_ERR_INVALID_ARGUMENT and text in _hip.last_error(), _hip.last_error()


def test_append_refusals():
    from asdsl import _hip

    def f(ptrs=(ONE,) * 7, dims=(1, 1, 24, 8, 128, 96, 64, 0, 64)):
        return _hip.LIB.asdsl_kv_append_f16(*ptrs, *dims, None)
    for i in range(7):
        refused(f(ptrs=[None if j == i else ONE for j in range(7)]), "null")
    refused(f(ptrs=(ODD,) + (ONE,) * 6), "aligned")
    for dims, text in (((0, 1, 24, 8, 128, 96, 64, 0, 64), "positive"), ((1, 0, 24, 8, 128, 96, 64, 0, 64), "positive"),
                       ((1, 1, 24, 7, 128, 96, 64, 0, 64), "multiple"), ((1, 1, 24, 8, 96, 96, 64, 0, 64), "head_dim"),
                       ((1, 1, 24, 8, 128, 95, 64, 0, 64), "rotary"), ((1, 1, 24, 8, 128, 130, 64, 0, 64), "rotary"),
                       ((1, 1, 24, 8, 128, 0, 64, 0, 64), "rotary"), ((1, 1, 24, 8, 128, 96, 0, 0, 64), "rows"),
                       ((1, 1, 24, 8, 128, 96, 64, -1, 64), "pos_offset"), ((1, 1, 24, 8, 128, 96, 64, 0, 0), "rope_rows"),
                       ((1 << 20, 1 << 12, 24, 8, 128, 96, 64, 0, 64), "2^31")):
        refused(f(dims=dims), text)
    refused(_hip.LIB.asdsl_kv_append_q8(ONE, ONE, ONE, None, ONE, ONE, ONE, ONE, ONE, 1, 1, 24, 8, 128, 96, 64, 0, 64,
                                        None), "scale")


def test_window_refusals():
    from asdsl import _hip

    lib = _hip.LIB

    def f(ptrs=(ONE,) * 5, dims=(1, 1, 24, 8, 128, 64, 0, 0)):
        return lib.asdsl_attention_window_f16kv(*ptrs, *dims, ONE, 0, None)
    for i in range(5):
        refused(f(ptrs=[None if j == i else ONE for j in range(5)]), "null")
    refused(f(ptrs=(ONE, ODD, ONE, ONE, ONE)), "aligned")
    for dims, text in (((1, 1, 9, 2, 128, 64, 0, 0), "multiple"), ((1, 1, 8, 2, 80, 64, 0, 0), "head_dim"),
                       ((1, 1, 8, 2, 128, 0, 0, 0), "rows"), ((1, 1, 8, 2, 128, 64, -1, 0), "window"),
                       ((1, 1, 8, 2, 128, 64, 0, -1), "sinks")):
        refused(f(dims=dims), text)
        assert lib.asdsl_attention_window_work_bytes(*dims) == 0
    refused(lib.asdsl_attention_window_q8kv(ONE, ONE, ONE, ONE, None, ONE, ONE, 1, 1, 8, 2, 128, 64, 0, 0, ONE, 0, None),
            "scale")


def test_prefix_refusals():
    from asdsl import _hip

    lib = _hip.LIB

    def f(ptrs=(ONE,) * 7, dims=(4, 24, 8, 128, 64, 64, 16)):
        return lib.asdsl_attention_prefix_f16kv(*ptrs, *dims, ONE, 0, None)
    for i in range(7):
        refused(f(ptrs=[None if j == i else ONE for j in range(7)]), "null")
    for dims, text in (((4, 24, 8, 128, 65, 64, 16), "prefix_len"), ((4, 24, 8, 128, -1, 64, 16), "prefix_len"),
                       ((0, 24, 8, 128, 64, 64, 16), "positive"), ((4, 24, 8, 128, 64, 64, 0), "own_rows"),
                       ((4, 24, 8, 32, 64, 64, 16), "head_dim")):
        refused(f(dims=dims), text)
    refused(lib.asdsl_attention_prefix_q8kv(*(ONE,) * 3, None, *(ONE,) * 7, 4, 24, 8, 128, 64, 64, 16, ONE, 0, None),
            "scale")


def test_logits_refusals():
    from asdsl import _hip

    lib = _hip.LIB

    def f(logits=ONE, out=ONE, tokens=ONE, hist=ONE, cap=4, rep=ONE, bias=ONE, bstride=0, allowed=ONE, astride=0, rows=1,
          vocab=100, work=ONE, nbytes=1 << 20):
        return lib.asdsl_logits_control(logits, out, tokens, hist, None, None, cap, rep, None, None, bias, bstride,
                                        allowed, astride, rows, vocab, work, nbytes, None)
    refused(f(logits=None), "null")
    refused(f(out=None), "null")
    refused(f(hist=None), "without a history")
    refused(f(cap=-1), "history_cap")
    refused(f(rows=0), "positive")
    refused(f(vocab=0), "positive")
    refused(f(bstride=99), "bias_stride")
    refused(f(astride=3), "allowed_stride")
    refused(f(work=None), "work buffer")
    refused(f(nbytes=1), "work buffer")
    refused(f(work=ODD), "aligned")
    refused(f(rows=1 << 30, vocab=1 << 20), "rows")
    assert lib.asdsl_logits_control_work_bytes(0, 5) == 0 and lib.asdsl_logits_control_work_bytes(3, 200064) % 256 == 0


def test_wrappers_refuse_what_does_not_fit():
    import torch

    from asdsl.kernels import attention_prefix, attention_window, control_logits, kv_append

    k = torch.zeros((2, 4, 8, 128), dtype=torch.float16)
    q = torch.zeros((2, 1, 8, 128))
    pos = torch.zeros(2, dtype=torch.int32)
    cs = torch.zeros((8, 48))
    codes, scale = k.to(torch.int8), torch.zeros((2, 4, 8, 2))
    bad = [
        (lambda: attention_window(q, k, k, pos), "device"),
        (lambda: attention_window(None, k, k, pos), "device"),
        (lambda: attention_window(q, k, k[:1], pos), "differ"),
        (lambda: attention_window(q, k.float(), k.float(), pos), "fp16 or int8"),
        (lambda: attention_window(q, k[..., :96], k[..., :96], pos), "head_dim"),
        (lambda: attention_window(q[:, :, :6], k, k, pos), "multiple"),
        (lambda: attention_window(q[:, :, :0], k, k, pos), "hold"),
        (lambda: attention_window(torch.zeros(3, 8 * 128), k, k, pos), "must be"),
        (lambda: attention_window(q.double(), k, k, pos), "float32"),
        (lambda: attention_prefix(q, k[0], k[0], codes, codes, pos), "differ"),
        (lambda: attention_prefix(q, k[0, :2], k[0, :2], k, k, pos), "differ"),
        (lambda: attention_prefix(q, k, k, k, k, pos), "3 are wanted"),
        (lambda: attention_prefix(q, k[0], k[0], k, k, pos, prefix_len=9), "prefix_len"),
        (lambda: kv_append(torch.zeros(2, 16 * 128), k, k, cs, cs, pos, n_heads=6), "multiple"),
        (lambda: kv_append(torch.zeros(2, 15 * 128), k, k, cs, cs, pos, n_heads=8), "hold"),
        (lambda: kv_append(torch.zeros(2, 16 * 128), k, k, cs, cs[:4], pos, n_heads=8), "one shape"),
        (lambda: control_logits(torch.zeros(0)), "logits"),
        (lambda: control_logits(torch.zeros(2, 40), repetition=torch.ones(2)), "without a history"),
        (lambda: control_logits(torch.zeros(2, 40), bias=torch.zeros(39)), "bias"),
        (lambda: control_logits(torch.zeros(2, 40), allowed=torch.zeros(3, 2, dtype=torch.int32)), "allowed"),
        (lambda: control_logits(torch.zeros(2, 40), history=torch.zeros(3, 4, dtype=torch.int32)), "history"),
        (lambda: control_logits(torch.zeros(2, 40)), "device"),
    ]
    for call, text in bad:
        with pytest.raises(ValueError, match=text):
            call()
    # scales exactly where the caches are int8 (checked ahead of the devices only for the pairing)
    with pytest.raises(ValueError):
        attention_window(q, codes, codes, pos)
    with pytest.raises(ValueError):
        attention_window(q, k, k, pos, k_scale=scale, v_scale=scale)


def test_sizes_past_the_kernels_ints():
    import torch

    from asdsl import _hip
    from asdsl.kernels import attention_window, control_logits, kv_append

    lib = _hip.LIB
    big = (1 << 30) + 1
    refused(lib.asdsl_attention_window_f16kv(*(ONE,) * 5, 1, 1, 8, 2, 64, big, 0, 0, ONE, 0, None), "2^30")
    assert lib.asdsl_attention_window_work_bytes(1, 1, 8, 2, 64, big, 0, 0) == 0
    refused(lib.asdsl_attention_prefix_f16kv(*(ONE,) * 7, 1, 8, 2, 64, big, big, 1, ONE, 0, None), "2^30")
    refused(lib.asdsl_attention_prefix_f16kv(*(ONE,) * 7, 1, 8, 2, 64, 1, 1, big, ONE, 0, None), "2^30")
    assert lib.asdsl_attention_prefix_work_bytes(1, 8, 2, 64, big, 1) == 0
    assert lib.asdsl_attention_prefix_work_bytes(1, 8, 2, 64, 1, big) == 0
    k = torch.zeros((2, 4, 8, 128), dtype=torch.float16)
    q, pos, cs = torch.zeros((2, 1, 8, 128)), torch.zeros(2, dtype=torch.int32), torch.zeros((8, 48))
    for call in (lambda x: attention_window(q, k, k, pos, window=x), lambda x: attention_window(q, k, k, pos, sinks=x),
                 lambda x: kv_append(torch.zeros(2, 16 * 128), k, k, cs, cs, pos, n_heads=8, pos_offset=x)):
        for x in (-1, 1 << 31, (1 << 32) + 5):
            with pytest.raises(ValueError, match=r"2\^31"):
                call(x)
    with pytest.raises(ValueError, match=r"2\^30"):
        control_logits(torch.zeros(1, 40), history=torch.zeros(1, dtype=torch.int32).expand((1 << 30) + 1))
