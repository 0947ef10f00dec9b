"""The 4-bit form of cache rows: what its definition promises (on the host), and the refusals of its operators."""

from __future__ import annotations

import kv4_reference as kv4
import numpy as np
import pytest
from test_attention_ops_api import ODD, ONE, refused


@pytest.mark.parametrize("loud", [1e-7, 1e-5, 1e-3, 1.0, 300.0, 30000.0])
@pytest.mark.parametrize("shift", [0.0, 3.0])
def test_values_are_fp16_numbers_within_a_step(loud, shift):
    rng = np.random.default_rng(0)
    x = np.clip((rng.standard_normal((50, 128)) + shift) * loud, -32768, 32768)
    codes, words = kv4.quantize(x)
    y = kv4.values(codes, words)
    assert np.array_equal(y.astype(np.float16).astype(np.float64), y)
    scale = np.repeat((words & ~np.int16(15)).view(np.float16).astype(np.float64), 32, axis=-1)
    # half a step of the code's rounding, or at a clamped end half a step of the zero point's
    assert (np.abs(y - x) <= scale * (1 + 1e-12)).all() and (np.abs(y - x) <= scale / 2 * (1 + 1e-12)).mean() > 0.9
    step = (np.maximum(x.reshape(50, 4, 32).max(-1), 0) - np.minimum(x.reshape(50, 4, 32).min(-1), 0)) / 15
    step = np.repeat(step, 32, axis=-1)
    assert (scale >= step).all() and (scale <= np.maximum(step * (1 + 1 / 64), step + 2.0 ** -20)).all()


def test_edges():
    x = np.zeros((5, 32))
    x[1] = np.linspace(0, 15, 32)  # a range that is 15 whole steps
    x[2, 3], x[3, 5] = np.inf, np.nan
    x[4] = -1e30
    codes, words = kv4.quantize(x)
    y = kv4.values(codes, words)
    assert (y[0] == 0).all() and y[1, 0] == 0 and y[1, -1] == 15 and words[1, 0] == np.float16(1).view(np.int16)
    assert np.isnan(y[2:4]).all() and np.isfinite(y[4]).all() and (np.abs(y[4] + 32768) <= 32768 / 15).all()


def test_abi_refusals():
    from asdsl import _hip

    lib = _hip.LIB
    dims = (1, 1, 24, 8, 128, 96, 64, 0, 64)
    for i in range(9):
        refused(lib.asdsl_kv_append_q4(*[None if j == i else ONE for j in range(9)], *dims, None), "null")
    odd2 = type(ONE)(258)
    refused(lib.asdsl_kv_append_q4(ONE, ONE, ONE, odd2, ONE, ONE, ONE, ONE, ONE, *dims, None), "aligned")
    refused(lib.asdsl_kv_append_q4(ONE, ODD, ONE, ONE, ONE, ONE, ONE, ONE, ONE, *dims, None), "aligned")
    win = (1, 1, 24, 8, 128, 64, 0, 0)
    for i in range(7):
        refused(lib.asdsl_attention_window_q4kv(*[None if j == i else ONE for j in range(7)], *win, ONE, 0, None),
                "null")
    refused(lib.asdsl_attention_window_q4kv(ONE, ONE, ONE, ONE, odd2, ONE, ONE, *win, ONE, 0, None), "aligned")
    pre = (4, 24, 8, 128, 64, 64, 16)
    for i in range(11):
        refused(lib.asdsl_attention_prefix_q4kv(*[None if j == i else ONE for j in range(11)], *pre, ONE, 0, None),
                "null")
    refused(lib.asdsl_attention_window_q4kv(*(ONE,) * 7, 1 << 24, 1, 1, 1, 64, 8, 0, 0, ONE, 1 << 60, None), "2^32")


def test_read_refusals():
    from asdsl import _hip

    lib = _hip.LIB
    for read in (lib.asdsl_kv_read_q8, lib.asdsl_kv_read_q4):
        def f(ptrs=(ONE,) * 7, out_fp32=0, dims=(2, 4, 128, 64, 10)):
            return read(*ptrs, out_fp32, *dims, None)
        for i in (0, 1, 2, 3, 5, 6):
            refused(f(ptrs=[None if j == i else ONE for j in range(7)]), "null")
        refused(f(ptrs=(ODD,) + (ONE,) * 6), "aligned")
        refused(f(ptrs=(ONE,) * 5 + (ODD, ONE)), "aligned")
        for dims, text in (((0, 4, 128, 64, 10), "positive"), ((2, 0, 128, 64, 10), "positive"),
                           ((2, 4, 96, 64, 10), "head_dim"), ((2, 4, 128, 0, 10), "positive"),
                           ((2, 4, 128, 64, 0), "positive"), ((1 << 20, 1 << 10, 64, 64, 1 << 10), "2^32"),
                           ((1 << 30, 1 << 30, 64, 64, 1 << 30), "2^32")):
            refused(f(dims=dims), text)


def test_read_refuses_one_output_for_keys_and_values():
    from asdsl import _hip

    lib = _hip.LIB
    for read in (lib.asdsl_kv_read_q8, lib.asdsl_kv_read_q4):
        for out_fp32 in (0, 1):
            refused(read(*(ONE,) * 7, out_fp32, 2, 4, 128, 64, 10, None), "an output each")


def test_wrappers_refuse_what_does_not_fit():
    import torch

    from asdsl.kernels import attention_prefix, attention_window, kv_append, kv_read

    k = torch.zeros((2, 4, 8, 64), dtype=torch.uint8)
    words = torch.zeros((2, 4, 8, 4), dtype=torch.int16)
    k8, s8 = torch.zeros((2, 4, 8, 128), dtype=torch.int8), torch.zeros((2, 4, 8, 2))
    q, pos = torch.zeros((2, 1, 8, 128)), torch.zeros(2, dtype=torch.int32)
    cs = torch.zeros((8, 48))
    bad = [
        (lambda: attention_window(q, k, k, pos, k_scale=words, v_scale=words), "device"),
        (lambda: attention_window(q, k, k8, pos, k_scale=words, v_scale=words), "differ"),
        (lambda: attention_window(q, k[..., :48], k[..., :48], pos, k_scale=words, v_scale=words), "head_dim"),
        (lambda: attention_prefix(q[:, 0], k8[0], k8[0], k, k, pos), "differ"),
        (lambda: kv_append(torch.zeros(2, 16 * 128), k, k, cs, cs, pos, n_heads=6), "multiple"),
        (lambda: kv_read(k.half(), k.half()), "fp16 caches"),
        (lambda: kv_read(k, k), "scales exactly"),
        (lambda: kv_read(k, k, k_scale=words), "scales exactly"),
        (lambda: kv_read(k8, k8, k_scale=s8, v_scale=s8, n_rows=0), "positive"),
        (lambda: kv_read(k8, k8, k_scale=s8, v_scale=s8, n_rows=-1), r"2\^31"),
        (lambda: kv_read(k8, k8, k_scale=s8, v_scale=s8, dtype=torch.float64), "float16 or float32"),
        (lambda: kv_read(k8, k8, k_scale=s8, v_scale=s8, out=s8), "pair"),
        (lambda: kv_read(k8, k8, k_scale=s8, v_scale=s8, out=(s8, None)), "pair"),
        (lambda: kv_read(k, k, k_scale=words, v_scale=words), "device"),
    ]
    for call, text in bad:
        with pytest.raises(ValueError, match=text):
            call()
