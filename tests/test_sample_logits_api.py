"""Refusals of sample_logits, before any HIP call: the C ABI and the Python wrapper."""

from __future__ import annotations

import pytest
from test_attention_ops_api import ODD, ONE, refused


def test_abi_refusals():
    from asdsl import _hip

    lib = _hip.LIB

    def f(ptrs=(ONE,) * 8, rows=1, vocab=100, work=ONE, nbytes=1 << 40):
        return lib.asdsl_sample_logits(*ptrs, rows, vocab, work, nbytes, None)
    for i in (0, 1, 6, 7):
        refused(f(ptrs=[None if j == i else ONE for j in range(8)]), "null")
    refused(f(rows=0), "positive")
    refused(f(vocab=0), "positive")
    refused(f(vocab=(1 << 20) + 1), "2^20")
    refused(f(rows=1 << 30, vocab=1 << 20), "2^32")
    refused(f(rows=1 << 23), "2^32")
    refused(f(work=None), "work buffer")
    refused(f(nbytes=1), "work buffer")
    refused(f(work=ODD), "aligned")
    size = lib.asdsl_sample_logits_work_bytes
    assert size(0, 5) == 0 and size(5, 0) == 0 and size(1, (1 << 20) + 1) == 0 and size(3, 200064) % 256 == 0


def test_work_bytes_without_cuts():
    """Calls without top-k and top-p need no bins and no lists, and are not refused for want of them."""
    from asdsl import _hip

    lib = _hip.LIB
    size, most = lib.asdsl_sample_logits_work_bytes_cuts, lib.asdsl_sample_logits_work_bytes
    for rows, vocab in ((1, 1), (1, 200064), (600, 300), (64, 200064), (11000, 200064)):
        assert size(rows, vocab, 1) == size(rows, vocab, -3) == most(rows, vocab)
        slices, tiles = most(rows, vocab) // (256 * 12 + 1024 * 8), rows * ((vocab + 1023) // 1024)
        # a largest and a small logit a slice, a weight for 1024 tokens
        assert tiles * 8 <= size(rows, vocab, 0) <= slices * 12 + tiles * 8 + 3 * 256 < most(rows, vocab)
    assert not any(size(rows, vocab, c) for c in (0, 1) for rows, vocab in ((0, 5), (5, 0), (1, (1 << 20) + 1)))

    def f(k, p, rows, vocab, nbytes):
        return lib.asdsl_sample_logits(ONE, ONE, ONE, k, p, ONE, ONE, ONE, rows, vocab, ONE, nbytes, None)
    for rows, vocab in ((1, 200064), (600, 300)):
        refused(f(None, None, rows, vocab, size(rows, vocab, 0) - 1), "work buffer")
        refused(f(ONE, None, rows, vocab, most(rows, vocab) - 1), "work buffer")
        refused(f(None, ONE, rows, vocab, most(rows, vocab) - 1), "work buffer")


def test_wrapper_refusals():
    import torch

    from asdsl.kernels import sample_logits

    x, u = torch.zeros(2, 40), torch.zeros(2)
    for call, text in ((lambda: sample_logits(torch.zeros(0), u), "logits"),
                       (lambda: sample_logits(None, u), "logits"),
                       (lambda: sample_logits(torch.zeros(2, 3, 4), u), "logits"),
                       (lambda: sample_logits(torch.zeros(1, 1).expand(1, (1 << 20) + 1), u), r"2\^20"),
                       (lambda: sample_logits(x.double(), u), "float32"),
                       (lambda: sample_logits(x, u), "device")):
        with pytest.raises(ValueError, match=text):
            call()
