"""Calls of more work items than one launch takes (2^32) are refused before
any HIP call, not by the launch."""

from __future__ import annotations

import ctypes

from test_attention_ops_api import ONE, refused


def test_calls_past_one_launch():
    from asdsl import _hip

    lib = _hip.LIB
    n, room = 1 << 24, 1 << 60  # workgroups of 256 lanes
    refused(lib.asdsl_kv_append_f16(*(ONE,) * 7, n, 1, 1, 1, 64, 64, 8, 0, 8, None), "2^32")
    refused(lib.asdsl_kv_append_q8(*(ONE,) * 9, n // 2, 2, 1, 1, 64, 64, 8, 0, 8, None), "2^32")
    refused(lib.asdsl_attention_window_f16kv(*(ONE,) * 5, n, 1, 1, 1, 64, 8, 0, 0, ONE, room, None), "2^32")
    refused(lib.asdsl_attention_prefix_f16kv(*(ONE,) * 7, n - 4, 1, 1, 64, 8, 8, 8, ONE, room, None), "2^32")
    # few workgroups, but 2^27 rows of pieces to join, four a workgroup
    refused(lib.asdsl_attention_prefix_f16kv(*(ONE,) * 7, 1 << 20, 128, 1, 64, 8, 8, 8, ONE, room, None), "2^32")
    for rows, vocab in ((n, 8), (1 << 14, 1 << 24)):
        refused(lib.asdsl_logits_control(ONE, ONE, ONE, None, None, None, 0, None, None, None, None, 0, None, 0, rows,
                                         vocab, ctypes.c_void_p(256), room, None), "2^32")
