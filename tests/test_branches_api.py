"""Refusals of the branch step at the C ABI, before any HIP call."""

from __future__ import annotations

import ctypes


def model():
    from asdsl.engine import _Layer, _Model

    layers = (_Layer * 1)()
    for name, _ in _Layer._fields_:
        if name != "fatrelu_threshold":
            setattr(layers[0], name, 256)
    m = _Model(hidden=1024, ffn=1024, vocab=100, n_layers=1, n_heads=8, n_kv_heads=4, head_dim=128, rotary_dim=96,
               max_seq=64, gs_attn=32, gs_ffn=128, gs_lm=128, rms_eps=1e-5)
    m.layers = ctypes.cast(layers, ctypes.POINTER(_Layer))
    for name in ("embed", "rms_out", "lm_meta", "lm_quant", "rope_cos", "rope_sin"):
        setattr(m, name, 256)
    m._hold = layers
    return m


def test_branch_step_refusals():
    from asdsl import _hip
    from asdsl.inference.branches import _BranchLayer

    lib, m = _hip.LIB, model()
    own = (_BranchLayer * 1)(_BranchLayer(256, 256, None, None))
    one = ctypes.c_void_p(256)
    size = lib.asdsl_decode_branches_work_bytes(ctypes.byref(m), 4, 32, 32)
    assert size > 0

    def f(own=own, n=4, prefix=32, rows=32, tokens=one, logits=one, work=one, nbytes=size):
        return lib.asdsl_decode_branches(ctypes.byref(m), own, n, prefix, rows, tokens, one, logits, work, nbytes, None)

    def refused(status, text):
        assert status == _hip.ASDSL_ERR_INVALID_ARGUMENT and text in _hip.last_error(), _hip.last_error()
    refused(lib.asdsl_decode_branches(None, own, 4, 32, 32, one, one, one, one, size, None), "null model")
    refused(f(own=None), "null")
    refused(f(tokens=None), "null")
    refused(f(work=None), "null")
    for n, prefix, rows in ((0, 32, 32), (257, 32, 32), (4, -1, 32), (4, 33, 32), (4, 32, 0)):
        refused(f(n=n, prefix=prefix, rows=rows), "max_seq")
        assert lib.asdsl_decode_branches_work_bytes(ctypes.byref(m), n, prefix, rows) == 0
    refused(f(nbytes=size - 1), "work buffer")
    refused(f(logits=ctypes.c_void_p(260)), "aligned")
    refused(f(own=(_BranchLayer * 1)(_BranchLayer(256, 264, None, None))), "own caches")
    m.kv_format = 1
    refused(f(), "scales")
