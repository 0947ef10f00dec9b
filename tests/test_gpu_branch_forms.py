"""The branch pass over other group sizes, head layouts and widths than
test_gpu_branches takes, against the single-sequence step."""

from __future__ import annotations

import numpy as np
import pytest
from test_gpu_branches import NEAR, VOCAB, prompt_of

pytestmark = pytest.mark.gpu


def engine(kv="fp16", gs=(32, 128), heads=(8, 4), ffn=1536, vocab=VOCAB, seed=31):
    from asdsl.engine import DecodeConfig, DecodeEngine

    cfg = DecodeConfig(hidden=128 * heads[0], ffn=ffn, vocab=vocab, n_layers=2, n_heads=heads[0], n_kv_heads=heads[1],
                       rotary_dim=96, max_seq=192, kv_format=kv, gs_attn=gs[0], gs_ffn=gs[1])
    return DecodeEngine.synthetic(cfg, seed=seed)


@pytest.mark.parametrize("gs", [(32, 128), (128, 32), (32, 32), (128, 128)])
@pytest.mark.parametrize("kv,heads,n", [("fp16", (8, 4), 3), ("int8", (12, 4), 17), ("fp16", (6, 2), 64)])
def test_forms(gpu, gs, kv, heads, n):
    follows(gs, kv, heads, n, steps=2)


def test_most_continuations(gpu):
    follows((32, 128), "int8", (8, 4), 256, steps=2)


def test_odd_sizes(gpu):
    """An odd vocabulary (rows of logits not aligned), K splits with masked units
    and empty classes of groups, a prompt of one token."""
    follows((32, 128), "fp16", (8, 8), 5, steps=3, prompt=1, ffn=3712, vocab=1003)
    follows((128, 32), "int8", (9, 3), 19, steps=3, prompt=4, ffn=1152, vocab=1003)


def follows(gs, kv, heads, n, steps, prompt=37, ffn=1536, vocab=VOCAB):
    import torch

    from asdsl.inference.branches import BranchDecoder

    eng, other = (engine(kv, gs, heads, ffn, vocab) for _ in range(2))
    ids = [t % vocab for t in prompt_of(prompt)]
    own = np.random.default_rng(n).integers(0, vocab, (steps, n))
    b = BranchDecoder(eng, n, steps)
    b.start(ids)
    got = torch.stack([b.forward(own[i]).clone() for i in range(steps)])
    for j in sorted({0, 1, n // 2, n - 2, n - 1}):
        other.reset_session()
        other.prefill(ids)
        for i in range(steps):
            want = other.forward_token(int(own[i, j]), len(ids) + i)
            assert float((got[i, j] - want).norm() / want.norm()) < NEAR, (i, j)
        at = slice(len(ids), len(ids) + steps)
        assert torch.equal(b.k[0, j], other.layers[0]["k_cache"][:, at])
        assert torch.equal(b.v[0, j], other.layers[0]["v_cache"][:, at])


def test_refused_under_the_factored_norm(gpu, monkeypatch):
    from asdsl.inference.branches import BranchDecoder

    b = BranchDecoder(engine(), 2, 4)
    b.start(prompt_of(9))
    monkeypatch.setenv("ASDSL_HIP_NORM_FACTORED", "1")
    with pytest.raises(Exception, match="factored norm"):
        b.step()
    monkeypatch.delenv("ASDSL_HIP_NORM_FACTORED")
    b.step()  # nothing was queued: the step is still to be taken
    assert b.own_pos.tolist() == [1, 1] and [len(r) for r in b.continuations()] == [2, 2]
