"""Continuations of one prompt decoded together (BranchDecoder): the pass
against the single-sequence engine, and the control of its tokens."""

from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

VOCAB = 2048


def engine(kv="fp16", seed=31, max_seq=256):
    from asdsl.engine import DecodeConfig, DecodeEngine

    cfg = DecodeConfig(hidden=1024, ffn=1536, vocab=VOCAB, n_layers=2, n_heads=8, n_kv_heads=4, rotary_dim=96,
                       max_seq=max_seq, kv_format=kv)
    return DecodeEngine.synthetic(cfg, seed=seed)


def prompt_of(n, seed=1):
    return np.random.default_rng(seed).integers(0, VOCAB, n).tolist()


# The projections are the step's own and the attention sums in another order:
# now and then an int8 activation code falls on the other side (0.0049 of the
# logits at two layers); four times that.
NEAR = 0.02


@pytest.mark.parametrize("kv", ["fp16", "int8"])
@pytest.mark.parametrize("n,prompt", [(1, 1), (3, 40), (17, 130), (40, 67)])
def test_forward_follows_the_single_sequence_step(gpu, kv, n, prompt):
    import torch

    from asdsl.inference.branches import BranchDecoder

    eng, other = engine(kv), engine(kv)
    ids, steps = prompt_of(prompt), 3
    own = np.random.default_rng(n).integers(0, VOCAB, (steps, n))
    b = BranchDecoder(eng, n, steps)
    b.start(ids)
    got = torch.stack([b.forward(own[i]).clone() for i in range(steps)])
    assert b.own_pos.tolist() == [steps] * n
    c = eng.cfg
    for j in sorted({0, n // 2, n - 1}):
        other.reset_session()
        other.prefill(ids)
        for i in range(steps):
            want = other.forward_token(int(own[i, j]), prompt + i)
            assert float((got[i, j] - want).norm() / want.norm()) < NEAR, (i, j)
        # the first layer's rows come from the same projection: the same bits
        rows = other.layers[0]["k_cache"][:, prompt:prompt + steps], other.layers[0]["v_cache"][:, prompt:prompt + steps]
        assert torch.equal(b.k[0, j], rows[0]) and torch.equal(b.v[0, j], rows[1])
        if kv == "int8":
            assert torch.equal(b.k_scale[0, j], other.layers[0]["k_scale"][:, prompt:prompt + steps])
            assert torch.equal(b.v_scale[0, j], other.layers[0]["v_scale"][:, prompt:prompt + steps])
    # the prompt's rows were only read
    for a, z in zip(eng.layers, other.layers):
        assert torch.equal(a["k_cache"][:, :prompt], z["k_cache"][:, :prompt])
        assert not a["k_cache"][:, prompt:c.max_seq].any()


def test_generate_is_greedy_and_begins_with_the_best_tokens(gpu):
    import torch

    from asdsl.inference.branches import BranchDecoder

    eng, other = engine(), engine()
    ids = prompt_of(30)
    out = BranchDecoder(eng, 4, 20).generate(ids, eos=())
    assert [len(r) for r in out] == [20] * 4
    other.prefill(ids)
    best = torch.topk(other.logits, 4).indices.tolist()
    assert [r[0] for r in out] == best
    for r in out:
        other.reset_session()
        other.prefill(ids)
        for i, t in enumerate(r[:-1]):
            logits = other.forward_token(t, len(ids) + i)
            # the chosen token is the step's largest, or as near as the two passes are
            assert float(logits.max() - logits[r[i + 1]]) <= 2 * NEAR * float(logits.norm()) / VOCAB ** 0.5 * 4


def test_graph_replays_are_the_eager_steps(gpu):
    import torch

    from asdsl.inference.branches import BranchDecoder, TokenControl

    control = TokenControl(repetition=1.2, frequency=0.3, presence=0.2, bias={5: 2.0, 7: -3.0})
    res = []
    for graphs in (True, False):
        eng = engine("int8")
        eng.graph_calls = graphs
        b = BranchDecoder(eng, 5, 24)
        out = b.generate(prompt_of(50), control=control, eos=())
        res.append((out, b.logits.clone(), b.k.clone(), b.own_pos.tolist()))
        assert (b._graph is not None) == graphs
        # a second prompt of another length with the same decoder
        res[-1] += (b.generate(prompt_of(33, 2), 9, control=control, eos=()),)
        torch.cuda.synchronize()
    a, z = res
    assert a[0] == z[0] and a[3] == z[3] and a[4] == z[4] and len(a[4][0]) == 9
    assert torch.equal(a[1], z[1]) and torch.equal(a[2], z[2])


def test_control_bears_on_every_choice(gpu):
    import torch

    from asdsl.inference.branches import BranchDecoder, TokenControl

    b = BranchDecoder(engine(), 3, 30)
    out = b.generate(prompt_of(20), control=TokenControl(frequency=1000.0), eos=())
    assert all(len(set(r)) == 30 for r in out)
    even = np.full(VOCAB // 32, 0x55555555, np.uint32).view(np.int32)
    out = b.generate(prompt_of(20), control=TokenControl(allowed=torch.from_numpy(even)), eos=())
    assert all(t % 2 == 0 for r in out for t in r)
    asked = []

    def mask(rows):
        """Token 10 (or one of 10, 11, 12 to begin with), then 20, then nothing."""
        asked.append([list(r) for r in rows])
        words = np.zeros((3, VOCAB // 32), np.int32)
        words[:, 0] = {0: 7 << 10, 1: 1 << 20}.get(len(rows[0]), 0)
        return torch.from_numpy(words)
    out = b.generate(prompt_of(20), control=TokenControl(allowed=mask), eos=())
    assert sorted(out) == [[10, 20], [11, 20], [12, 20]]
    assert asked[0] == [[], [], []] and [r[1:] for r in asked[2]] == [[20]] * 3
    # an end-of-sequence token ends a continuation and is not returned
    out = b.generate(prompt_of(20), control=TokenControl(bias={42: 1e6}), eos=(42,))
    assert [] in out and all(42 not in r for r in out)


def test_refusals(gpu):
    from asdsl.inference.branches import BranchDecoder, TokenControl

    eng = engine(max_seq=64)
    for bad in (lambda: BranchDecoder(eng, 0, 4), lambda: BranchDecoder(eng, 257, 4), lambda: BranchDecoder(eng, 2, 0),
                lambda: BranchDecoder(eng, 2, 65)):
        with pytest.raises(ValueError):
            bad()
    b = BranchDecoder(eng, 2, 10)
    with pytest.raises(RuntimeError):
        b.step()
    for bad in (lambda: b.start([]), lambda: b.start(prompt_of(55)), lambda: b.start([VOCAB]),
                lambda: b.start([1], TokenControl(repetition=0.0)), lambda: b.start([1], TokenControl(bias={VOCAB: 1.0})),
                lambda: b.generate([1], 11)):
        with pytest.raises(ValueError):
            bad()
    b.start(prompt_of(54))
    for bad in ([1], [1, VOCAB], [1, -1]):
        with pytest.raises(ValueError):
            b.forward(bad)
    for _ in range(10):
        b.step()
    with pytest.raises(ValueError):
        b.step()
    assert b.generate(prompt_of(5), 0) == [[], []]


def test_a_mask_row_for_each_continuation(gpu):
    """Every choice, the first among them, is one that the continuation's own row allows."""
    import torch

    from asdsl.inference.branches import BranchDecoder, TokenControl

    n = 5
    b = BranchDecoder(engine(), n, 6)
    v = np.arange(VOCAB)
    may = np.stack([v % n == j for j in range(n)])
    may[4] = may[3]  # two rows with one set: distinct first tokens
    words = np.packbits(may, axis=1, bitorder="little").view(np.int32)
    out = b.generate(prompt_of(20), control=TokenControl(allowed=torch.from_numpy(words)), eos=())
    assert all(may[j, t] for j in range(n) for t in out[j]) and out[3][0] != out[4][0]
    other = engine()  # the first tokens are each row's best after the prompt
    other.prefill(prompt_of(20))
    want = other.logits.reshape(-1).cpu().numpy()
    for j in range(4):
        assert out[j][0] == int(np.argmax(np.where(may[j], want, -np.inf)))
    assert out[4][0] == int(np.argmax(np.where(may[4] & (v != out[3][0]), want, -np.inf)))
    only = np.zeros((n, VOCAB // 32), np.int32)
    only[:, 0] = 0b1111  # four tokens for five continuations
    with pytest.raises(ValueError, match="fewer than"):
        b.start(prompt_of(20), TokenControl(allowed=torch.from_numpy(only)))
    with pytest.raises(RuntimeError):  # and nothing to step from
        b.step()
