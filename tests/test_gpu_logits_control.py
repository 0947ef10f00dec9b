"""Logits control on the GPU against its definition, bit for bit (each step rounds to fp32 on both sides)."""

from __future__ import annotations

import numpy as np
import ops_reference as ref
import pytest

pytestmark = pytest.mark.gpu


def dev(a):
    import torch

    return None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()


def run(logits, **kw):
    from asdsl.kernels import control_logits

    out, tokens = control_logits(dev(logits), **{k: dev(v) for k, v in kw.items()})
    return out.cpu().numpy().reshape(logits.shape), tokens.cpu().numpy()


def words_of(may):
    rows, vocab = may.shape
    pad = np.zeros((rows, (vocab + 31) // 32 * 32), bool)
    pad[:, :vocab] = may
    return np.packbits(pad, axis=1, bitorder="little").view(np.int32)


def check(logits, **kw):
    got, tokens = run(logits, **kw)
    want, best = ref.control(logits, **kw)
    assert np.array_equal(got.view(np.int32), want.view(np.int32)) or np.array_equal(got, want, equal_nan=True)
    assert np.array_equal(tokens, best)


@pytest.mark.parametrize("rows,vocab,cap", [(1, 1, 1), (1, 31, 5), (2, 33, 64), (3, 4096, 300), (2, 4097, 1000),
                                            (5, 32003, 77), (1, 200064, 5000), (9, 8193, 2)])
@pytest.mark.parametrize("form", ["all", "penalties", "bias", "mask", "none", "shared"])
def test_control(gpu, rows, vocab, cap, form):
    rng = np.random.default_rng(rows * vocab + cap)
    logits = (rng.standard_normal((rows, vocab)) * 3).astype(np.float32)
    kw = {}
    if form in ("all", "penalties", "shared"):
        kw["history"] = (rng.zipf(1.3, (rows, cap)) % (vocab + 3) - 1).astype(np.int32)  # -1 and vocab.. among them
        kw["history_len"] = rng.integers(0, cap + 1, rows).astype(np.int32)
        kw["history_len"][0] = cap + 7 if rows > 1 else cap
        kw["prompt_len"] = (kw["history_len"] // 3).astype(np.int32)
        kw["repetition"] = rng.uniform(0.8, 1.5, rows).astype(np.float32)
        kw["frequency"] = rng.uniform(-0.2, 0.7, rows).astype(np.float32)
        kw["presence"] = rng.uniform(-0.2, 0.7, rows).astype(np.float32)
    if form in ("all", "bias", "shared"):
        kw["bias"] = rng.standard_normal((rows, vocab) if form != "shared" else vocab).astype(np.float32)
    if form in ("all", "mask", "shared"):
        may = rng.random((1 if form == "shared" else rows, vocab)) < 0.3
        if form != "shared" and rows > 1:
            may[1] = False  # nothing allowed
        kw["allowed"] = words_of(may)
        if form == "shared":
            kw["allowed"] = kw["allowed"][0]
    check(logits, **kw)


def test_odd_values_and_ties(gpu):
    """Infinities and NaN, zeros of both signs, equal values, bits past the vocabulary."""
    x = np.zeros((6, 70), np.float32)
    x[0, ::2] = -0.0
    x[1] = -np.inf
    x[2] = np.nan
    x[3, 40:] = 5.0
    x[4, 10], x[4, 20], x[4, 30] = np.inf, np.nan, np.inf
    x[5] = np.finfo(np.float32).min
    may = np.ones((6, 70), bool)
    may[:, :3] = False
    words = words_of(may)
    words[:, 2] |= np.int32(-1) << np.int32(6)  # tokens 70..95 do not exist
    check(x)
    check(x, allowed=words)
    got = run(x, allowed=words)[1]
    assert got.tolist() == [3, 3, -1, 40, 10, 3]
    hist = np.array([[40, 40, 3, 10]] * 6, np.int32)
    one = np.ones(6, np.float32)
    check(x, allowed=words, history=hist, repetition=one * 2, frequency=one, presence=one)


def test_one_row_in_place_and_without_tokens(gpu):
    import torch

    from asdsl.kernels import control_logits

    rng = np.random.default_rng(1)
    x = rng.standard_normal(5000).astype(np.float32)
    hist = rng.integers(0, 5000, 40).astype(np.int32)
    rep = np.array([1.3], np.float32)
    want, best = ref.control(x[None], history=hist[None], repetition=rep)
    t = dev(x)
    out, tokens = control_logits(t, history=dev(hist), repetition=dev(rep), out=t)
    assert out is t and np.array_equal(t.cpu().numpy(), want[0]) and tokens.tolist() == best.tolist()
    out, none = control_logits(dev(x), history=dev(hist), repetition=dev(rep), pick=False)
    assert none is None and np.array_equal(out.cpu().numpy(), want[0])
    empty = torch.empty((1, 0), dtype=torch.int32, device="cuda")
    out, _ = control_logits(dev(x), history=empty, repetition=dev(rep))
    assert np.array_equal(out.cpu().numpy(), x)


def test_captured_and_replayed_with_a_growing_history(gpu):
    """Two graphs of one call, replayed in turn, the history growing on the device."""
    import torch

    from asdsl.kernels import control_logits

    rng = np.random.default_rng(2)
    rows, vocab, cap = 3, 9000, 12
    x = (rng.standard_normal((rows, vocab))).astype(np.float32)
    t, hist = dev(x), dev(np.full((rows, cap), -1, np.int32))
    length = torch.zeros(rows, dtype=torch.int32, device="cuda")
    pen = np.full(rows, 0.75, np.float32)
    kw = {"history": hist, "history_len": length, "frequency": dev(pen), "presence": dev(pen)}
    control_logits(t, **kw)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = control_logits(t, **kw)
        graphs.append((g, res))
    for i in range(cap):
        g, (out, tokens) = graphs[i % 2]
        g.replay()
        torch.cuda.synchronize()
        h = hist.cpu().numpy()
        want, best = ref.control(x, history=h, history_len=length.cpu().numpy(), frequency=pen, presence=pen)
        assert np.array_equal(out.cpu().numpy(), want) and np.array_equal(tokens.cpu().numpy(), best)
        hist[:, i] = tokens
        length += 1


def test_more_than_2_31_logits(gpu):
    import torch

    from asdsl.kernels import control_logits

    rows, vocab = 11_000, 200_064
    assert rows * vocab > 2 ** 31
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.empty((rows, vocab), device="cuda").normal_(generator=gen)
    words = torch.randint(-2 ** 31, 2 ** 31 - 1, (rows, vocab // 32), generator=gen, device="cuda").int()
    history = torch.randint(0, vocab, (rows, 50), generator=gen, device="cuda").int()
    rep = torch.empty(rows, device="cuda").uniform_(1, 2, generator=gen)
    at = [0, 1, rows // 2, rows - 1]
    host = [t[at].cpu().numpy() for t in (x, words, history, rep)]
    out, tokens = control_logits(x, history=history, repetition=rep, frequency=rep, allowed=words, out=x)
    want, best = ref.control(host[0], history=host[2], repetition=host[3], frequency=host[3], allowed=host[1])
    assert np.array_equal(out[at].cpu().numpy(), want) and np.array_equal(tokens[at].cpu().numpy(), best)
