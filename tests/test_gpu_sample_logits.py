"""Sampling on the GPU against its definition in 64 bits."""

from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

NAMES = ("temperature", "top_k", "top_p", "min_p")


def dev(a):
    import torch

    return None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()


def row_kept(x, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(indices in rising order, weights) of the kept tokens of one row."""
    x = np.asarray(x, np.float64)
    can = np.flatnonzero(x > -np.inf)
    if len(can) == 0:
        return can, np.zeros(0)
    order = can[np.argsort(-x[can], kind="stable")]
    with np.errstate(all="ignore"):
        d = np.where(x[order] == x[order[0]], 0.0, x[order] - x[order[0]])
        w = np.where(d == -np.inf, 0.0, np.exp(d / np.float64(temperature))) if temperature > 0 else np.zeros(len(d))
    w[0] = 1.0
    w[w < 2.0 ** -44] = 0.0
    most = len(w) if temperature > 0 else 1
    if top_k > 0:
        most = min(most, top_k)
    if top_p < 1:
        run = np.cumsum(w[:most])
        most = min(most, int(np.searchsorted(run, np.float64(top_p) * run[-1], side="left")) + 1)
    keep = np.arange(len(w)) < most
    keep &= (w >= min_p) & (w > 0)
    keep[0] = True
    ids, w = order[keep], w[keep]
    by = np.argsort(ids)
    return ids[by], w[by]


def reference(x, u, **kw):
    """(tokens, probs, room): room is how far u * total lies from the nearest border of the running sum, in totals."""
    tokens, probs, room = [], [], []
    for i in range(len(x)):
        ids, w = row_kept(x[i], **{name: a[i] for name, a in kw.items()})
        if len(ids) == 0:
            tokens.append(-1), probs.append(0.0), room.append(1.0)
            continue
        run = np.cumsum(w)
        at = np.clip(np.float64(u[i]) if u[i] > 0 else 0.0, 0, 1 - 2.0 ** -53) * run[-1]
        j = min(int(np.searchsorted(run, at, side="right")), len(ids) - 1)
        tokens.append(int(ids[j])), probs.append(w[j] / run[-1])
        room.append(np.abs(np.concatenate([[0.0 if at > 0 else 1.0], run[:-1]]) - at).min() / run[-1] if at > 0 else 1)
    return np.array(tokens, np.int32), np.array(probs), np.array(room)


def run(x, u, **kw):
    from asdsl.kernels import sample_logits

    tokens, probs = sample_logits(dev(x), dev(np.asarray(u, np.float32)), **{n: dev(a) for n, a in kw.items()})
    return tokens.cpu().numpy(), probs.cpu().numpy()


def check(x, u, **kw):
    got, probs = run(x, u, **kw)
    want, share, room = reference(x, u, **kw)
    # a weight is off by half a unit of 2^-43 and by 2^-43 of fp64 rounding at most, a sum of n of them by n of those:
    # beside a border by less than that either token is the definition's
    near = room < x.shape[1] * 2.0 ** -42
    assert near.sum() <= 1 + len(near) // 50  # draws beside a border are rare
    assert np.array_equal(got[~near], want[~near]), (got, want)
    # rounded to fp32 once; the sums' own error is far below
    same = got == want
    assert (np.abs(probs - share)[same] <= share[same] * (2.0 ** -24 + x.shape[1] * 2.0 ** -42)).all()


def settings(rng, rows, form):
    kw = {}
    if form != "plain":
        kw["temperature"] = rng.uniform(0.3, 2.0, rows).astype(np.float32)
    if form in ("k", "all"):
        kw["top_k"] = rng.choice([0, 1, 2, 7, 40, 1000, 10 ** 6, -3], rows).astype(np.int32)
    if form in ("p", "all"):
        kw["top_p"] = rng.choice([0.0, 0.1, 0.5, 0.9, 0.99, 1.0, 1.5, -1.0], rows).astype(np.float32)
    if form in ("min", "all"):
        kw["min_p"] = rng.choice([0.0, 0.01, 0.2, 1.0, 1.5, -1.0], rows).astype(np.float32)
    return kw


@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (2, 255), (5, 256), (4, 1023), (3, 1025), (7, 4099), (30, 5003),
                                        (2, 32003), (3, 131072), (2, 200064), (600, 300), (1, 1 << 20)])
@pytest.mark.parametrize("form", ["plain", "temperature", "k", "p", "min", "all"])
def test_sample(gpu, rows, vocab, form):
    rng = np.random.default_rng(rows * vocab + len(form))
    x = (rng.standard_normal((rows, vocab)) * 3).astype(np.float32)
    check(x, rng.random(rows, dtype=np.float32), **settings(rng, rows, form))


@pytest.mark.parametrize("vocab", [9, 9001, 70000])
def test_flat_and_tied_logits(gpu, vocab):
    """All or many logits equal: cuts fall among ties, by index; the lists overflow."""
    rng = np.random.default_rng(vocab)
    rows = 24
    for x in (np.zeros((rows, vocab), np.float32), np.round(rng.standard_normal((rows, vocab))).astype(np.float32),
              (rng.integers(0, 2, (rows, vocab)) * -0.0).astype(np.float32)):
        kw = {"top_k": rng.integers(1, vocab + 1, rows).astype(np.int32),
              "top_p": rng.uniform(0.05, 1, rows).astype(np.float32)}
        u = rng.random(rows, dtype=np.float32)
        for use in (("top_k",), ("top_p",), ("top_k", "top_p")):
            check(x, u, **{n: kw[n] for n in use})
        # a tie's border is a whole number of equal weights, which the sums hold exactly
        half = {"top_k": np.full(rows, 4, np.int32), "top_p": np.full(rows, 0.5, np.float32)}
        if not x.any():
            got = run(x, np.full(rows, 0.5, np.float32), **half)
            assert (got[0] == 1).all() and (got[1] == 0.5).all()


@pytest.mark.parametrize("vocab", [70001, 200064])
def test_a_far_logit_leaves_the_others_in_one_bin(gpu, vocab):
    """Bins reach from the largest logit to the smallest: one below the others makes them wide, and more tokens of
    different logits lie in the cut's bin than its lists hold."""
    rng = np.random.default_rng(vocab)
    rows = 6
    x = (rng.standard_normal((rows, vocab)) * np.array([.02, .1, .3, .02, .1, .3])[:, None]).astype(np.float32)
    x[:, 17] = -5.0
    x[3:, 5] = 3.0
    kw = {"top_k": rng.integers(1, vocab, rows).astype(np.int32), "top_p": rng.uniform(0.05, 1, rows).astype(np.float32),
          "min_p": np.array([0, .8, .3, 0, .04, .04], np.float32)}
    u = rng.random(rows, dtype=np.float32)
    for use in (("top_k",), ("top_p",), ("top_k", "top_p"), ("top_p", "min_p"), tuple(kw)):
        check(x, u, **{n: kw[n] for n in use})


def test_logits_for_tokens_that_do_not_exist(gpu):
    """-10000 for many tokens, a far one, and cuts that fall among the smallest that have a weight."""
    rng = np.random.default_rng(4)
    rows, vocab = 8, 40000
    x = (rng.standard_normal((rows, vocab)) * 2).astype(np.float32)
    x[:, 33000:] = -10000.0
    x[1::2, rng.permutation(vocab)[:30000]] = -65504.0
    x[2, 77] = -31.0 + x[2].max()  # nearly no weight
    x[3, 0] = -1e30
    for t, p in ((1.0, .999999), (.5, .9), (2.0, .95), (30.0, .99), (1e4, .5), (1e-3, .9)):
        check(x, rng.random(rows, dtype=np.float32), temperature=np.full(rows, t, np.float32),
              top_p=np.full(rows, p, np.float32))
        check(x, rng.random(rows, dtype=np.float32), temperature=np.full(rows, t, np.float32),
              top_k=np.array([5, 100, 9000, 3, 32999, 33001, 39999, 1], np.int32))


@pytest.mark.parametrize("rows,vocab", [(1, 8), (3, 1021), (2, 4096), (600, 3000), (2, 70000)])
def test_bins_that_end_beside_the_largest_logit(gpu, rows, vocab):
    """Four neighbouring tokens without weight but for the two largest logits, a bit of fp32 apart, and -31 among all
    others, which is out of the largest one's reach but not of theirs: the bins' range is that bit, and tokens with
    weights lie some 10^10 of its 255th parts below it.  Others of a lane and of its later steps alike."""
    top = np.float32(0.3)
    x = np.full((rows, vocab), -0.7, np.float32)
    x[:, 1::4] = -31.0
    for i in range(rows):
        at = (4 * 307 * i + (i % 2) * 2048) % max(4, (vocab - 4) // 4 * 4)  # in a lane's first steps and in later ones
        x[i, at:at + 4] = top, np.nextafter(top, np.float32(0)), -np.inf, -np.inf
    rng = np.random.default_rng(vocab)
    k = rng.integers(3, vocab // 2 + 1, rows).astype(np.int32)
    k[0] = 3
    p = rng.uniform(0.5, 0.99, rows).astype(np.float32)
    u = rng.random(rows, dtype=np.float32)
    for kw in ({"top_k": k}, {"top_p": p}, {"top_k": k, "top_p": p},
               {"top_k": k, "temperature": np.full(rows, 1e-3, np.float32)},
               {"top_p": p, "min_p": np.full(rows, 0.3, np.float32)}):
        check(x, u, **kw)
    if rows == 1:  # the share of the third token is that of three kept ones
        got, probs = run(x, [0.999], top_k=k)
        assert got[0] == 4 and abs(probs[0] - np.exp(-1) / (2 + np.exp(-1))) < 1e-6


@pytest.mark.parametrize("rows,vocab", [(1, 5000), (5, 5003), (3, 70001), (2, 200064), (1, 1 << 20)])
@pytest.mark.parametrize("others", [False, True])
def test_more_infinite_logits_than_the_lists_hold(gpu, rows, vocab, others):
    """Rows of +inf, all or (others) three of four of them, share evenly: cuts among the first of them, where the
    topmost part of a selection reaches past the largest rank that there is."""
    rng = np.random.default_rng(rows + vocab)
    x = np.full((rows, vocab), np.inf, np.float32)
    if others:
        away = rng.random((rows, vocab)) < 0.25
        x[away] = rng.choice(np.array([3e38, 0, -np.inf, np.nan], np.float32), int(away.sum()))
    u = rng.random(rows, dtype=np.float32)
    for k in (2, 3, 4, 100, 385, 1025, vocab // 2, vocab):
        check(x, u, top_k=np.full(rows, k, np.int32))
    for p in (1e-6, 3.3 / vocab, 70.7 / vocab, 0.4):
        check(x, u, top_p=np.full(rows, p, np.float32))
    check(x, u, top_k=np.full(rows, 400, np.int32), top_p=np.full(rows, 0.011, np.float32))
    if not others:  # the last of four
        got, probs = run(x, np.full(rows, 0.8, np.float32), top_k=np.full(rows, 4, np.int32))
        assert (got == 3).all() and (probs == 0.25).all()


def test_every_kept_token_by_its_share(gpu):
    """u over a grid draws each kept token as often as its share, in index order, and no other."""
    rng = np.random.default_rng(1)
    vocab, rows = 700, 4096
    x = np.repeat((rng.standard_normal((1, vocab)) * 2).astype(np.float32), rows, axis=0)
    u = (np.arange(rows) / rows).astype(np.float32)
    kw = {"temperature": 0.8, "top_k": 60, "top_p": 0.9, "min_p": 0.02}
    ids, w = row_kept(x[0], **{n: np.float32(v) if n != "top_k" else v for n, v in kw.items()})
    got, probs = run(x, u, **{n: np.full(rows, v, np.int32 if n == "top_k" else np.float32) for n, v in kw.items()})
    assert (np.diff(got) >= 0).all() and set(got) <= set(ids.tolist())
    share = w / w.sum()
    times = np.array([(got == i).sum() for i in ids])
    assert (np.abs(times - share * rows) <= 1).all()
    assert np.allclose(probs, share[np.searchsorted(ids, got)], rtol=2.0 ** -23)


def test_odd_values(gpu):
    """Infinities, NaN, rows with nothing to draw, zeros of both signs, settings and numbers past their ranges."""
    x = np.zeros((12, 70), np.float32)
    x[0] = -np.inf
    x[1] = np.nan
    x[2, 5], x[2, 60], x[2, 61] = np.inf, np.inf, np.nan
    x[3], x[3, 33] = -np.inf, -3e38
    x[4, ::2] = -0.0
    x[5, 7:9] = 3e38, -3e38
    x[6, 0], x[6, 69] = np.nan, 1.0
    u = np.array([.5, .5, .75, .9, .51, .3, .999999, 1.0, -2.0, np.nan, 5.0, 0.0], np.float32)
    got, probs = run(x, u)
    assert got[:4].tolist() == [-1, -1, 60, 33] and got[5] == 7 and probs[:4].tolist() == [0, 0, .5, 1]
    assert got[4] == 35 and got[6] == 69 and got[7] == 69 and got[8] == 0 and got[9] == 0 and got[10] == 69
    assert got[11] == 0
    check(x[2:7], u[2:7])
    nan = np.full(12, np.nan, np.float32)
    assert np.array_equal(run(x, u, top_p=nan, min_p=nan)[0], got)
    # NaN beside a cut: of both signs, in rows whose first bin is cut
    y = (np.arange(4 * 300).reshape(4, 300) % 7 * -1e-3).astype(np.float32)
    y[:, 5::9], y[:, 6::9] = np.nan, -np.float32(np.nan)
    y[1:, 7] = 2.0
    cuts = {"top_k": np.array([100, 100, 3, 250], np.int32), "top_p": np.array([.5, .9, .3, 1], np.float32)}
    for use in (("top_k",), ("top_p",), ("top_k", "top_p")):
        check(y, u[:4], **{n: cuts[n] for n in use})
    for t in (0.0, -1.0, np.nan):  # the first of the ranking
        first = run(x, u, temperature=np.full(12, t, np.float32))
        assert first[0].tolist() == [-1, -1, 5, 33, 0, 7, 69, 0, 0, 0, 0, 0]
        assert first[1].tolist() == [0, 0] + [1] * 10
    hot = run(x, u, temperature=np.full(12, np.inf, np.float32))[0]  # all that are finite share evenly
    assert hot[0] == -1 and hot[2] == 60 and hot[3] == 33 and hot[5] == 21 and hot[4] == 35
    cold = run(x[4:6], u[4:6], temperature=np.full(2, 1e-45, np.float32))[0]
    assert cold.tolist() == [35, 7]


def test_one_row_another_stream_and_graphs(gpu):
    """One row's [vocab]; two captured graphs replayed in turn with new numbers and logits, eager calls between."""
    import torch

    from asdsl.kernels import control_logits, sample_logits

    rng = np.random.default_rng(9)
    rows, vocab = 3, 50257
    x = dev((rng.standard_normal((rows, vocab)) * 3).astype(np.float32))
    u = dev(rng.random(rows, dtype=np.float32))
    kw = {"temperature": dev(np.array([.7, 1.0, 1.3], np.float32)), "top_k": dev(np.array([50, 0, 3000], np.int32)),
          "top_p": dev(np.array([.9, .95, .8], np.float32)), "min_p": dev(np.array([.02, 0, .01], np.float32))}
    words = dev(rng.integers(-2 ** 31, 2 ** 31, (rows, (vocab + 31) // 32)).astype(np.int32))
    one = sample_logits(x[0], u[:1], top_p=kw["top_p"][:1])
    assert one[0].tolist() == sample_logits(x[:1], u[:1], top_p=kw["top_p"][:1])[0].tolist()

    def step():
        y, _ = control_logits(x, allowed=words, pick=False)
        return sample_logits(y, u, **kw)

    side = torch.cuda.Stream()
    graphs = []
    for _ in range(2):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = step()
        graphs.append((g, out))
    for i in range(8):
        x.copy_(dev((rng.standard_normal((rows, vocab)) * 3).astype(np.float32)))
        u.copy_(dev(rng.random(rows, dtype=np.float32)))
        want = step()
        torch.cuda.synchronize()
        g, out = graphs[i % 2]
        with torch.cuda.stream(side):
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
        allowed = (words.cpu().numpy().astype(np.uint32)[np.arange(rows), want[0].cpu() // 32] >>
                   (want[0].cpu().numpy() % 32).astype(np.uint32)) & 1
        assert allowed.all()


def test_two_streams_at_once_and_the_same_each_time(gpu):
    import torch

    from asdsl.kernels import sample_logits

    rng = np.random.default_rng(10)
    x = [dev((rng.standard_normal((16, 60000)) * 3).astype(np.float32)) for _ in range(2)]
    u = dev(rng.random(16, dtype=np.float32))
    p = dev(rng.uniform(0.5, 1, 16).astype(np.float32))
    want = [sample_logits(a, u, top_p=p) for a in x]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for a, st in zip(x, streams):
            with torch.cuda.stream(st):
                got.append(sample_logits(a, u, top_p=p))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1])


@pytest.mark.parametrize("rows,vocab", [(1, 200064), (600, 300), (40, 5003)])
def test_work_of_the_filters_that_a_call_has(gpu, rows, vocab):
    """Without top-k and top-p a call allocates its outputs and a weight for 1024 tokens, no bins and lists; its
    results in a buffer of that size alone are those beside all filters that keep everything."""
    import torch

    from asdsl.kernels import sample_logits

    rng = np.random.default_rng(vocab)
    x, u = dev((rng.standard_normal((rows, vocab)) * 3).astype(np.float32)), dev(rng.random(rows, dtype=np.float32))
    t, m = dev(rng.uniform(0.3, 2, rows).astype(np.float32)), dev(rng.uniform(0, 0.1, rows).astype(np.float32))
    k, p = torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.ones(rows, device="cuda")
    size = gpu.LIB.asdsl_sample_logits_work_bytes_cuts
    for kw in ({}, {"temperature": t}, {"min_p": m}, {"temperature": t, "min_p": m}, {"top_k": k}, {"top_p": p}):
        before = torch.cuda.memory_stats()["requested_bytes.all.allocated"]
        got = sample_logits(x, u, **kw)
        taken = torch.cuda.memory_stats()["requested_bytes.all.allocated"] - before
        assert taken == size(rows, vocab, "top_k" in kw or "top_p" in kw) + 8 * rows
        want = sample_logits(x, u, **{**kw, "top_k": k, "top_p": p})
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_more_than_2_31_logits(gpu):
    import torch

    from asdsl.kernels import sample_logits

    rows, vocab = 11_000, 200_064
    assert rows * vocab > 2 ** 31
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.empty((rows, vocab), device="cuda").normal_(generator=gen).mul_(3)
    u = torch.rand(rows, generator=gen, device="cuda")
    p = torch.full((rows,), 0.9, device="cuda")
    at = [0, 1, rows // 2, rows - 1]
    tokens, probs = sample_logits(x, u, top_p=p)
    want, share, room = reference(x[at].cpu().numpy(), u[at].cpu().numpy(), top_p=p[at].cpu().numpy())
    assert (room > vocab * 2.0 ** -42).all() and np.array_equal(tokens[at].cpu().numpy(), want)
    assert np.allclose(probs[at].cpu().numpy(), share, rtol=2.0 ** -23)


def test_a_chat_over_4_bits_drawn_token_by_token(gpu):
    """A step as a program runs it: new rows into a 4-bit cache, attention over it, logits, a mask and penalties, the
    token drawn; captured twice and replayed in turn, against eager steps, and each token against its logits in 64 bits."""
    import torch

    from asdsl.kernels import attention_window, control_logits, kv_append, sample_logits

    rng = np.random.default_rng(11)
    n, h, kvh, d, rows, vocab, steps = 3, 8, 2, 64, 40, 5003, 7
    width = (h + 2 * kvh) * d
    embed = dev(rng.standard_normal((vocab, width)).astype(np.float32))
    head = dev((rng.standard_normal((h * d, vocab)) / 8).astype(np.float32))
    angle = np.arange(rows)[:, None] * 100.0 ** (-np.arange(16) / 16)
    cos, sin = dev(np.cos(angle).astype(np.float32)), dev(np.sin(angle).astype(np.float32))
    may = rng.random((n, (vocab + 31) // 32 * 32)) < 0.8
    words = dev(np.packbits(may, axis=1, bitorder="little").view(np.int32))
    kw = {"temperature": dev(np.array([.8, 1.0, .5], np.float32)), "top_k": dev(np.array([40, 0, 500], np.int32)),
          "top_p": dev(np.array([.95, .9, 1], np.float32)), "min_p": dev(np.array([0, .01, .001], np.float32))}
    uniform = dev(rng.random((steps, n), dtype=np.float32))
    penalty = torch.full((n,), 1.2, device="cuda")

    def chat():
        return {"k": torch.zeros((n, kvh, rows, d // 2), dtype=torch.uint8, device="cuda"),
                "ks": torch.zeros((n, kvh, rows, d // 32), dtype=torch.int16, device="cuda"),
                "v": torch.zeros((n, kvh, rows, d // 2), dtype=torch.uint8, device="cuda"),
                "vs": torch.zeros((n, kvh, rows, d // 32), dtype=torch.int16, device="cuda"),
                "pos": torch.zeros(n, dtype=torch.int32, device="cuda"),
                "tokens": torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda"),
                "history": torch.full((n, steps + 1), -1, dtype=torch.int32, device="cuda")}

    def step(c, u):
        q = kv_append(embed[c["tokens"].long()], c["k"], c["v"], cos, sin, c["pos"], n_heads=h, k_scale=c["ks"],
                      v_scale=c["vs"])
        out = attention_window(q, c["k"], c["v"], c["pos"], n_heads=h, k_scale=c["ks"], v_scale=c["vs"])
        y, _ = control_logits(torch.mm(out, head), history=c["history"], repetition=penalty, allowed=words, pick=False)
        tokens, probs = sample_logits(y, u, **kw)
        c["history"].scatter_(1, c["pos"].long()[:, None], tokens[:, None])
        c["tokens"].copy_(tokens)
        c["pos"].add_(1)
        return y, tokens, probs

    eager, other = chat(), chat()
    u = torch.empty(n, device="cuda")
    spare = chat()
    graphs = []
    for _ in range(2):
        step(spare, u.zero_())
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(other, u)
        graphs.append((g, out))
    for name, t in chat().items():
        other[name].copy_(t)
    for i in range(steps):
        want = step(eager, uniform[i])
        u.copy_(uniform[i])
        graphs[i % 2][0].replay()
        torch.cuda.synchronize()
        for a, b in zip(want, graphs[i % 2][1]):
            assert torch.equal(a, b)
        assert all(torch.equal(eager[name], other[name]) for name in eager)
        token, share, room = reference(want[0].cpu().numpy(), uniform[i].cpu().numpy(),
                                       **{name: t.cpu().numpy() for name, t in kw.items()})
        sure = room > vocab * 2.0 ** -42
        assert sure.any() and np.array_equal(want[1].cpu().numpy()[sure], token[sure])
        assert may[np.arange(n), want[1].cpu().numpy()].all()
