"""Windowed and shared-prefix attention at sizes about the kernels' two forms,
for few and for many query rows, against the definitions in 64 bits.  The form
goes by rows a KV head, keys, head dim and cache type; most of the sizes here
take the one for many rows, which for int8 caches asks for long caches (of
which little is seen)."""

from __future__ import annotations

import numpy as np
import ops_reference as ref
import pytest
from test_gpu_attention_ops import check, dev, make_cache

pytestmark = pytest.mark.gpu

# n_seq, tokens, heads, kv heads, head_dim, cache, rows, positions, window, sinks
WINDOW = [
    (1, 33, 24, 8, 128, "fp16", 6000, [700], 0, 0),
    (1, 33, 24, 8, 128, "int8", 6000, [700], 0, 0),
    (1, 130, 8, 2, 128, "int8", 4000, [1900], 0, 0),
    (8, 70, 8, 1, 128, "fp16", 1000, [0, 1, 31, 32, 500, 929, 930, -69], 500, 5),
    (20, 9, 16, 4, 128, "int8", 700, [-9, -8, -5, 0, 20, 23, 24, 300, 690, 691, 695, 699, 700, 2**31 - 9, -2**31, 64,
                                      127, 128, 129, 255], 0, 0),
    (20, 9, 16, 4, 128, "fp16", 700, [-9, -8, -5, 0, 20, 23, 24, 300, 690, 691, 695, 699, 700, 2**31 - 9, -2**31, 64,
                                      127, 128, 129, 255], 650, 40),
    (3, 257, 12, 4, 128, "fp16", 500, [0, 200, 243], 490, 0),
    (20, 128, 8, 8, 128, "fp16", 128, [0] * 20, 0, 0),
    (16, 90, 6, 2, 128, "int8", 400, [20 * i for i in range(16)], 60, 31),
    (16, 90, 6, 2, 128, "fp16", 400, [20 * i for i in range(16)], 1, 0),
    (1, 17, 1, 1, 128, "fp16", 70000, [3], 0, 0),
    (1, 200, 16, 4, 64, "fp16", 20000, [300], 0, 0),
    (1, 200, 16, 4, 64, "int8", 20000, [300], 0, 0),
    (6, 65, 12, 6, 64, "int8", 4000, [3935, 100, -64, 0, 3999, 77], 3900, 3),
    (40, 65, 12, 3, 64, "fp16", 200, [3 * i for i in range(40)], 170, 2),
    (1, 64, 24, 8, 128, "int8", 8000, [700], 0, 0),
    (1, 130, 8, 2, 128, "int8", 8000, [1900], 0, 0),
    (20, 30, 16, 4, 128, "int8", 700, [-30, -29, -5, 0, 20, 23, 24, 300, 670, 671, 695, 699, 700, 2**31 - 9, -2**31,
                                       64, 127, 128, 129, 255], 0, 0),
    (60, 90, 6, 2, 128, "int8", 400, [5 * i for i in range(60)], 60, 31),
    (1, 128, 8, 1, 64, "int8", 214000, [300], 0, 0),
    (1, 131, 8, 1, 64, "int8", 256000, [-3], 255000, 3),
    (130, 65, 12, 3, 64, "fp16", 200, [3 * (i % 46) for i in range(130)], 170, 2),
    (12, 96, 12, 6, 64, "fp16", 1600, [131 * i for i in range(12)], 0, 0),
]


@pytest.mark.parametrize("case", WINDOW, ids=lambda c: str(c[:7] + c[8:]))
def test_window(gpu, case):
    from asdsl.kernels import attention_window

    n, t, h, kvh, d, kv, rows, pos, win, sinks = case
    rng = np.random.default_rng(rows + t)
    q = rng.standard_normal((n, t, h, d)).astype(np.float32)
    k, ks, kw = make_cache(rng, kv, n, kvh, rows, d)
    v, vs, vw = make_cache(rng, kv, n, kvh, rows, d)
    want, bound = ref.window(q, kw, vw, pos, win, sinks)
    p = dev(np.array(pos, np.int32))
    got = attention_window(dev(q), k, v, p, window=win, sinks=sinks, k_scale=ks, v_scale=vs)
    check(got, want, bound, str(case))
    again = attention_window(dev(q), k, v, p, window=win, sinks=sinks, k_scale=ks, v_scale=vs)
    assert np.array_equal(again.cpu().numpy(), got.cpu().numpy())


@pytest.mark.parametrize("n,rows,win,sinks", [(1, 9000, 0, 0), (24, 400, 40, 3), (1, 400, 0, 0)])
@pytest.mark.parametrize("d", [128, 64])
@pytest.mark.parametrize("kv", ["fp16", "int8"])
def test_unseen_rows_do_not_reach_the_output(gpu, kv, d, n, rows, win, sinks):
    """NaN, infinities and the types' lowest values in rows that no token sees;
    then, in a row that only the last token sees, also values that are finite
    and far from the others.  (The last case takes the form for few rows.)"""
    import torch

    from asdsl.kernels import attention_window

    rng = np.random.default_rng(5)
    tokens, p0 = 90, 200
    h, kvh = (6, 2) if d == 128 else (24, 12)
    q = rng.standard_normal((n, tokens, h, d)).astype(np.float32)
    k, ks, kw = make_cache(rng, kv, n, kvh, rows, d)
    v, vs, vw = make_cache(rng, kv, n, kvh, rows, d)
    want, bound = ref.window(q, kw, vw, [p0] * n, win, sinks)
    seen = np.zeros(rows, bool)
    for t in range(tokens):
        seen[ref.seen_rows(p0 + t, rows, win, sinks)] = True
    bad = np.flatnonzero(~seen)
    for i, x in enumerate((float("nan"), float("inf"), float("-inf"), -65504.0)):
        at = torch.from_numpy(bad[i::4]).cuda()
        if kv == "fp16":
            k[:, :, at], v[:, :, at] = x, x
        else:
            ks[:, :, at], vs[:, :, at] = x, x
    pos = dev(np.array([p0] * n, np.int32))

    def call():
        return attention_window(dev(q), k, v, pos, window=win, sinks=sinks, k_scale=ks, v_scale=vs)
    check(call(), want, bound)
    last = p0 + tokens - 1
    for x in (float("nan"), float("inf")) + ((65504.0,) if kv == "fp16" else (1e6, 1e20)):
        if kv == "fp16":
            k[:, :, last], v[:, :, last] = 1.0, x
        else:
            vs[:, :, last] = x
        got = call()
        check(got[:, :-1].contiguous(), want[:, :-1], bound[:, :-1], str(x))
        if not np.isfinite(x):
            assert not torch.isfinite(got[:, -1]).any()


@pytest.mark.parametrize("d,n,tokens,h,kvh,rows,win", [(128, 1, 90, 6, 2, 16400, 0), (128, 64, 90, 6, 2, 400, 200),
                                                     (64, 1, 128, 8, 1, 216000, 0)])
def test_unseen_rows_of_int8_caches(gpu, d, n, tokens, h, kvh, rows, win):
    """As above, at sizes where int8 caches take the form for many rows."""
    import torch

    from asdsl.kernels import attention_window

    rng = np.random.default_rng(15)
    p0 = 200
    q = rng.standard_normal((n, tokens, h, d)).astype(np.float32)
    k, ks, kw = make_cache(rng, "int8", n, kvh, rows, d)
    v, vs, vw = make_cache(rng, "int8", n, kvh, rows, d)
    want, bound = ref.window(q, kw, vw, [p0] * n, win, 3)
    seen = np.zeros(rows, bool)
    for t in range(tokens):
        seen[ref.seen_rows(p0 + t, rows, win, 3)] = True
    bad = np.flatnonzero(~seen)
    for i, x in enumerate((float("nan"), float("inf"), float("-inf"), 1e20)):
        at = torch.from_numpy(bad[i::4]).cuda()
        ks[:, :, at], vs[:, :, at] = x, x
    pos = dev(np.array([p0] * n, np.int32))

    def call():
        return attention_window(dev(q), k, v, pos, window=win, sinks=3, k_scale=ks, v_scale=vs)
    check(call(), want, bound)
    last = p0 + tokens - 1
    for x in (float("nan"), float("inf"), 1e6, 1e20):
        vs[:, :, last] = x
        got = call()
        check(got[:, :-1].contiguous(), want[:, :-1], bound[:, :-1], str(x))
        if not np.isfinite(x):
            assert not torch.isfinite(got[:, -1]).any()


def test_prefix_of_a_long_int8_cache_of_narrow_heads(gpu):
    """Some rows of a call that takes the form for many rows."""
    from asdsl.kernels import attention_prefix

    rng = np.random.default_rng(16)
    n, h, d, plen, rows = 128, 8, 64, 214001, 5
    q = rng.standard_normal((n, h, d)).astype(np.float32)
    kp, kps, kpw = make_cache(rng, "int8", 1, plen + 9, d)
    vp, vps, vpw = make_cache(rng, "int8", 1, plen + 9, d)
    ko, kos, kow = make_cache(rng, "int8", n, 1, rows, d)
    vo, vos, vow = make_cache(rng, "int8", n, 1, rows, d)
    for s in (kps, vps):
        s[:, plen:] = float("nan")
    own = np.array([i % 6 - 1 for i in range(n)], np.int32)
    got = attention_prefix(dev(q), kp, vp, ko, vo, dev(own), prefix_len=plen, k_prefix_scale=kps, v_prefix_scale=vps,
                           k_scale=kos, v_scale=vos)
    for i in (0, 1, 15, 16, 17, 127):
        for a in (0, 7):
            m = int(own[i]) + 1
            want, bound = ref.attend_row(q[i, a].astype(np.float64), np.concatenate([kpw[0, :plen], kow[i, 0, :m]]),
                                         np.concatenate([vpw[0, :plen], vow[i, 0, :m]]))
            assert (np.abs(got[i, a].cpu().numpy() - want) <= bound).all(), (i, a)


def test_tokens_outside_the_cache_beside_infinite_rows(gpu):
    """A padded token shares its tiles with tokens that see every key: zero all
    the same, where theirs are not finite."""
    import torch

    from asdsl.kernels import attention_window

    rng = np.random.default_rng(9)
    n, tokens, h, kvh, d, rows = 48, 40, 8, 8, 128, 128
    for kv in ("fp16", "int8"):
        k, ks, _ = make_cache(rng, kv, n, kvh, rows, d)
        v, vs, _ = make_cache(rng, kv, n, kvh, rows, d)
        (v if vs is None else vs)[:, :, 3] = float("inf")
        q = dev(rng.standard_normal((n, tokens, h, d)).astype(np.float32))
        first = [rows - 7 if i % 2 else -10 for i in range(n)]
        got = attention_window(q, k, v, dev(np.array(first, np.int32)), k_scale=ks, v_scale=vs)
        for i, p in enumerate(first):
            at = np.arange(tokens) + p
            outside = torch.from_numpy((at < 0) | (at >= rows)).cuda()
            sees = torch.from_numpy((at >= 3) & (at < rows)).cuda()
            assert (got[i][outside] == 0).all() and not torch.isfinite(got[i][sees]).any()
            assert torch.isfinite(got[i][~outside & ~sees]).all()


@pytest.mark.parametrize("tokens,rows", [(5, 300), (64, 300), (64, 6000)])
def test_window_value_scales_of_a_wide_range(gpu, tokens, rows):
    """Value scales 2^11 apart.  A key's weight times its scale is held with an
    error of at most half of fp16's least step (2^-25), the row's largest weight
    being 2^8 or more and the largest scale in [1, 2): 2^-33 of the product of
    the two, for each key's codes."""
    from asdsl.kernels import attention_window

    rng = np.random.default_rng(8)
    n, h, kvh, d, p0 = 1, 24, 8, 128, 200
    q = rng.standard_normal((n, tokens, h, d)).astype(np.float32)
    k, ks, kw = make_cache(rng, "int8", n, kvh, rows, d)
    codes = rng.integers(-127, 128, (n, kvh, rows, d)).astype(np.int8)
    scale = np.exp2(rng.uniform(-11, 0, (n, kvh, rows, 2))).astype(np.float32)
    vw = ref.wide(codes, scale)
    want, bound = ref.window(q, kw, vw, [p0], 0, 0)
    bound = bound + (p0 + tokens) * 2.0 ** -33 * 127 * scale.max()
    got = attention_window(dev(q), k, dev(codes), dev(np.array([p0], np.int32)), k_scale=ks, v_scale=dev(scale))
    check(got, want, bound)


@pytest.mark.parametrize("loud", [1e-3, 300.0])
@pytest.mark.parametrize("kv", ["fp16", "int8"])
def test_window_quiet_and_loud_queries(gpu, kv, loud):
    """Flat and one-hot weights.  Beside a one-hot weight the others lose their
    bits: all are held in fp16 parts, off by at most 2^-25 where the largest is
    2^8 or more, so by 2^-33 of the row's largest weight times its key's values
    (which shows where an int8 cache's one value is exactly 0)."""
    from asdsl.kernels import attention_window

    rng = np.random.default_rng(6)
    q = (rng.standard_normal((1, 140, 8, 128)) * loud).astype(np.float32)
    k, ks, kw = make_cache(rng, kv, 1, 2, 9000, 128)
    v, vs, vw = make_cache(rng, kv, 1, 2, 9000, 128)
    want, bound = ref.window(q, kw, vw, [300], 0, 0)
    bound = bound + (300 + 140) * 2.0 ** -33 * np.abs(vw).max()
    got = attention_window(dev(q), k, v, dev(np.array([300], np.int32)), k_scale=ks, v_scale=vs).cpu().numpy()
    assert (np.abs(got - want) <= bound).all()


# n_seq, heads, kv heads, head_dim, cache, prefix rows, prefix_len, own rows, own positions
PREFIX = [
    (70, 4, 2, 128, "fp16", 8100, 8099, 5, [i % 6 - 1 for i in range(70)]),
    (70, 4, 2, 128, "int8", 8100, 8099, 5, [i % 6 - 1 for i in range(70)]),
    (40, 24, 8, 128, "int8", 2113, 2113, 9, [i % 10 - 1 for i in range(39)] + [9]),
    (43, 6, 2, 128, "fp16", 9000, 8500, 140, [(i * 17) % 141 - 1 for i in range(42)] + [-2]),
    (130, 16, 16, 64, "fp16", 6000, 5999, 4, [i % 4 for i in range(130)]),
    (64, 8, 2, 64, "int8", 26000, 25601, 3, [i % 4 - 1 for i in range(64)]),
    (96, 8, 2, 128, "int8", 8300, 8299, 5, [i % 6 - 1 for i in range(96)]),
    (64, 16, 8, 128, "int8", 6200, 6151, 70, [(i * 13) % 71 - 1 for i in range(64)]),
    (130, 24, 12, 64, "fp16", 5300, 5300, 4, [i % 4 for i in range(130)]),
]


@pytest.mark.parametrize("case", PREFIX, ids=lambda c: str(c[:8]))
def test_prefix(gpu, case):
    from asdsl.kernels import attention_prefix

    n, h, kvh, d, kv, prows, plen, rows, own = case
    rng = np.random.default_rng(n * 100 + h)
    q = rng.standard_normal((n, h, d)).astype(np.float32)
    kp, kps, kpw = make_cache(rng, kv, kvh, prows, d)
    vp, vps, vpw = make_cache(rng, kv, kvh, prows, d)
    ko, kos, kow = make_cache(rng, kv, n, kvh, rows, d)
    vo, vos, vow = make_cache(rng, kv, n, kvh, rows, d)
    want, bound = ref.prefix(q, kpw, vpw, plen, kow, vow, own)

    def call():
        return attention_prefix(dev(q), kp, vp, ko, vo, dev(np.array(own, np.int32)), prefix_len=plen,
                                k_prefix_scale=kps, v_prefix_scale=vps, k_scale=kos, v_scale=vos)
    check(call(), want, bound, str(case))
    for t, s in ((kp, kps), (vp, vps)):
        (t if s is None else s)[:, plen:] = float("nan")
    for t, s in ((ko, kos), (vo, vos)):
        for i, m in enumerate(own):
            if m < rows:
                (t if s is None else s)[i, :, max(m + 1, 0):] = float("inf")
    check(call(), want, bound, "unseen rows")


def test_two_graphs_at_once(gpu):
    """Two captured calls, each with splits to join in a work buffer of its own,
    replayed together on two streams, with eager calls between the replays."""
    import torch

    from asdsl.kernels import attention_prefix, attention_window

    gen = torch.Generator(device="cuda").manual_seed(2)

    def halves(*shape):
        return torch.randn(shape, generator=gen, device="cuda").half()
    k, v, ko, vo = halves(8, 5000, 128), halves(8, 5000, 128), halves(20, 8, 30, 128), halves(20, 8, 30, 128)
    pos = torch.tensor([4000], dtype=torch.int32, device="cuda")
    own = torch.arange(-1, 19, dtype=torch.int32, device="cuda")
    qs = [torch.randn(s, generator=gen, device="cuda") for s in ((1, 64, 24, 128), (20, 24, 128))]
    calls = [lambda q: attention_window(q, k, v, pos), lambda q: attention_prefix(q, k, v, ko, vo, own)]
    streams, graphs, outs = [torch.cuda.Stream() for _ in qs], [], []
    for q, call, stream in zip(qs, calls, streams):
        call(q)
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=stream):
            outs.append(call(q))
    for i in range(4):
        for q in qs:
            q.normal_(generator=gen)
        want = [call(q) for q, call in zip(qs, calls)]
        torch.cuda.synchronize()
        for g, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                g.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b), i


@pytest.mark.parametrize("h,n", [(64, 270_000), (12, 1_400_000)])
def test_more_than_2_31_query_values(gpu, h, n):
    """Queries, outputs and qkv rows past 2^31 elements, in both forms."""
    import torch

    from asdsl.kernels import attention_window, kv_append

    d, rows, p = 128, 2, 1
    assert n * h * d > 2 ** 31
    gen = torch.Generator(device="cuda").manual_seed(4)
    qkv = torch.empty((n, (h + 2) * d), device="cuda").uniform_(-1, 1, generator=gen)
    k = torch.randn((n, 1, rows, d), generator=gen, device="cuda").half()
    v = torch.randn((n, 1, rows, d), generator=gen, device="cuda").half()
    pos = torch.full((n,), p, dtype=torch.int32, device="cuda")
    cos, sin = torch.ones((4, d // 2), device="cuda"), torch.zeros((4, d // 2), device="cuda")  # no turn
    q = kv_append(qkv, k, v, cos, sin, pos, n_heads=h)
    out = attention_window(q, k, v, pos)
    for i in (0, 1, n // 2, n - 2, n - 1):
        x = qkv[i].cpu().numpy().reshape(h + 2, d)
        assert np.array_equal(q[i].cpu().numpy().reshape(h, d), x[:h])
        kw, vw = (t[i, 0].cpu().numpy().astype(np.float64) for t in (k, v))
        assert np.array_equal(kw[p], x[h].astype(np.float16)) and np.array_equal(vw[p], x[h + 1].astype(np.float16))
        for a in (0, h - 1):
            want, bound = ref.attend_row(x[a].astype(np.float64), kw, vw)
            assert (np.abs(out[i].cpu().numpy().reshape(h, d)[a] - want) <= bound).all(), (i, a)
