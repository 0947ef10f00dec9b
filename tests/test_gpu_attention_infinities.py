"""fp16 caches that hold infinities and NaN where tokens see them: what the
definition makes of them, and nothing else in the output."""

from __future__ import annotations

import numpy as np
import ops_reference as ref
import pytest
from test_gpu_attention_ops import dev

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


def same(got, want, bound, what):
    """Equal where the definition is infinite or NaN, near it elsewhere; a row
    all of whose scores are -inf is zero."""
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf]) and np.isfinite(got[~inf & ~np.isnan(want)]).all(), what
    fin = np.isfinite(want)
    assert (np.abs(got[fin] - want[fin]) <= bound[fin]).all(), what


def attend(q, k, v):
    """softmax(k q / sqrt(d)) v with its infinities: a score of +inf or NaN
    makes the row NaN; a key of score -inf has no weight, which times an
    infinite value is NaN; any other key's infinite value is the dim's."""
    d = len(q)
    with np.errstate(invalid="ignore"):
        s = (k * q).sum(axis=1)
    if np.isnan(s).any() or (s == INF).any():
        return np.full(d, NAN), np.zeros(d)
    ok = s > -INF
    if not ok.any():
        return np.zeros(d), np.zeros(d)
    out, bound = ref.attend_row(q, k[ok], np.where(np.isfinite(v[ok]), v[ok], 0.0))
    for x in (INF, -INF):
        with np.errstate(invalid="ignore"):
            out = out + np.where((v[ok] == x).any(axis=0), x, 0.0)
    return np.where(np.isnan(v).any(axis=0) | ~np.isfinite(v[~ok]).all(axis=0), NAN, out), bound


# tokens, heads, kv heads, head_dim, rows, first position, window (few-row and many-row forms, one piece and several)
CASES = [(1, 8, 4, 128, 64, 40, 0), (1, 8, 4, 128, 3000, 2900, 0), (1, 14, 7, 64, 900, 700, 300), (9, 14, 7, 128, 200, 100, 0),
         (40, 14, 7, 64, 400, 200, 60), (90, 14, 7, 128, 2000, 300, 0), (70, 56, 7, 64, 8000, 300, 0),
         (130, 28, 7, 128, 3000, 200, 100)]


@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("kind", ["key down", "value up", "value down", "both", "all"])
def test_window(gpu, case, kind):
    from asdsl.kernels import attention_window

    tokens, h, kvh, d, rows, p0, win = case
    rng = np.random.default_rng(tokens + rows)
    n = 1 if tokens < 90 else 3
    q = rng.standard_normal((n, tokens, h, d)).astype(np.float32)
    q[..., 0] = np.abs(q[..., 0]) + 0.1  # dim 0 is positive in every query, dim 1 zero in every third token
    q[:, ::3, :, 1] = 0.0
    k = rng.standard_normal((n, kvh, rows, d)).astype(np.float16)
    v = rng.standard_normal((n, kvh, rows, d)).astype(np.float16)
    mid, late = p0 - 5, p0 + tokens - 2 if tokens > 2 else p0 - 1
    if kind == "key down":
        k[:, :, (0, mid, late), 0] = -INF  # scores of -inf: the keys drop out
        k[:, 0, late, 2] = INF             # with both signs of q[2]: also inf - inf
    elif kind == "value up":
        v[:, :, mid, 3], v[:, 0, late, d - 1] = INF, NAN
    elif kind == "value down":
        v[:, :, mid, 3], v[:, :, late, 3], v[:, 0, late, 9] = -INF, INF, -INF
    elif kind == "both":
        k[:, :, mid, 0], v[:, :, mid, 4], v[:, :, late, 8] = -INF, INF, INF
    else:
        k[:, 0, mid, 0], k[:, 0, late, 1] = INF, -INF
        if kvh > 1:
            k[:, 1, late, 5], k[:, 1:, :, 0] = NAN, -INF  # all seen keys out in the other heads
    got = attention_window(dev(q), dev(k), dev(v), dev(np.full(n, p0, np.int32)), window=win).cpu().numpy()
    kw, vw = k.astype(np.float64), v.astype(np.float64)
    for t in sorted({0, 1, 2, tokens // 2, tokens - 3, tokens - 2, tokens - 1} & set(range(tokens))):
        at = ref.seen_rows(p0 + t, rows, win, 0)
        for i in (0, n - 1):
            for a in range(h):
                j = a // (h // kvh)
                want, bound = attend(q[i, t, a].astype(np.float64), kw[i, j, at], vw[i, j, at])
                same(got[i, t, a], want, bound, (kind, i, t, a))


@pytest.mark.parametrize("n,h,kvh,d,plen", [(3, 8, 4, 128, 700), (70, 4, 2, 128, 8099), (5, 8, 4, 64, 0), (130, 16, 16, 64, 5999)])
def test_prefix(gpu, n, h, kvh, d, plen):
    from asdsl.kernels import attention_prefix

    rng = np.random.default_rng(n)
    q = rng.standard_normal((n, h, d)).astype(np.float32)
    q[..., 0] = np.abs(q[..., 0]) + 0.1
    kp = rng.standard_normal((kvh, plen, d)).astype(np.float16)
    vp = rng.standard_normal((kvh, plen, d)).astype(np.float16)
    ko = rng.standard_normal((n, kvh, 9, d)).astype(np.float16)
    vo = rng.standard_normal((n, kvh, 9, d)).astype(np.float16)
    own = np.array([i % 10 - 1 for i in range(n)], np.int32)
    if plen:
        kp[:, (3, plen - 1), 0] = -INF
        vp[0, plen // 2, 6] = INF
        vp[1, 5, 6], kp[1, 6, 2] = -INF, INF
    ko[:, :, 2, 0] = -INF
    vo[::2, :, 4, 11] = INF
    got = attention_prefix(dev(q), dev(kp), dev(vp), dev(ko), dev(vo), dev(own)).cpu().numpy()
    for i in sorted({0, 1, 2, 3, 4, n // 2, n - 2, n - 1} & set(range(n))):
        m = int(own[i]) + 1
        for a in range(h):
            j = a // (h // kvh)
            kw = np.concatenate([kp[j], ko[i, j, :m]]).astype(np.float64)
            vw = np.concatenate([vp[j], vo[i, j, :m]]).astype(np.float64)
            want, bound = attend(q[i, a].astype(np.float64), kw, vw)
            same(got[i, a], want, bound, (i, a))


@pytest.mark.parametrize("tokens,rows", [(1, 64), (1, 5000), (64, 6000)])
def test_an_infinite_value_of_next_to_no_weight(gpu, tokens, rows):
    """A key e^-400 below the others, early or late: its value is infinite in
    the definition, however the keys are split."""
    from asdsl.kernels import attention_window

    rng = np.random.default_rng(3)
    h, kvh, d, p0 = 24, 8, 128, rows - tokens
    u = rng.choice([-1.0, 1.0], d)
    q = np.broadcast_to(u, (1, tokens, h, d)).astype(np.float32)
    for at in (1, p0 - 1):
        k = (0.01 * rng.standard_normal((1, kvh, rows, d))).astype(np.float16)
        k[:, :, at] = (-36 * u).astype(np.float16)  # a score of -36 * 128 / sqrt(128)
        v = rng.standard_normal((1, kvh, rows, d)).astype(np.float16)
        v[:, :, at, 5], v[:, :, at, 6] = INF, -INF
        got = attention_window(dev(q), dev(k), dev(v), dev(np.array([p0], np.int32))).cpu().numpy()
        assert (got[..., 5] == INF).all() and (got[..., 6] == -INF).all()
        assert np.isfinite(np.delete(got, (5, 6), axis=-1)).all()


@pytest.mark.parametrize("kv", ["fp16", "int8"])
@pytest.mark.parametrize("tokens,h,kvh,d,rows", [(1, 12, 4, 128, 300), (5, 12, 4, 64, 2000), (90, 12, 4, 128, 16400)])
def test_queries_that_are_not_finite(gpu, kv, tokens, h, kvh, d, rows):
    """Their own rows alone are NaN, whatever shares a tile with them."""
    import torch

    from asdsl.kernels import attention_window
    from test_gpu_attention_ops import make_cache

    rng = np.random.default_rng(tokens)
    p0 = 200
    q = rng.standard_normal((1, tokens, h, d)).astype(np.float32)
    k, ks, kw = make_cache(rng, kv, 1, kvh, rows, d)
    v, vs, vw = make_cache(rng, kv, 1, kvh, rows, d)
    spoilt = [(tokens - 1, 2, NAN), (0, 7, INF), (tokens // 2, 11, -INF)]
    for t, a, x in spoilt:
        q[0, t, a, 5] = x
    got = attention_window(dev(q), k, v, dev(np.array([p0], np.int32)), k_scale=ks, v_scale=vs).cpu().numpy()
    for t in sorted({0, 1, tokens // 2, tokens - 1} & set(range(tokens))):
        for a in range(h):
            if any((t, a) == x[:2] for x in spoilt):
                assert np.isnan(got[0, t, a]).all(), (t, a)
                continue
            m = p0 + t + 1
            want, bound = ref.attend_row(q[0, t, a].astype(np.float64), kw[0, a // 3, :m], vw[0, a // 3, :m])
            assert (np.abs(got[0, t, a] - want) <= bound).all(), (t, a)
    assert int(torch.from_numpy(np.isnan(got).any(axis=-1)).sum()) == len(spoilt)
