"""int8 caches whose value scales are far apart: every key counts by its
product of weight and scale, however loud the values of small weight are."""

from __future__ import annotations

import numpy as np
import ops_reference as ref
import pytest
from test_gpu_attention_ops import dev

pytestmark = pytest.mark.gpu


def make(rng, pattern, s, n_kv, keys, d):
    """q direction, key caches (codes, scales, wide) with scores of about t[i],
    and the value scales: one loud key of weight e^-18, or scores that rise
    while the scales fall by 2^s over the keys, or the other way round."""
    x = np.linspace(0, 1, keys)
    t, level = {"one": (np.where(np.arange(keys) == 3, -18.0, 0.0), np.where(np.arange(keys) == 3, s, 0.0)),
                "last": (np.where(np.arange(keys) == keys - 2, -18.0, 0.0), np.where(np.arange(keys) == keys - 2, s, 0.0)),
                "rising": (0.69 * s * (x - 1), s * (1 - x)), "falling": (-0.69 * s * x, s * x)}[pattern]
    u = rng.choice([-1.0, 1.0], d)
    k = t[None, :, None] * u + 0.3 * rng.standard_normal((n_kv, keys, d))
    scale = (np.abs(k).reshape(n_kv, keys, -1, 64).max(-1) / 127).astype(np.float32)
    codes = np.rint(k / np.repeat(scale, 64, -1)).astype(np.int8)
    vscale = np.exp2(level[None, :, None] + rng.uniform(-1, 1, (n_kv, keys, d // 64))).astype(np.float32)
    return u, codes, scale, ref.wide(codes, scale), vscale


def bounded(got, q, kw, codes, vscale):
    """Each value within fp32's bound, and 2^-33 of the row's largest product of
    weight and scale a key, times its code (fp16 parts end at 2^-25, the largest
    product is held at 2^8 or more).  The row as a whole within what random
    roundings make of a score: sqrt(d) of 2^-24 of its magnitudes (2^-20 for both
    operands' parts), four of its own, and as much for the sums over the keys."""
    want, bound = ref.attend_row(q, kw, ref.wide(codes, vscale))
    z = kw @ q / np.sqrt(len(q))
    w = np.exp(z - z.max())
    most = (w[:, None] / w.sum() * vscale).max()
    mags = np.max(np.abs(kw) @ np.abs(q)) / np.sqrt(len(q))
    near = np.linalg.norm(got - want) / np.linalg.norm(want)
    return (np.abs(got - want) <= bound + len(kw) * 2.0 ** -33 * 127 * most).all() and \
        near <= 2.0 ** -20 * (mags + 1) + 2.0 ** -22 * np.abs(z).max()


@pytest.mark.parametrize("tokens,h,kvh,d,rows", [(1, 8, 2, 128, 4000), (5, 24, 8, 128, 300), (90, 6, 2, 128, 16400),
                                                 (1, 8, 1, 64, 300), (128, 8, 1, 64, 216000)])
@pytest.mark.parametrize("pattern,s", [("one", 12), ("one", 20), ("one", 24), ("one", 30), ("last", 24), ("rising", 30),
                                       ("rising", 60), ("falling", 30), ("falling", 60)])
def test_window(gpu, tokens, h, kvh, d, rows, pattern, s):
    import torch

    from asdsl.kernels import attention_window

    rng = np.random.default_rng(s + tokens)
    keys, p0 = 250, 250 - tokens
    u, kc, ks, kw, vs = make(rng, pattern, s, kvh, keys, d)
    vc = rng.integers(-127, 128, (kvh, keys, d)).astype(np.int8)
    q = (u / np.sqrt(d) + 0.3 * rng.standard_normal((tokens, h, d))).astype(np.float32)

    def cache(x):
        full = torch.zeros((1, kvh, rows, x.shape[-1]), dtype=torch.int8 if x.dtype == np.int8 else torch.float32,
                           device="cuda")
        full[0, :, :keys] = dev(x)
        return full
    got = attention_window(dev(q[None]), cache(kc), cache(vc), dev(np.array([p0], np.int32)), k_scale=cache(ks),
                           v_scale=cache(vs)).cpu().numpy()[0]
    for t in sorted({0, tokens // 2, tokens - 1}):
        m = p0 + t + 1
        for a in range(h):
            j = a // (h // kvh)
            assert bounded(got[t, a], q[t, a].astype(np.float64), kw[j, :m], vc[j, :m], vs[j, :m]), (t, a)


@pytest.mark.parametrize("n,h,kvh,d,plen", [(3, 8, 2, 128, 700), (96, 8, 2, 128, 8299)])
@pytest.mark.parametrize("pattern,s", [("one", 20), ("one", 24), ("rising", 60), ("falling", 30)])
def test_prefix(gpu, n, h, kvh, d, plen, pattern, s):
    from asdsl.kernels import attention_prefix

    rng = np.random.default_rng(s + n)
    u, kc, ks, kw, vs = make(rng, pattern, s, kvh, plen, d)
    vc = rng.integers(-127, 128, (kvh, plen, d)).astype(np.int8)
    own = np.zeros((n, kvh, 1, d), np.int8)
    own_scale = np.ones((n, kvh, 1, d // 64), np.float32)
    q = (u / np.sqrt(d) + 0.3 * rng.standard_normal((n, h, d))).astype(np.float32)
    got = attention_prefix(dev(q), dev(kc), dev(vc), dev(own), dev(own), dev(np.full(n, -1, np.int32)),
                           k_prefix_scale=dev(ks), v_prefix_scale=dev(vs), k_scale=dev(own_scale),
                           v_scale=dev(own_scale)).cpu().numpy()
    for i in sorted({0, n // 2, n - 1}):
        for a in range(h):
            j = a // (h // kvh)
            assert bounded(got[i, a], q[i, a].astype(np.float64), kw[j], vc[j], vs[j]), (i, a)
