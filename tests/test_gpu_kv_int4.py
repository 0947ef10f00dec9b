"""Caches of 4 bits on the GPU: append, reading back and attention, against their definitions in 64 bits."""

from __future__ import annotations

import kv4_reference as kv4
import numpy as np
import ops_reference as ref
import pytest
from test_gpu_attention_ops import PREFIX, WINDOW, check, dev

pytestmark = pytest.mark.gpu


def cache4(rng, *shape, loud=1.0):
    codes, words, wide = kv4.random_cache(rng, *shape, loud=loud)
    return dev(codes), dev(words), wide


def tables(positions, half, seed=0):
    angle = np.arange(positions)[:, None] * 10000.0 ** (-np.arange(half) / half)
    return np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)


# n_seq, tokens, heads, kv heads, head_dim, rotary, rows, positions, pos_offset
APPEND = [
    (1, 1, 24, 8, 128, 96, 64, [0], 0),
    (5, 1, 8, 4, 128, 128, 33, [0, 32, -1, 33, 7], 100),
    (1, 70, 8, 8, 64, 48, 100, [20], 3),
    (3, 9, 16, 1, 128, 32, 40, [31, 35, -4], 0),  # the second and third reach past an end
    (2, 3, 6, 2, 64, 20, 16, [0, 13], 0),  # rotary pairs that are no whole 16-byte units
    (1, 2, 4, 2, 128, 96, 30, [10], 2 ** 31 - 1),  # past the tables
]


@pytest.mark.parametrize("case", APPEND, ids=str)
@pytest.mark.parametrize("loud", [1.0, 1e-6, 1e5])
def test_append(gpu, case, loud):
    """Codes, words and every other row bit for bit."""
    from asdsl.kernels import kv_append

    n, t, h, kvh, d, rot, rows, pos, offset = case
    rng = np.random.default_rng(rows + t)
    half, positions = rot // 2, min(offset, 1000) + rows + 5
    cos, sin = tables(positions, half)
    qkv = (rng.standard_normal((n * t, (h + 2 * kvh) * d)) * loud).astype(np.float32)
    held = [kv4.random_cache(rng, n, kvh, rows, d)[:2] for _ in range(2)]
    want = [(c.copy(), w.copy()) for c, w in held]
    x = qkv.reshape(n, t, h + 2 * kvh, d)
    want_q = np.zeros((n, t, h, d))
    for i in range(n):
        for j in range(t):
            r = pos[i] + j
            p = r + offset
            if not (0 <= r < rows and 0 <= p < positions):
                continue
            y = ref.rotate(x[i, j, :h + kvh], cos[p], sin[p], half)
            want_q[i, j] = y[:h]
            for (c, w), new in zip(want, (y[h:], x[i, j, h + kvh:])):
                c[i, :, r], w[i, :, r] = kv4.quantize(new)
    (kc, kw), (vc, vw) = [(dev(c), dev(w)) for c, w in held]
    args = (dev(qkv), kc, vc, dev(cos), dev(sin), dev(np.array(pos, np.int32)))
    q = kv_append(*args, n_heads=h, pos_offset=offset, k_scale=kw, v_scale=vw)
    for got, name in ((kc, "k"), (vc, "v")):
        assert np.array_equal(got.cpu().numpy(), want[name == "v"][0]), name
    for got, name in ((kw, "k"), (vw, "v")):
        assert np.array_equal(got.cpu().numpy(), want[name == "v"][1]), name
    # two fp32 products and their sum, each off by half a step at most
    big = np.abs(x[:, :, :h]).astype(np.float64)
    bound = 3 * ref.EPS * (big + np.concatenate([big[..., half:2 * half], big[..., :half], big[..., 2 * half:]], -1))
    assert (np.abs(q.cpu().numpy().reshape(want_q.shape) - want_q) <= bound + 1e-37).all()


def test_append_borders(gpu):
    """Values on and beside the borders of codes and scales, zeros, and what is not finite."""
    from asdsl.kernels import kv_append

    rng = np.random.default_rng(3)
    rows, d = 64, 128
    x = np.zeros((rows, d), np.float32)
    for r in range(40):
        step = np.float32(np.ldexp(rng.integers(64, 128), rng.integers(-20, 4)))
        z = rng.integers(0, 16)
        v = (np.arange(d) % 31 / 2 - z) * step  # whole and half steps
        v = np.clip(v, -z * step, (15 - z) * step).astype(np.float32)
        x[r] = np.where(rng.random(d) < 0.3, np.nextafter(v, np.float32(rng.choice([-np.inf, np.inf]))), v)
    x[40] = -0.0
    x[41, 5], x[42, 70], x[43, 127], x[44, 0] = np.inf, np.nan, -np.inf, 3e38
    x[45], x[46] = np.finfo(np.float32).tiny / 8, 2.0 ** -20
    x[47:] = rng.standard_normal((rows - 47, d)) * 2.0 ** rng.integers(-24, 16, (rows - 47, 1))
    qkv = np.concatenate([x, x, x], axis=1)  # one head each
    one, zero = np.ones((rows, 1), np.float32), np.zeros((rows, 1), np.float32)
    empty = [np.full((1, 1, rows, n), 7, t) for n, t in ((d // 2, np.uint8), (d // 32, np.int16))]
    k, ks, v, vs = (dev(a) for a in (*empty, *empty))
    kv_append(dev(qkv), k, v, dev(one), dev(zero), dev(np.zeros(1, np.int32)), n_heads=1, k_scale=ks, v_scale=vs)
    codes, words = kv4.quantize(x.astype(np.float64))
    assert np.array_equal(v.cpu().numpy()[0, 0], codes) and np.array_equal(vs.cpu().numpy()[0, 0], words)
    # dims 0 and 1 are turned by no angle: a * 1 - b * 0, NaN where b is not finite
    with np.errstate(all="ignore"):
        turned = ref.rotate(x[:, None], one, zero, 1)[:, 0]
    codes, words = kv4.quantize(turned)
    assert np.array_equal(k.cpu().numpy()[0, 0], codes) and np.array_equal(ks.cpu().numpy()[0, 0], words)


@pytest.mark.parametrize("n,kvh,rows,d,n_rows,pos", [(1, 8, 40, 128, 40, None), (3, 2, 77, 64, 21, [0, 70, -5]),
                                                     (2, 1, 5, 128, 1, [4, 5]), (1, 3, 700, 64, 333, [200]),
                                                     (4, 5, 9, 128, 20, [0, -20, 9, -7])])
@pytest.mark.parametrize("kv", ["int4", "int8"])
@pytest.mark.parametrize("to", ["float16", "float32"])
def test_read(gpu, n, kvh, rows, d, n_rows, pos, kv, to):
    import torch

    from asdsl.kernels import kv_read

    rng = np.random.default_rng(rows + n_rows)
    sides, want = [], []
    for _ in range(2):
        if kv == "int4":
            codes, words, wide = kv4.random_cache(rng, n, kvh, rows, d)
            sides += [dev(codes), dev(words)]
        else:
            codes = rng.integers(-128, 128, (n, kvh, rows, d)).astype(np.int8)
            scale = rng.uniform(1e-3, 1, (n, kvh, rows, d // 64)).astype(np.float32)
            sides += [dev(codes), dev(scale)]
            wide = codes.astype(np.float32) * np.repeat(scale, 64, axis=-1)
        y = np.zeros((n, kvh, n_rows, d), np.dtype(to))
        for i in range(n):
            for j in range(n_rows):
                r = (0 if pos is None else pos[i]) + j
                if 0 <= r < rows:
                    y[i, :, j] = wide[i, :, r].astype(to)
        want.append(y)
    k, ks, v, vs = sides
    kw = {"k_scale": ks, "v_scale": vs, "dtype": getattr(torch, to), "n_rows": n_rows,
          "pos": None if pos is None else dev(np.array(pos, np.int32))}
    got = kv_read(k, v, **kw)
    for a, b in zip(got, want):
        assert a.dtype is kw["dtype"] and np.array_equal(a.cpu().numpy(), b)
    out = tuple(torch.full_like(t, 9) for t in got)
    del kw["dtype"]
    again = kv_read(k, v, out=out, **kw)
    assert again[0] is out[0] and all(torch.equal(a, b) for a, b in zip(out, got))
    if n == 1:
        flat = kv_read(k[0], v[0], **{**kw, "k_scale": ks[0], "v_scale": vs[0]}, dtype=got[0].dtype)
        assert flat[0].shape == (kvh, n_rows, d) and torch.equal(flat[1], got[1][0])


@pytest.mark.parametrize("case", [c[:5] + c[6:] for c in WINDOW], ids=str)
def test_window(gpu, case):
    from asdsl.kernels import attention_window

    n, t, h, kvh, d, rows, pos, win, sinks = case
    rng = np.random.default_rng(rows + t)
    q = rng.standard_normal((n, t, h, d)).astype(np.float32)
    k, ks, kw = cache4(rng, n, kvh, rows, d)
    v, vs, vw = cache4(rng, n, kvh, rows, d)
    want, bound = ref.window(q, kw, vw, pos, win, sinks)
    kw = {"window": win, "sinks": sinks, "k_scale": ks, "v_scale": vs}
    p = dev(np.array(pos, np.int32))
    got = attention_window(dev(q), k, v, p, **kw)
    check(got, want, bound, str(case))
    again = attention_window(dev(q.reshape(n * t, h * d)), k, v, p, n_heads=h, **kw)
    assert np.array_equal(again.cpu().numpy().reshape(q.shape), got.cpu().numpy())


@pytest.mark.parametrize("n,kvh,d,rows,win", [(40, 16, 128, 700, 0), (64, 16, 64, 1100, 200), (65, 16, 64, 1100, 0),
                                              (2, 300, 64, 530, 0), (127, 8, 64, 530, 0), (128, 8, 128, 300, 40),
                                              (129, 8, 64, 300, 0), (193, 4, 64, 530, 0), (256, 4, 128, 270, 0),
                                              (257, 4, 64, 300, 0)])
def test_window_of_many_ragged_sequences(gpu, n, kvh, d, rows, win):
    """More workgroups than run at once, which take the longest sequences first; equal positions, padded sequences."""
    from asdsl.kernels import attention_window

    rng = np.random.default_rng(n)
    pos = rng.integers(-1, rows, n)
    pos[rng.integers(0, n, n // 3)] = rows - 1
    pos[1] = rows  # outside
    q = rng.standard_normal((n, 1, kvh, d)).astype(np.float32)
    k, ks, kw = cache4(rng, n, kvh, rows, d)
    v, vs, vw = cache4(rng, n, kvh, rows, d)
    want, bound = ref.window(q, kw, vw, pos, win, 2 if win else 0)
    got = attention_window(dev(q), k, v, dev(pos.astype(np.int32)), window=win, sinks=2 if win else 0, k_scale=ks,
                           v_scale=vs)
    check(got, want, bound)


@pytest.mark.parametrize("case", [c[:4] + c[5:] for c in PREFIX], ids=lambda c: str(c[:7]))
def test_prefix(gpu, case):
    from asdsl.kernels import attention_prefix

    n, h, kvh, d, prows, plen, rows, own = case
    rng = np.random.default_rng(n * 100 + h)
    q = rng.standard_normal((n, h, d)).astype(np.float32)
    kp, kps, kpw = cache4(rng, kvh, prows, d)
    vp, vps, vpw = cache4(rng, kvh, prows, d)
    ko, kos, kow = cache4(rng, n, kvh, rows, d)
    vo, vos, vow = cache4(rng, n, kvh, rows, d)
    want, bound = ref.prefix(q, kpw, vpw, plen, kow, vow, own)
    kw = {"prefix_len": plen, "k_prefix_scale": kps, "v_prefix_scale": vps, "k_scale": kos, "v_scale": vos}
    p = dev(np.array(own, np.int32))
    got = attention_prefix(dev(q), kp, vp, ko, vo, p, **kw)
    check(got, want, bound, str(case))
    again = attention_prefix(dev(q), kp, vp, ko, vo, p, **kw)
    assert np.array_equal(again.cpu().numpy(), got.cpu().numpy())


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("tokens,win,sinks", [(1, 0, 0), (1, 40, 3), (5, 40, 3), (700, 0, 0), (900, 40, 3)])
def test_window_scales_that_are_not_finite(gpu, d, tokens, win, sinks):
    """NaN and infinite scales: rows that no token sees never reach an output, rows that some see only theirs."""
    import torch

    from asdsl.kernels import attention_window

    rng = np.random.default_rng(5)
    h, kvh, rows, p0 = 6, 2, 1500, 200
    q = rng.standard_normal((1, tokens, h, d)).astype(np.float32)
    k, ks, kw = cache4(rng, 1, kvh, rows, d)
    v, vs, vw = cache4(rng, 1, kvh, rows, d)
    some = sorted({0, 1, tokens // 2, tokens - 2, tokens - 1} & set(range(tokens)))  # the others as well, on the device
    want, bound = [np.concatenate([ref.window(q[:, j:j + 1], kw, vw, [p0 + j], win, sinks)[i] for j in some], 1)
                   for i in range(2)]
    at = torch.tensor(some, device="cuda")
    pos = dev(np.array([p0], np.int32))
    args = {"window": win, "sinks": sinks, "k_scale": ks, "v_scale": vs}
    clean = attention_window(dev(q), k, v, pos, **args)
    check(clean[:, at], want, bound)
    seen = np.zeros(rows, bool)
    for t in range(tokens):
        seen[ref.seen_rows(p0 + t, rows, win, sinks)] = True
    bad = np.flatnonzero(~seen)
    for i, word in enumerate((0x7E07, 0x7C03, -0x0400 + 3)):  # NaN, inf, -inf
        rows_at = torch.from_numpy(bad[i::3]).cuda()
        ks[:, :, rows_at], vs[:, :, rows_at] = word, word
    assert torch.equal(attention_window(dev(q), k, v, pos, **args), clean)
    # the last token's own row: no earlier token may feel it
    last = p0 + tokens - 1
    for word in (0x7E00, 0x7C0F):
        vs[:, :, last] = word
        got = attention_window(dev(q), k, v, pos, **args)
        check(got[:, at[:-1]].contiguous(), want[:, :-1], bound[:, :-1]) if tokens > 1 else None
        assert not torch.isfinite(got[:, -1]).any()
    ks[:, :, last], vs[:, :, last] = 0x7E00, 0  # a key that is NaN
    assert torch.isnan(attention_window(dev(q), k, v, pos, **args)[:, -1]).all()


def test_values_past_fp16_and_quiet_ones(gpu):
    """Scales of the largest and smallest kind beside ordinary ones."""
    from asdsl.kernels import attention_window

    rng = np.random.default_rng(8)
    h, kvh, d, rows = 4, 2, 128, 300
    q = (rng.standard_normal((1, 1, h, d)) * 1e-3).astype(np.float32)
    k, ks, kw = cache4(rng, 1, kvh, rows, d)
    for loud in (2.0 ** -15, 4000.0):
        v, vs, vw = cache4(rng, 1, kvh, rows, d, loud=loud)
        want, bound = ref.window(q, kw, vw, [rows - 1], 0, 0)
        got = attention_window(dev(q), k, v, dev(np.array([rows - 1], np.int32)), k_scale=ks, v_scale=vs)
        assert np.isfinite(want).all()
        check(got, want, bound, str(loud))


def test_far_rows_of_a_long_cache(gpu):
    """Byte offsets past 2^31 and 2^32: written, read back and attended to."""
    import torch

    from asdsl.kernels import attention_window, kv_append, kv_read

    rows, d, kvh, h, t = 20_000_000, 128, 4, 8, 100  # 5.1 GB of codes a cache
    k = torch.zeros((kvh, rows, d // 2), dtype=torch.uint8, device="cuda")
    ks = torch.zeros((kvh, rows, d // 32), dtype=torch.int16, device="cuda")
    v, vs = torch.zeros_like(k), torch.zeros_like(ks)
    rng = np.random.default_rng(2)
    qkv = rng.standard_normal((t, (h + 2 * kvh) * d)).astype(np.float32)
    one, zero = np.ones((rows // 1000, 1), np.float32), np.zeros((rows // 1000, 1), np.float32)
    first = rows - 3 - t
    x = qkv.reshape(t, h + 2 * kvh, d)
    # tables are short: outside them nothing is written, and a token's queries are zero
    pos = dev(np.array([first], np.int32))
    kv_append(dev(qkv), k, v, dev(one), dev(zero), pos, n_heads=h, k_scale=ks, v_scale=vs)
    assert not ks[:, first:].any()
    table = torch.ones((rows, 1), device="cuda"), torch.zeros((rows, 1), device="cuda")
    q = kv_append(dev(qkv), k, v, *table, pos, n_heads=h, k_scale=ks, v_scale=vs)
    codes, words = kv4.quantize(x[:, h:].astype(np.float64))
    wide = kv4.values(codes, words).transpose(1, 0, 2)
    got = kv_read(k, v, pos=pos, n_rows=t + 5, k_scale=ks, v_scale=vs, dtype=torch.float32)
    for side, y in zip(got, (wide[:kvh], wide[kvh:])):
        assert np.array_equal(side[:, :t].cpu().numpy(), y) and not side[:, t:].any()
    for n in (1, t):
        a = attention_window(q[t - n:].reshape(1, n, h, d), k, v, dev(np.array([first + t - n], np.int32)), window=64,
                             k_scale=ks, v_scale=vs)
        for j in {0, n - 1}:
            at = np.arange(t)[max(0, t - n + j - 63):t - n + j + 1]
            if len(at) < 64:
                continue
            for i in range(h):
                want, bound = ref.attend_row(q[t - n + j].cpu().numpy().reshape(h, d)[i].astype(np.float64),
                                             wide[i // 2, at], wide[kvh + i // 2, at])
                assert (np.abs(a[0, j, i].cpu().numpy() - want) <= bound).all()


def test_a_chat_captured_and_replayed(gpu):
    """Prompt and steps of two chats over 4-bit caches, as a program runs them: append, attend, read back; the step
    twice captured, replayed in turn on another stream with eager calls between, against eager runs and 64 bits."""
    import torch

    from asdsl.kernels import attention_window, kv_append, kv_read

    rng = np.random.default_rng(4)
    n, t, h, kvh, d, rows, steps = 2, 37, 12, 4, 128, 60, 6
    cos, sin = tables(rows, 48)
    cos, sin = dev(cos), dev(sin)
    width = (h + 2 * kvh) * d
    prompt = dev(rng.standard_normal((n * t, width)).astype(np.float32))
    tokens = dev(rng.standard_normal((steps, n, width)).astype(np.float32))

    def caches():
        return [torch.zeros((n, kvh, rows, w), dtype=kind, device="cuda")
                for w, kind in ((d // 2, torch.uint8), (d // 32, torch.int16)) * 2]

    def step(x, cache, pos):
        k, ks, v, vs = cache
        q = kv_append(x, k, v, cos, sin, pos, n_heads=h, k_scale=ks, v_scale=vs)
        return attention_window(q, k, v, pos, n_heads=h, k_scale=ks, v_scale=vs)

    eager, replayed = caches(), caches()
    pos = torch.zeros(n, dtype=torch.int32, device="cuda")
    first = step(prompt, eager, pos)
    assert torch.equal(step(prompt, replayed, pos), first)
    side = torch.cuda.Stream()
    x, pos = torch.empty_like(tokens[0]), torch.full((n,), t, dtype=torch.int32, device="cuda")
    pos[1] = t - 5  # the second chat was cut
    graphs = []
    torch.cuda.synchronize()
    spare = caches()
    for _ in range(2):
        with torch.cuda.stream(side):
            step(x, spare, pos)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = step(x, replayed, pos)
        graphs.append((g, out))
    for i in range(steps):
        want = step(tokens[i], eager, pos)
        x.copy_(tokens[i])
        torch.cuda.synchronize()
        g, out = graphs[i % 2]
        with torch.cuda.stream(side):
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(eager, replayed))
        k, v = (a.cpu().numpy().astype(np.float64) for a in kv_read(eager[0], eager[2], k_scale=eager[1],
                                                                    v_scale=eager[3]))
        assert np.array_equal(k, kv4.values(eager[0].cpu().numpy(), eager[1].cpu().numpy()))
        qkv = tokens[i].cpu().numpy().reshape(n, 1, h + 2 * kvh, d)
        at = pos.cpu().numpy()
        q = ref.rotate(qkv[:, :, :h], cos.cpu().numpy()[at][:, None], sin.cpu().numpy()[at][:, None], 48)
        wide, bound = ref.window(q.astype(np.float32), k, v, at, 0, 0)
        # and the queries' own rounding, half a step each of two products and a sum: 3 EPS a dim of a score
        norms = np.linalg.norm(q, axis=-1).max() * np.linalg.norm(k, axis=-1).max() / np.sqrt(d)
        extra = 2 * 4 * ref.EPS * norms * np.abs(v).max()
        assert (np.abs(out.cpu().numpy().reshape(wide.shape) - wide) <= bound + extra).all()
        pos += 1
