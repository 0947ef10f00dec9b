"""Cache append, windowed attention and shared-prefix attention on the GPU
against their definitions in 64 bits."""

from __future__ import annotations

import ctypes

import numpy as np
import ops_reference as ref
import pytest

pytestmark = pytest.mark.gpu


def dev(a):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def make_cache(rng, kv, *shape, loud=1.0):
    """(device cache, device scales or None, wide values)."""
    x = (rng.standard_normal(shape) * loud).astype(np.float16)
    if kv == "fp16":
        return dev(x), None, ref.wide(x)
    codes = rng.integers(-127, 128, shape).astype(np.int8)
    scale = (rng.uniform(0.5, 1.5, (*shape[:-1], shape[-1] // 64)) * loud / 60).astype(np.float32)
    return dev(codes), dev(scale), ref.wide(codes, scale)


def check(got, want, bound, what=""):
    got = got.cpu().numpy().astype(np.float64).reshape(want.shape)
    assert np.isfinite(got).all(), what
    worst = np.max(np.abs(got - want) - bound)
    assert worst <= 0, f"{what}: {worst:.3e} over the bound"
    norm = np.linalg.norm(want)
    # random roundings: sqrt(128) of 2^-24 of the magnitudes in a score, some ten of them
    assert norm == 0 or np.linalg.norm(got - want) / norm < 1e-5, what
    zero = (want == 0).all(axis=-1)
    assert (got[zero] == 0).all(), what


# n_seq, tokens, heads, kv heads, head_dim, cache, rows, positions, window, sinks
WINDOW = [
    (1, 1, 24, 8, 128, "fp16", 64, [0], 0, 0),
    (1, 1, 24, 8, 128, "fp16", 700, [513], 0, 0),
    (1, 1, 24, 8, 128, "int8", 700, [699], 100, 4),
    (3, 1, 8, 4, 128, "fp16", 333, [332, -1, 17], 64, 2),
    (5, 1, 8, 8, 64, "int8", 130, [0, 63, 64, 129, 130], 0, 0),
    (2, 1, 16, 1, 128, "fp16", 200, [199, 31], 33, 64),
    (2, 1, 48, 2, 64, "int8", 97, [96, 32], 1, 0),
    (1, 1, 40, 1, 128, "fp16", 2100, [2050], 0, 0),
    (1, 2, 24, 8, 128, "int8", 150, [100], 0, 0),
    (2, 5, 8, 4, 64, "fp16", 100, [-2, 97], 7, 1),
    (1, 7, 24, 8, 128, "fp16", 300, [0], 1, 0),
    (3, 16, 8, 4, 128, "int8", 256, [0, 100, 250], 31, 5),
    (1, 33, 12, 4, 128, "fp16", 256, [31], 0, 0),
    (1, 65, 16, 4, 64, "int8", 512, [200], 64, 130),
    (2, 70, 8, 1, 128, "fp16", 200, [0, 129], 40, 4),
    (1, 130, 6, 2, 128, "int8", 400, [63], 100, 4),
    (1, 130, 6, 2, 64, "fp16", 150, [65], 0, 0),
    (1, 257, 4, 4, 128, "fp16", 700, [300], 129, 3),
    (1, 300, 3, 1, 128, "int8", 300, [0], 300, 0),
    (1, 64, 4, 2, 128, "fp16", 1000, [900], 1, 1),
]


@pytest.mark.parametrize("case", WINDOW, ids=str)
def test_window(gpu, case):
    from asdsl.kernels import attention_window

    n, t, h, kvh, d, kv, rows, pos, win, sinks = case
    rng = np.random.default_rng(hash(case[:5]) % 1000 + rows)
    q = rng.standard_normal((n, t, h, d)).astype(np.float32)
    k, ks, kw = make_cache(rng, kv, n, kvh, rows, d)
    v, vs, vw = make_cache(rng, kv, n, kvh, rows, d)
    want, bound = ref.window(q, kw, vw, pos, win, sinks)
    p = dev(np.array(pos, np.int32))
    got = attention_window(dev(q), k, v, p, window=win, sinks=sinks, k_scale=ks, v_scale=vs)
    assert got.shape == q.shape
    check(got, want, bound, str(case))
    # two calls give the same bits; the flat form of q too
    again = attention_window(dev(q.reshape(n * t, h * d)), k, v, p, window=win, sinks=sinks, k_scale=ks, v_scale=vs)
    assert np.array_equal(again.cpu().numpy().reshape(q.shape), got.cpu().numpy())


@pytest.mark.parametrize("tokens,win,sinks", [(1, 0, 0), (1, 40, 3), (3, 40, 3), (90, 0, 0), (150, 40, 3)])
@pytest.mark.parametrize("kv", ["fp16", "int8"])
def test_window_unseen_rows_do_not_reach_the_output(gpu, kv, tokens, win, sinks):
    """NaN, infinities and the types' lowest values in rows that no token, or
    not every token, sees."""
    import torch

    from asdsl.kernels import attention_window

    rng = np.random.default_rng(5)
    n, h, kvh, d, rows, p0 = 1, 6, 2, 128, 400, 200
    q = rng.standard_normal((n, tokens, h, d)).astype(np.float32)
    k, ks, kw = make_cache(rng, kv, n, kvh, rows, d)
    v, vs, vw = make_cache(rng, kv, n, kvh, rows, d)
    want, bound = ref.window(q, kw, vw, [p0], win, sinks)
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
    pos = dev(np.array([p0], np.int32))
    check(attention_window(dev(q), k, v, pos, window=win, sinks=sinks, k_scale=ks, v_scale=vs), want, bound)
    # the last token's own row: no earlier token may feel it
    last = p0 + tokens - 1
    for x in (float("nan"), float("inf")):
        if kv == "fp16":
            k[:, :, last], v[:, :, last] = 1.0, x
        else:
            vs[:, :, last] = x
        got = attention_window(dev(q), k, v, pos, window=win, sinks=sinks, k_scale=ks, v_scale=vs)
        if tokens > 1:
            check(got[:, :-1].contiguous(), want[:, :-1], bound[:, :-1], str(x))
        assert not torch.isfinite(got[:, -1]).any()


@pytest.mark.parametrize("loud", [1e-3, 300.0])
@pytest.mark.parametrize("tokens", [1, 40, 140])
def test_window_quiet_and_loud_queries(gpu, tokens, loud):
    """Queries far from one: flat and one-hot weights."""
    from asdsl.kernels import attention_window

    rng = np.random.default_rng(6)
    q = (rng.standard_normal((1, tokens, 8, 128)) * loud).astype(np.float32)
    k, _, kw = make_cache(rng, "fp16", 1, 2, 500, 128)
    v, _, vw = make_cache(rng, "fp16", 1, 2, 500, 128)
    want, bound = ref.window(q, kw, vw, [300], 0, 0)
    got = attention_window(dev(q), k, v, dev(np.array([300], np.int32))).cpu().numpy()
    assert (np.abs(got - want) <= bound).all()


def test_window_far_rows_of_a_long_cache(gpu):
    """Element offsets past 2^31 and 2^32 bytes; the engine's three-dimensional caches."""
    import torch

    from asdsl.kernels import attention_window

    rows, d, kvh = 5_000_000, 128, 4  # 5.1 GB a cache
    k = torch.zeros((kvh, rows, d), dtype=torch.float16, device="cuda")
    v = torch.zeros_like(k)
    gen = torch.Generator(device="cuda").manual_seed(1)
    p = rows - 3
    k[:, p - 99:p + 1] = torch.randn((kvh, 100, d), generator=gen, device="cuda").half()
    v[:, p - 99:p + 1] = torch.randn((kvh, 100, d), generator=gen, device="cuda").half()
    for tokens in (1, 100):
        q = torch.randn((1, tokens, 8, d), generator=gen, device="cuda")
        first = p - tokens + 1
        got = attention_window(q, k, v, dev(np.array([first], np.int32)), window=64)
        lo = p - 99
        kw, vw = (x[None, :, lo:].cpu().numpy().astype(np.float64) for x in (k, v))
        j = np.arange(rows - lo)
        for t in range(max(0, tokens - 30), tokens):
            at = j[(j <= first + t - lo) & (j > first + t - lo - 64)]
            at = at[at >= 0]
            for a in range(8):
                if first + t - 63 < lo:
                    continue
                want, bound = ref.attend_row(q[0, t, a].cpu().numpy().astype(np.float64), kw[0, a // 2, at],
                                             vw[0, a // 2, at])
                assert (np.abs(got[0, t, a].cpu().numpy() - want) <= bound).all(), (tokens, t, a)


# n_seq, heads, kv heads, head_dim, cache, prefix rows, prefix_len, own rows, own positions
PREFIX = [
    (1, 24, 8, 128, "fp16", 40, 40, 8, [3]),
    (4, 24, 8, 128, "fp16", 777, 777, 64, [0, -1, 63, 40]),
    (5, 8, 4, 128, "int8", 300, 129, 33, [32, 31, -1, 0, 7]),
    (3, 16, 16, 64, "fp16", 200, 0, 20, [19, -1, 5]),
    (3, 16, 1, 128, "int8", 65, 65, 300, [299, 300, -2]),
    (17, 12, 4, 64, "int8", 1000, 999, 10, list(range(-1, 9)) + [9] * 7),
    (33, 6, 2, 128, "fp16", 130, 130, 40, [i % 41 - 1 for i in range(33)]),
    (70, 4, 2, 128, "fp16", 600, 600, 5, [i % 6 - 1 for i in range(70)]),
    (50, 6, 1, 64, "int8", 515, 513, 3, [2] * 50),
    (2, 4, 2, 128, "fp16", 1, 1, 1, [-1, 0]),
    (130, 3, 1, 128, "int8", 257, 257, 2, [i % 3 - 1 for i in range(130)]),
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

    def call(x):
        return attention_prefix(x, kp, vp, ko, vo, dev(np.array(own, np.int32)), prefix_len=plen, k_prefix_scale=kps,
                                v_prefix_scale=vps, k_scale=kos, v_scale=vos)
    got = call(dev(q))
    check(got, want, bound, str(case))
    assert np.array_equal(call(dev(q.reshape(n, h * d))).cpu().numpy().reshape(q.shape), got.cpu().numpy())
    # rows past the prefix's length and past each sequence's newest row: anything
    for t, s in ((kp, kps), (vp, vps)):
        (t if s is None else s)[:, plen:] = float("nan")
    for t, s in ((ko, kos), (vo, vos)):
        for i, m in enumerate(own):
            if m < rows:
                (t if s is None else s)[i, :, max(m + 1, 0):] = float("inf")
    check(call(dev(q)), want, bound, "unseen rows")


# n_seq, tokens, heads, kv heads, head_dim, rotary, cache, rows, positions, offset, table rows
APPEND = [
    (1, 1, 24, 8, 128, 96, "fp16", 64, [5], 0, 64),
    (3, 1, 24, 8, 128, 128, "int8", 32, [0, 31, 7], 100, 132),
    (2, 5, 8, 4, 64, 32, "fp16", 16, [0, 11], 3, 40),
    (2, 5, 8, 4, 64, 64, "int8", 16, [-2, 13], 3, 17),
    (1, 130, 6, 2, 128, 96, "int8", 200, [60], 0, 150),
    (4, 1, 3, 1, 64, 2, "fp16", 4, [0, 3, 4, -1], 0, 3),
]


@pytest.mark.parametrize("case", APPEND, ids=str)
def test_append(gpu, case):
    from asdsl.kernels import kv_append

    n, t, h, kvh, d, rot, kv, rows, pos, off, table = case
    rng = np.random.default_rng(n + t + d)
    qkv = rng.standard_normal((n, t, h + 2 * kvh, d)).astype(np.float32)
    ang = rng.uniform(0, 6.28, (table, rot // 2))
    cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
    k, ks, k0 = make_cache(rng, kv, n, kvh, rows, d)
    v, vs, v0 = make_cache(rng, kv, n, kvh, rows, d)
    q = kv_append(dev(qkv.reshape(n * t, -1)), k, v, dev(cos), dev(sin), dev(np.array(pos, np.int32)), n_heads=h,
                  pos_offset=off, k_scale=ks, v_scale=vs)
    got_q = q.cpu().numpy().reshape(n, t, h, d).astype(np.float64)
    host = lambda c, s: ref.wide(c.cpu().numpy(), None if s is None else s.cpu().numpy())  # noqa: E731
    got_k, got_v = host(k, ks), host(v, vs)
    for i in range(n):
        for j in range(t):
            r = pos[i] + j
            if not (0 <= r < rows and 0 <= r + off < table):
                assert (got_q[i, j] == 0).all()
                continue
            turned = ref.rotate(qkv[i, j, :h + kvh], cos[r + off], sin[r + off], rot // 2)
            mag = np.abs(qkv[i, j]).max() * 2
            assert np.abs(got_q[i, j] - turned[:h]).max() <= 3 * ref.EPS * mag
            for got, want in ((got_k[i, :, r], turned[h:]), (got_v[i, :, r], qkv[i, j, h + kvh:].astype(np.float64))):
                if kv == "fp16":  # half a step of fp16, and the rotation's roundings
                    assert (np.abs(got - want) <= 2.0 ** -11 * np.abs(want) + 2.0 ** -24 + 3 * ref.EPS * mag).all()
                else:  # half a step of the block's codes (and the scale's own roundings)
                    step = np.abs(want.reshape(kvh, -1, 64)).max(-1).repeat(64, -1) / 127
                    assert (np.abs(got - want) <= 0.501 * step + 3 * ref.EPS * mag).all()
            k0[i, :, r], v0[i, :, r] = got_k[i, :, r], got_v[i, :, r]
    # every other row as it was
    assert np.array_equal(got_k, k0) and np.array_equal(got_v, v0)


@pytest.mark.parametrize("kv", ["fp16", "int8"])
def test_append_and_window_follow_the_decode_steps_attention(gpu, kv):
    """One token: the cache rows have the bits that asdsl_attention_*kv writes,
    and attention over them is its result."""
    import torch

    from asdsl.engine import rope_tables
    from asdsl.kernels import attention_window, kv_append

    h, kvh, d, rot, rows, p = 24, 8, 128, 96, 300, 211
    rng = np.random.default_rng(3)
    qkv = dev(rng.standard_normal((1, (h + 2 * kvh) * d)).astype(np.float32))
    cos, sin = (dev(x) for x in rope_tables(rows, rot))
    k, ks, _ = make_cache(rng, kv, kvh, rows, d)
    v, vs, _ = make_cache(rng, kv, kvh, rows, d)
    k2, v2 = k.clone(), v.clone()
    pos = dev(np.array([p], np.int32))
    att = torch.empty(h * d, device="cuda")
    work = torch.empty(gpu.LIB.asdsl_attention_work_floats(h, rows), device="cuda")
    tail = (gpu.ptr(cos), gpu.ptr(sin), gpu.ptr(pos), gpu.ptr(att), gpu.ptr(work), h, kvh, d, rot, rows,
            gpu.stream_handle())
    if kv == "int8":
        ks2, vs2 = ks.clone(), vs.clone()
        gpu.call("asdsl_attention_q8kv", gpu.ptr(qkv), gpu.ptr(k2), gpu.ptr(v2), gpu.ptr(ks2), gpu.ptr(vs2), *tail)
    else:
        gpu.call("asdsl_attention_f16kv", gpu.ptr(qkv), gpu.ptr(k2), gpu.ptr(v2), *tail)
    q = kv_append(qkv, k, v, cos, sin, pos, n_heads=h, k_scale=ks, v_scale=vs)
    out = attention_window(q, k, v, pos, k_scale=ks, v_scale=vs)
    assert torch.equal(k, k2) and torch.equal(v, v2)
    if kv == "int8":
        assert torch.equal(ks, ks2) and torch.equal(vs, vs2)
    a, b = out.double().flatten(), att.double()
    assert float((a - b).norm() / b.norm()) < 2e-5  # each within 1e-5 of the definition


def test_prompt_chunk_then_branches_in_one_captured_run(gpu):
    """As they are used together: a prompt's rows appended and attended in a
    chunk, then steps of three continuations (append, shared prefix) captured
    once and replayed with the positions advancing on the device, on a side
    stream; every replay against the definition."""
    import torch

    from asdsl.engine import rope_tables
    from asdsl.kernels import attention_prefix, attention_window, kv_append

    h, kvh, d, rot, prompt, own, n = 12, 4, 128, 96, 150, 6, 3
    rng = np.random.default_rng(11)
    cos, sin = rope_tables(prompt + own, rot)
    dcos, dsin = dev(cos), dev(sin)
    k = torch.zeros((kvh, prompt + 9, d), dtype=torch.float16, device="cuda")
    v = torch.zeros_like(k)
    ko = torch.zeros((n, kvh, own, d), dtype=torch.float16, device="cuda")
    vo = torch.zeros_like(ko)
    chunk = dev(rng.standard_normal((prompt, (h + 2 * kvh) * d)).astype(np.float32))
    zero = dev(np.zeros(1, np.int32))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        q = kv_append(chunk, k, v, dcos, dsin, zero, n_heads=h)
        att = attention_window(q, k, v, zero, window=64, sinks=4)
    torch.cuda.current_stream().wait_stream(side)
    kw, vw = k.cpu().numpy().astype(np.float64)[None], v.cpu().numpy().astype(np.float64)[None]
    want, bound = ref.window(q.cpu().numpy().reshape(1, prompt, h, d), kw, vw, [0], 64, 4)
    check(att, want, bound)
    step = torch.zeros((n, (h + 2 * kvh) * d), device="cuda")
    pos = torch.zeros(n, dtype=torch.int32, device="cuda")

    def queue():
        rq = kv_append(step, ko, vo, dcos, dsin, pos, n_heads=h, pos_offset=prompt)
        out = attention_prefix(rq, k, v, ko, vo, pos, prefix_len=prompt)
        pos.add_(1)
        return rq, out
    queue()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rq, out = queue()
    pos.zero_()
    for i in range(own):
        step.copy_(dev(rng.standard_normal(tuple(step.shape)).astype(np.float32)))
        graph.replay()
        torch.cuda.synchronize()
        kow, vow = ko.cpu().numpy().astype(np.float64), vo.cpu().numpy().astype(np.float64)
        want, bound = ref.prefix(rq.cpu().numpy().reshape(n, h, d), kw[0], vw[0], prompt, kow, vow, [i] * n)
        check(out, want, bound, f"replay {i}")
    assert pos.tolist() == [own] * n


def test_refusals_on_the_device(gpu):
    import torch

    from asdsl.kernels import attention_prefix, attention_window, kv_append

    k = torch.zeros((1, 2, 16, 128), dtype=torch.float16, device="cuda")
    q = torch.zeros((1, 1, 4, 128), device="cuda")
    pos = torch.zeros(1, dtype=torch.int32, device="cuda")
    wide = torch.zeros((1, 2, 16, 256), dtype=torch.float16, device="cuda")[..., ::2]
    for bad in (lambda: attention_window(q, wide, wide, pos), lambda: attention_window(q, k, k, pos.cpu()),
                lambda: attention_window(q.half(), k, k, pos), lambda: attention_window(q, k, k, pos.long()),
                lambda: attention_window(q, k, k, pos, window=-1), lambda: attention_window(q, k, k, pos, sinks=-1),
                lambda: attention_window(q, k, k, pos, out=torch.empty(3, device="cuda")),
                lambda: attention_prefix(q[0], k[0], k[0], k, k, pos, prefix_len=17),
                lambda: kv_append(torch.zeros(8 * 128 + 1, device="cuda")[1:], k, k, q[0, 0, :, :4].contiguous(),
                                  q[0, 0, :, :4].contiguous(), pos, n_heads=4)):
        with pytest.raises(ValueError):
            bad()
    # a work buffer that is too small is an argument error before any launch
    lib = gpu.LIB
    need = lib.asdsl_attention_window_work_bytes(1, 1, 24, 8, 128, 4096, 0, 0)
    if need:
        one = ctypes.c_void_p(256)
        assert lib.asdsl_attention_window_f16kv(one, one, one, one, one, 1, 1, 24, 8, 128, 4096, 0, 0, one, need - 1,
                                                None) == gpu.ASDSL_ERR_INVALID_ARGUMENT
        assert "work buffer" in gpu.last_error()


@pytest.mark.parametrize("kv", ["fp16", "int8"])
def test_calls_that_need_no_work_buffer_allocate_none(gpu, kv):
    """With its output given a call whose keys are taken in one piece allocates nothing, and one in pieces the bytes
    of its own form, not those of another."""
    import torch

    from asdsl.kernels import attention_prefix, attention_window

    rng = np.random.default_rng(1)
    form = "f16kv" if kv == "fp16" else "q8kv"

    def taken(call, *args, **kw):
        out = torch.empty_like(args[0])
        before = torch.cuda.memory_stats()["requested_bytes.all.allocated"]
        call(*args, out=out, **kw)
        return torch.cuda.memory_stats()["requested_bytes.all.allocated"] - before

    for n, t, h, kvh, d, rows in ((99, 16, 8, 4, 128, 12139), (60, 24, 16, 4, 64, 5000), (1, 1, 24, 8, 128, 4352)):
        k, ks, _ = make_cache(rng, kv, n, kvh, 1, d)
        k = k.expand(n, kvh, rows, d).contiguous()
        ks = None if ks is None else ks.expand(n, kvh, rows, d // 64).contiguous()
        pos = dev(rng.integers(0, 300, n).astype(np.int32))
        q = torch.randn((n, t, h, d), device="cuda")
        need = getattr(gpu.LIB, f"asdsl_attention_window_{form}_work_bytes")(n, t, h, kvh, d, rows, 0, 0)
        got = taken(attention_window, q, k, k, pos, k_scale=ks, v_scale=ks)
        assert got == need
    own, own_s, _ = make_cache(rng, kv, 3, 8, 100, 128)
    q, pos = torch.randn((3, 24, 128), device="cuda"), dev(np.array([5, -1, 99], np.int32))
    pre, pre_s, _ = make_cache(rng, kv, 8, 3000, 128)
    need = getattr(gpu.LIB, f"asdsl_attention_prefix_{form}_work_bytes")(3, 24, 8, 128, 3000, 100)
    got = taken(attention_prefix, q, pre, pre, own, own, pos, k_prefix_scale=pre_s, v_prefix_scale=pre_s, k_scale=own_s,
                v_scale=own_s)
    assert got == need
