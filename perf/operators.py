"""The operators of many sequences and long contexts, as cases that can be timed and checked.

Four operators beside the batch-1 decode step: the rotated queries and cache
rows of many tokens (``kv_append``), attention over a KV cache with a sliding
window and first tokens that stay visible (``attention_window``), attention of
many sequences that share a prefix (``attention_prefix``), and penalties,
biases and grammar masks on logits with the greedy token (``control_logits``).
``run`` computes them in plain torch operations, or, where ``own`` is true,
through ``asdsl.kernels``.  Inputs are synthetic and drawn on the device from a
seed: activations, queries and cached rows ~ N(0, 1), logits ~ N(0, 3).
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

_PKG = str(Path.cwd() / "asdsl-framework_amd")
if _PKG not in sys.path:
    sys.path.insert(0, _PKG)

own = False

PHI = {"heads": 24, "kv_heads": 8, "dim": 128}  # the decode engine's defaults
MID = {"heads": 16, "kv_heads": 4, "dim": 128}  # head layouts of the engine's tests
SMALL = {"heads": 8, "kv_heads": 4, "dim": 128}
NARROW = {"heads": 32, "kv_heads": 8, "dim": 64}
KV_BLOCK = 64  # dims per scale of an int8 cache


def listed():
    return [
        # One step of sixteen continuations: their queries and new cache rows.
        {"name": "append_16", "kind": "append", **PHI, "seqs": 16, "tokens": 1, "rows": 512, "rotary": 96},
        # A prompt chunk's rows into the cache of one sequence (an odd length).
        {"name": "append_prompt_2045", "kind": "append", **PHI, "seqs": 1, "tokens": 2045, "rows": 4352, "rotary": 96},
        # One token of a short chat: the smallest attention call, all launch and latency.
        {"name": "window_step_200", "kind": "window", **PHI, "seqs": 1, "tokens": 1, "rows": 4352, "longest": 200,
         "window": 0, "sinks": 0, "kv": "fp16"},
        # A batch of long chats of ragged lengths that attend to their last 4096 positions and 4 first ones.
        {"name": "window_steps_32", "kind": "window", **PHI, "seqs": 32, "tokens": 1, "rows": 16384, "longest": 16000,
         "window": 4096, "sinks": 4, "kv": "int8"},
        # A chat turn's prompt (an odd length) behind what was said before, all of it visible.
        {"name": "window_prompt_517", "kind": "window", **MID, "seqs": 1, "tokens": 517, "rows": 2048,
         "longest": 1000, "window": 0, "sinks": 0, "kv": "fp16"},
        # A long document with a window: the largest call, bound by its products.
        {"name": "window_prompt_4096", "kind": "window", **PHI, "seqs": 1, "tokens": 4096, "rows": 8192,
         "longest": 6000, "window": 2048, "sinks": 4, "kv": "fp16"},
        # Four continuations of a chat, shortly after its prompt.
        {"name": "prefix_4", "kind": "prefix", **PHI, "seqs": 4, "prefix": 777, "rows": 64, "kv": "fp16"},
        # Many samples of one long prompt, as for voting over answers.
        {"name": "prefix_64", "kind": "prefix", **PHI, "seqs": 64, "prefix": 16384, "rows": 512, "kv": "fp16"},
        # The same over int8 caches and narrow heads, an odd number of sequences and an odd prefix.
        {"name": "prefix_27_int8", "kind": "prefix", **NARROW, "seqs": 27, "prefix": 5001, "rows": 300,
         "kv": "int8"},
        # The next token of one chat: penalties over its history, a grammar's mask.
        {"name": "logits_1", "kind": "logits", "seqs": 1, "vocab": 200064, "history": 1500, "allowed": 0.9,
         "bias": "none"},
        # A serving batch, each row with its own mask, one bias for all.
        {"name": "logits_64", "kind": "logits", "seqs": 64, "vocab": 200064, "history": 4000, "allowed": 0.5,
         "bias": "shared"},
        # A small vocabulary of an odd size, a grammar that allows few tokens, a bias a row.
        {"name": "logits_7_odd", "kind": "logits", "seqs": 7, "vocab": 32003, "history": 700, "allowed": 0.01,
         "bias": "rows"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "window_steps", "window_prompt", "prefix", "logits"])
    if kind == "logits":
        vocab = _log_int(rng, 1000, 200064)
        return {"kind": kind, "seqs": _log_int(rng, 1, max(1, 12_000_000 // vocab) if vocab > 100_000 else 64),
                "vocab": vocab, "history": _log_int(rng, 1, 8000), "allowed": rng.choice([0.01, 0.5, 0.9, 1.0]),
                "bias": rng.choice(["none", "shared", "rows"])}
    c = {"kind": kind, **rng.choice([PHI, MID, SMALL, NARROW, {"heads": 8, "kv_heads": 8, "dim": 64},
                                     {"heads": 16, "kv_heads": 1, "dim": 128}])}
    if kind == "append":
        c["tokens"] = rng.choice([1, _log_int(rng, 2, 2045)])
        c["seqs"] = _log_int(rng, 1, min(64, max(1, 2045 // c["tokens"])))
        c["rows"] = c["tokens"] + rng.randint(1, 500)
        c["rotary"] = rng.choice([c["dim"], c["dim"] * 3 // 4, 32])
        return c
    c["kv"] = rng.choice(["fp16", "int8"])
    if kind == "prefix":
        c["seqs"] = _log_int(rng, 2, 64)
        c["prefix"] = _log_int(rng, 1, 16384)
        c["rows"] = _log_int(rng, 4, 512)
        return c
    c["kind"] = "window"
    if kind == "window_steps":
        c["seqs"], c["tokens"] = _log_int(rng, 1, 32), 1
        c["longest"] = _log_int(rng, 2, 16000)
    else:
        c["seqs"], c["tokens"] = 1, _log_int(rng, 2, 2048)
        if c["tokens"] < 64:
            c["seqs"] = _log_int(rng, 1, 16)
        c["longest"] = c["tokens"] + _log_int(rng, 1, 2000)
    c["rows"] = c["longest"] + rng.randint(1, 300)
    c["window"] = rng.choice([0, _log_int(rng, 1, 2048)])
    c["sinks"] = rng.choice([0, 1, 4, 64]) if c["window"] else 0
    return c


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)


def _cache(gen, kv, *shape):
    """Cache rows ~ N(0, 1): fp16, or int8 codes with a scale per 64 dims."""
    x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float16)
    if kv == "fp16":
        return x, None
    b = x.reshape(*shape[:-1], shape[-1] // KV_BLOCK, KV_BLOCK)
    scale = b.abs().amax(dim=-1).float() / 127.0
    codes = torch.round(b / scale.half()[..., None]).clamp_(-127, 127).to(torch.int8)
    return codes.reshape(shape), scale


def _lengths(case, first):
    """Ragged lengths of the sequences, the longest first, from the case alone."""
    rng = random.Random(case["seqs"] * 1000003 + first)
    return [first] + [rng.randint(1, first) for _ in range(case["seqs"] - 1)]


def _first_positions(case):
    """Per sequence the position of its first token of the call; a batch of several has a padded one (-1)."""
    pos = [n - case["tokens"] if n >= case["tokens"] else 0 for n in _lengths(case, case["longest"])]
    if case["seqs"] > 2 and case["tokens"] == 1:
        pos[-1] = -1
    return pos


def _own_positions(case):
    """Per sequence its newest own row; one of several has no own row yet (-1)."""
    pos = [n - 1 for n in _lengths(case, case["rows"])]
    if case["seqs"] > 2:
        pos[1] = -1
    return pos


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen, kind = _gen(seed), case["kind"]
    s = {"case": case, "kind": kind}
    n = case["seqs"]
    if kind == "logits":
        v, cap = case["vocab"], case["history"]
        s["logits"] = _randn(gen, n, v) * 3.0
        # a history repeats itself: ids fall off as one over their rank
        u = torch.rand((n, cap), generator=gen, device="cuda")
        ids = (torch.exp(u * math.log(v)) - 1.0).to(torch.int64).clamp_(0, v - 1)
        s["history"] = ((ids * 7919 + 13) % v).to(torch.int32)
        total = _lengths(case, cap)
        s["history_len"], s["prompt_len"] = _ints(total), _ints([t // 3 for t in total])
        s["repetition"] = 1.0 + 0.3 * torch.rand(n, generator=gen, device="cuda")
        s["frequency"] = 0.5 * torch.rand(n, generator=gen, device="cuda")
        s["presence"] = 0.5 * torch.rand(n, generator=gen, device="cuda")
        s["bias"] = None if case["bias"] == "none" else _randn(gen, v) if case["bias"] == "shared" else \
            _randn(gen, n, v)
        words = (v + 31) // 32
        bits = torch.rand((n, words, 32), generator=gen, device="cuda") < case["allowed"]
        weights = torch.ones(32, dtype=torch.int64, device="cuda") << torch.arange(32, device="cuda")
        s["allowed"] = (bits.long() * weights).sum(dim=2).to(torch.int32)
        s["out"] = torch.empty_like(s["logits"])
        return s
    h, kvh, d, rows = case["heads"], case["kv_heads"], case["dim"], case["rows"]
    if kind == "append":
        s["qkv"] = _randn(gen, n * case["tokens"], (h + 2 * kvh) * d)
        s["k"], _ = _cache(gen, "fp16", n, kvh, rows, d)
        s["v"], _ = _cache(gen, "fp16", n, kvh, rows, d)
        first = rows - case["tokens"]
        s["pos"] = _ints([p % (first + 1) for p in _lengths(case, first + 1)])
        half = case["rotary"] // 2
        freq = 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
        s["offset"] = 100
        angle = torch.arange(rows + s["offset"], device="cuda", dtype=torch.float64)[:, None] * freq
        s["cos"], s["sin"] = torch.cos(angle).float(), torch.sin(angle).float()
        return s
    s["q"] = _randn(gen, n, case["tokens"], h, d) if kind == "window" else _randn(gen, n, h, d)
    if kind == "prefix":
        s["k_prefix"], s["k_prefix_scale"] = _cache(gen, case["kv"], kvh, case["prefix"], d)
        s["v_prefix"], s["v_prefix_scale"] = _cache(gen, case["kv"], kvh, case["prefix"], d)
        s["pos"] = _ints(_own_positions(case))
    else:
        first = _first_positions(case)
        s["pos"] = _ints(first)
        # the cache rows from which any token of the call sees, per sequence, and how many there are at most
        w, t = case["window"], case["tokens"]
        low = [max(case["sinks"], p - w + 1) if w else 0 for p in first]
        s["low"] = torch.tensor(low, device="cuda")
        s["span"] = max([p + t - a for p, a in zip(first, low)] + [0])
    s["k"], s["k_scale"] = _cache(gen, case["kv"], n, kvh, rows, d)
    s["v"], s["v_scale"] = _cache(gen, case["kv"], n, kvh, rows, d)
    return s


# -------------------------------------------------------------- plain forms
def _rows_of(cache, scale, *at):
    """The rows `at` of a cache in 32 bits (all without `at`)."""
    x = (cache[at] if at else cache).float()
    if scale is None:
        return x
    scale = scale[at] if at else scale
    return (x.reshape(*x.shape[:-1], -1, KV_BLOCK) * scale[..., None]).reshape(x.shape)


def _plain_append(s):
    c = s["case"]
    n, t, h, kvh, d, half = c["seqs"], c["tokens"], c["heads"], c["kv_heads"], c["dim"], c["rotary"] // 2
    x = s["qkv"].reshape(n, t, h + 2 * kvh, d)
    rows = s["pos"].long()[:, None] + torch.arange(t, device=x.device)
    cos, sin = s["cos"][rows + s["offset"]][:, :, None], s["sin"][rows + s["offset"]][:, :, None]
    a, b = x[:, :, :h + kvh, :half], x[:, :, :h + kvh, half:2 * half]
    turned = torch.cat((a * cos - b * sin, a * sin + b * cos, x[:, :, :h + kvh, 2 * half:]), dim=3)
    seq = torch.arange(n, device=x.device)[:, None]
    s["k"][seq, :, rows] = turned[:, :, h:].half()
    s["v"][seq, :, rows] = x[:, :, h + kvh:].half()
    return {"q": turned[:, :, :h].reshape(n * t, h * d), "k": s["k"], "v": s["v"]}


def _plain_window(s):
    c = s["case"]
    n, t, kvh, d, w, sinks = c["seqs"], c["tokens"], c["kv_heads"], c["dim"], c["window"], c["sinks"]
    g = c["heads"] // kvh
    near = s["low"][:, None] + torch.arange(s["span"], device="cuda")
    at = torch.cat((torch.arange(sinks if w else 0, device="cuda").expand(n, -1), near), dim=1)
    seq, head = torch.arange(n, device="cuda")[:, None, None], torch.arange(kvh, device="cuda")[:, None]
    held = at.clamp(0, c["rows"] - 1)[:, None]
    k, v = _rows_of(s["k"], s["k_scale"], seq, head, held), _rows_of(s["v"], s["v_scale"], seq, head, held)
    q = s["q"].reshape(n, t, kvh, g, d).permute(0, 2, 1, 3, 4).reshape(n, kvh, t * g, d)
    scores = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(d))
    p = s["pos"].long()[:, None, None] + torch.arange(t, device="cuda")[:, None]
    key = at[:, None]
    seen = (key <= p) & (p >= 0) & (p < c["rows"])
    if w:
        first = torch.arange(at.shape[1], device="cuda") < sinks
        seen = seen & ((key > p - w) | first)
    scores = scores.reshape(n, kvh, t, g, -1).masked_fill(~seen[:, None, :, None], float("-inf"))
    top = scores.amax(dim=-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == float("-inf"), torch.zeros_like(top), top))
    total = e.sum(dim=-1, keepdim=True)
    out = torch.matmul(e.reshape(n, kvh, t * g, -1), v).reshape(n, kvh, t, g, d)
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    return out.permute(0, 2, 1, 3, 4).reshape(n, t, c["heads"], d)


def _plain_prefix(s):
    c = s["case"]
    n, kvh, d = c["seqs"], c["kv_heads"], c["dim"]
    g = c["heads"] // kvh
    q = s["q"].reshape(n, kvh, g, d) * (1.0 / math.sqrt(d))
    kp, vp = _rows_of(s["k_prefix"], s["k_prefix_scale"]), _rows_of(s["v_prefix"], s["v_prefix_scale"])
    ko, vo = _rows_of(s["k"], s["k_scale"]), _rows_of(s["v"], s["v_scale"])
    shared = q.transpose(0, 1).reshape(kvh, n * g, d)
    sp = torch.matmul(shared, kp.transpose(1, 2)).reshape(kvh, n, g, -1).transpose(0, 1)
    so = torch.matmul(q, ko.transpose(2, 3))
    seen = torch.arange(c["rows"], device="cuda") <= s["pos"].long()[:, None]
    so = so.masked_fill(~seen[:, None, None], float("-inf"))
    top = torch.maximum(sp.amax(dim=-1, keepdim=True), so.amax(dim=-1, keepdim=True))
    ep, eo = torch.exp(sp - top), torch.exp(so - top)
    out = torch.matmul(ep.transpose(0, 1).reshape(kvh, n * g, -1), vp).reshape(kvh, n, g, d).transpose(0, 1)
    out = (out + torch.matmul(eo, vo)) / (ep.sum(dim=-1, keepdim=True) + eo.sum(dim=-1, keepdim=True))
    return out.reshape(n, c["heads"], d)


def _plain_logits(s):
    x, ids = s["logits"], s["history"].long()
    n, v = x.shape
    at = torch.arange(ids.shape[1], device=x.device)
    told = at < s["history_len"].long()[:, None]
    made = told & (at >= s["prompt_len"].long()[:, None])
    count = torch.zeros_like(x).scatter_add_(1, ids, made.float())
    seen = torch.zeros_like(x).scatter_add_(1, ids, told.float()) > 0
    r = s["repetition"][:, None]
    y = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    y = y - s["frequency"][:, None] * count
    y = torch.where(count > 0, y - s["presence"][:, None], y)
    if s["bias"] is not None:
        y = y + s["bias"]
    token = torch.arange(v, device=x.device)
    ok = ((s["allowed"][:, token // 32] >> (token % 32)) & 1) != 0
    y = torch.where(ok, y, torch.full_like(y, float("-inf")))
    best = torch.where(ok & (y == y.amax(dim=1, keepdim=True)), token, v).amin(dim=1)
    return {"logits": y, "tokens": torch.where(best < v, best, -1).to(torch.int32)}


def _own_run(s):
    from asdsl import kernels

    kind, c = s["kind"], s["case"]
    if kind == "append":
        q = kernels.kv_append(s["qkv"], s["k"], s["v"], s["cos"], s["sin"], s["pos"], n_heads=c["heads"],
                              pos_offset=s["offset"])
        return {"q": q, "k": s["k"], "v": s["v"]}
    if kind == "window":
        return kernels.attention_window(s["q"], s["k"], s["v"], s["pos"], window=c["window"], sinks=c["sinks"],
                                        k_scale=s["k_scale"], v_scale=s["v_scale"])
    if kind == "prefix":
        return kernels.attention_prefix(s["q"], s["k_prefix"], s["v_prefix"], s["k"], s["v"], s["pos"],
                                        k_prefix_scale=s["k_prefix_scale"], v_prefix_scale=s["v_prefix_scale"],
                                        k_scale=s["k_scale"], v_scale=s["v_scale"])
    y, tokens = kernels.control_logits(s["logits"], history=s["history"], history_len=s["history_len"],
                                       prompt_len=s["prompt_len"], repetition=s["repetition"],
                                       frequency=s["frequency"], presence=s["presence"], bias=s["bias"],
                                       allowed=s["allowed"], out=s["out"])
    return {"logits": y, "tokens": tokens}


def run(state):
    if own:
        return _own_run(state)
    return {"append": _plain_append, "window": _plain_window, "prefix": _plain_prefix,
            "logits": _plain_logits}[state["kind"]](state)


# ------------------------------------------------------------- what it takes
def _row_bytes(c):
    """Bytes of one position's K and V rows over all KV heads."""
    return 2 * c["kv_heads"] * c["dim"] * (2.0 if c.get("kv", "fp16") == "fp16" else 1.0 + 4.0 / KV_BLOCK)


def _visible(c):
    """(cache rows that any token of the call sees, pairs of a token and a row it sees), over all sequences."""
    rows = pairs = 0
    w, sinks, t = c["window"], c["sinks"], c["tokens"]
    for p0 in _first_positions(c):
        if p0 < 0:
            continue
        end = p0 + t
        rows += end if not w else min(end, sinks + max(0, end - max(sinks, p0 - w + 1)))
        for p in range(p0, end):
            pairs += p + 1 if not w else min(p + 1, sinks) + max(0, p + 1 - max(sinks, p - w + 1))
    return rows, pairs


def work(c):
    kind, n = c["kind"], c["seqs"]
    if kind == "logits":
        v = c["vocab"]
        bias = {"none": 0, "shared": v, "rows": n * v}[c["bias"]]
        return {"bytes": 8 * n * v + 4 * n * ((v + 31) // 32) + 4 * bias + 4 * sum(_lengths(c, c["history"])) + 4 * n,
                "flops": 6 * n * v}
    width = c["heads"] * c["dim"]
    if kind == "append":
        t = n * c["tokens"]
        qkv = (c["heads"] + 2 * c["kv_heads"]) * c["dim"]
        table = 4 * c["rotary"] * min(t, c["rows"])
        return {"bytes": t * (4 * qkv + 4 * width + _row_bytes(c)) + table, "flops": 3 * t * qkv}
    if kind == "window":
        rows, pairs = _visible(c)
        return {"bytes": rows * _row_bytes(c) + 8 * n * c["tokens"] * width, "flops": 4 * pairs * width}
    own_rows = sum(p + 1 for p in _own_positions(c))
    return {"bytes": (c["prefix"] + own_rows) * _row_bytes(c) + 8 * n * width,
            "flops": 4 * (n * c["prefix"] + own_rows) * width}


# ------------------------------------------------------------------ 64 bits
def _wide(cache, scale):
    x = cache.double()
    if scale is not None:
        x = x * scale.double().repeat_interleave(KV_BLOCK, dim=-1)
    return x


def _attend(q, k, v, seen):
    """softmax(q k' / sqrt(d)) v over the rows that `seen` (tokens x rows) leaves; q (tokens, heads of one KV head, d)."""
    out = torch.zeros_like(q)
    for h in range(q.shape[1]):
        w = torch.where(seen, torch.exp((q[:, h] @ k.T / math.sqrt(q.shape[2])).clamp(-600, 600)), 0.0)
        total = w.sum(dim=1, keepdim=True)
        out[:, h] = (w @ v) / torch.where(total > 0, total, torch.ones_like(total))
    return out


def exact(case, seed):
    s, kind, n = prepare(case, seed), case["kind"], case["seqs"]
    if kind == "logits":
        y = s["logits"].double()
        tokens = []
        for i in range(n):
            told, made = int(s["history_len"][i]), int(s["prompt_len"][i])
            ids = s["history"][i].long()
            again = torch.unique(ids[:told])
            z, r = y[i, again], s["repetition"][i].double()
            y[i, again] = torch.where(z > 0, z / r, z * r)
            times = torch.bincount(ids[made:told], minlength=case["vocab"]).double()
            y[i] -= s["frequency"][i].double() * times + s["presence"][i].double() * (times > 0)
            if s["bias"] is not None:
                y[i] += s["bias"].double() if s["bias"].dim() == 1 else s["bias"][i].double()
            words = s["allowed"][i].long() & 0xFFFFFFFF
            bits = torch.stack([(words >> b) & 1 for b in range(32)], dim=1).reshape(-1)[:case["vocab"]]
            y[i, bits == 0] = float("-inf")
            tokens.append(int(y[i].argmax()) if bool(bits.any()) else -1)
        return {"logits": y, "tokens": _ints(tokens)}
    h, kvh, d = case["heads"], case["kv_heads"], case["dim"]
    g = h // kvh
    if kind == "append":
        t, half = case["tokens"], case["rotary"] // 2
        k, v = s["k"].double(), s["v"].double()
        q = torch.zeros((n, t, h, d), dtype=torch.float64, device="cuda")
        x = s["qkv"].double().reshape(n, t, h + 2 * kvh, d)
        for i in range(n):
            p = int(s["pos"][i])
            cos, sin = (s[name][p + s["offset"]:p + s["offset"] + t].double()[:, None] for name in ("cos", "sin"))
            turn = x[i, :, :h + kvh].clone()
            pair = torch.complex(x[i, :, :h + kvh, :half], x[i, :, :h + kvh, half:2 * half]) * torch.complex(cos, sin)
            turn[..., :half], turn[..., half:2 * half] = pair.real, pair.imag
            q[i], k[i, :, p:p + t], v[i, :, p:p + t] = turn[:, :h], turn[:, h:].transpose(0, 1), \
                x[i, :, h + kvh:].transpose(0, 1)
        return {"q": q.reshape(n * t, h * d), "k": k, "v": v}
    q = s["q"].double()
    out = torch.zeros_like(q)
    if kind == "prefix":
        for j in range(kvh):
            kp = _wide(s["k_prefix"][j], None if s["k_prefix_scale"] is None else s["k_prefix_scale"][j])
            vp = _wide(s["v_prefix"][j], None if s["v_prefix_scale"] is None else s["v_prefix_scale"][j])
            for i in range(n):
                m = int(s["pos"][i]) + 1
                ko = _wide(s["k"][i, j, :m], None if s["k_scale"] is None else s["k_scale"][i, j, :m])
                vo = _wide(s["v"][i, j, :m], None if s["v_scale"] is None else s["v_scale"][i, j, :m])
                seen = torch.ones((1, len(kp) + m), dtype=torch.bool, device="cuda")
                out[i, j * g:(j + 1) * g] = _attend(q[i, None, j * g:(j + 1) * g], torch.cat((kp, ko)),
                                                    torch.cat((vp, vo)), seen)[0]
        return out
    first = _first_positions(case)
    for i in range(n):
        if first[i] < 0:
            continue
        at = torch.arange(first[i], first[i] + case["tokens"], device="cuda")[:, None]
        key = torch.arange(first[i] + case["tokens"], device="cuda")
        seen = key <= at
        if case["window"]:
            seen = seen & ((key < case["sinks"]) | (at - key < case["window"]))
        for j in range(kvh):
            k = _wide(s["k"][i, j, :len(key)], None if s["k_scale"] is None else s["k_scale"][i, j, :len(key)])
            v = _wide(s["v"][i, j, :len(key)], None if s["v_scale"] is None else s["v_scale"][i, j, :len(key)])
            out[i, :, j * g:(j + 1) * g] = _attend(q[i, :, j * g:(j + 1) * g], k, v, seen)
    return out
