"""Operators of 4-bit caches and of sampling, as cases that can be timed and checked.

Keys and values written into a cache of 4 bits and read back (``kv_append``,
``kv_read``), attention over such caches (``attention_window``,
``attention_prefix``), rows of int8 caches read back, and the next token drawn
with temperature, top-k, top-p and min-p from a given random number
(``sample_logits``).  ``run`` computes them in plain torch operations, or,
where ``own`` is true, through ``asdsl.kernels``.  Inputs are synthetic and
drawn on the device from a seed: activations, queries and cached rows ~ N(0, 1),
logits ~ N(0, 3).

A cache of 4 bits holds per row and 32 dims a 16-bit word (an fp16 scale of 7
significant bits, its low 4 bits the zero point z) and codes c, two a byte, the
low nibble the even dim's: value = (c - z) * scale.
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import numpy as np
import torch

_PKG = str(Path.cwd() / "asdsl-framework_amd")
if _PKG not in sys.path:
    sys.path.insert(0, _PKG)

own = False

PHI = {"heads": 24, "kv_heads": 8, "dim": 128}  # the decode engine's defaults
MID = {"heads": 16, "kv_heads": 4, "dim": 128}  # head layouts of the engine's tests
SMALL = {"heads": 8, "kv_heads": 4, "dim": 128}
NARROW = {"heads": 32, "kv_heads": 8, "dim": 64}
GROUP = 32  # dims per scale word of a 4-bit cache
KV_BLOCK = 64  # dims per scale of an int8 cache
MOST = 32768.0  # values are held to this


def listed():
    return [
        # One step of sixteen short continuations: their queries and new rows, and their caches read back as values.
        {"name": "append4_16", "kind": "append", **PHI, "seqs": 16, "tokens": 1, "rows": 48, "rotary": 96},
        # A prompt's rows (an odd length) into the cache of one sequence, and the cache read back.
        {"name": "append4_prompt_2045", "kind": "append", **PHI, "seqs": 1, "tokens": 2045, "rows": 2112, "rotary": 96},
        # A long chat's 4-bit rows back into fp16, from its first row on.
        {"name": "read4_4001", "kind": "read", **PHI, "seqs": 1, "rows": 4352, "take": 4001, "kv": "int4", "to": "fp16"},
        # Ragged pieces of several int8 caches of narrow heads as fp32 values.
        {"name": "read8_12", "kind": "read", **NARROW, "seqs": 12, "rows": 1024, "take": 701, "kv": "int8", "to": "fp32"},
        # One token of a short chat: the smallest attention call, all launch and latency.
        {"name": "window4_step_200", "kind": "window", **PHI, "seqs": 1, "tokens": 1, "rows": 4352, "longest": 200,
         "window": 0, "sinks": 0},
        # A batch of long chats of ragged lengths that attend to all they hold.
        {"name": "window4_steps_32", "kind": "window", **PHI, "seqs": 32, "tokens": 1, "rows": 16384, "longest": 16000,
         "window": 0, "sinks": 0},
        # A long document with a window and first rows that stay visible: the largest call, bound by its products.
        {"name": "window4_prompt_4096", "kind": "window", **PHI, "seqs": 1, "tokens": 4096, "rows": 8192,
         "longest": 6000, "window": 2048, "sinks": 4},
        # Four continuations of a chat of narrow heads, shortly after its prompt (an odd length).
        {"name": "prefix4_4", "kind": "prefix", **NARROW, "seqs": 4, "prefix": 777, "rows": 64},
        # Many samples of one long prompt, as for voting over answers.
        {"name": "prefix4_64", "kind": "prefix", **PHI, "seqs": 64, "prefix": 16384, "rows": 512},
        # The next token of one chat, every filter on.
        {"name": "sample_1", "kind": "sample", "seqs": 1, "vocab": 200064, "temperature": 0.7, "top_k": 50,
         "top_p": 0.9, "min_p": 0.02},
        # A serving batch with top-p alone, each row with its own temperature and share.
        {"name": "sample_64", "kind": "sample", "seqs": 64, "vocab": 200064, "temperature": 1.0, "top_k": 0,
         "top_p": 0.95, "min_p": 0.0},
        # A small vocabulary of an odd size, a high temperature, min-p alone.
        {"name": "sample_7_odd", "kind": "sample", "seqs": 7, "vocab": 32003, "temperature": 1.5, "top_k": 0,
         "top_p": 1.0, "min_p": 0.05},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "read", "window_steps", "window_prompt", "prefix", "sample", "sample"])
    if kind == "sample":
        vocab = _log_int(rng, 1000, 200064)
        return {"kind": kind, "vocab": vocab, "seqs": _log_int(rng, 1, max(1, min(64, 12_000_000 // vocab))),
                "temperature": round(rng.uniform(0.3, 2.0), 2), "top_k": rng.choice([0, 1, 40, _log_int(rng, 2, 5000)]),
                "top_p": rng.choice([1.0, 0.98, 0.9, 0.5, round(rng.random(), 3)]),
                "min_p": rng.choice([0.0, 0.02, 0.1, round(rng.random(), 3)])}
    c = {"kind": kind, **rng.choice([PHI, MID, SMALL, NARROW, {"heads": 8, "kv_heads": 8, "dim": 64},
                                     {"heads": 16, "kv_heads": 1, "dim": 128}])}
    if kind == "append":
        c["tokens"] = rng.choice([1, _log_int(rng, 2, 2045)])
        c["seqs"] = _log_int(rng, 1, min(64, max(1, 2045 // c["tokens"])))
        c["rows"] = c["tokens"] + rng.randint(1, 60)
        c["rotary"] = rng.choice([c["dim"], c["dim"] * 3 // 4, 32])
        return c
    if kind == "read":
        c["seqs"], c["take"] = _log_int(rng, 1, 32), _log_int(rng, 1, 2000)
        c["rows"] = c["take"] + rng.randint(1, 300)
        c["kv"], c["to"] = rng.choice(["int4", "int4", "int8"]), rng.choice(["fp16", "fp32"])
        return c
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


def _pack4(x):
    """Values [..., dim] as (codes [..., dim / 2], scale words [..., dim / 32]); what x's type keeps decides."""
    g = x.reshape(*x.shape[:-1], -1, GROUP).clamp(-MOST, MOST)
    lo, hi = g.amin(dim=-1).clamp(max=0), g.amax(dim=-1).clamp(min=0)
    step = (hi - lo) / 15
    unit = torch.exp2(torch.floor(torch.log2(step.clamp(min=2.0 ** -14))) - 6)  # a power of two within one of the right one
    unit = torch.where(step < 64 * unit, unit / 2, torch.where(step >= 128 * unit, unit * 2, unit)).clamp(min=2.0 ** -20)
    scale = (torch.ceil(step / unit) * unit).clamp(min=2.0 ** -20)
    zero = torch.round(-lo / scale)
    codes = (torch.round(g / scale[..., None]) + zero[..., None]).clamp(0, 15).to(torch.uint8).reshape(x.shape)
    words = scale.half().view(torch.int16) | zero.to(torch.int16)
    return codes[..., 0::2] | (codes[..., 1::2] << 4), words


def _cache(gen, kv, *shape):
    """Cache rows ~ N(0, 1): 4-bit codes with a word per 32 dims, or int8 codes with a scale per 64."""
    x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float16)
    if kv == "int4":
        parts = [_pack4(part.float()) for part in x.flatten(0, -3).split(64)]  # some heads at a time
        codes, words = (torch.cat(t) for t in zip(*parts))
        return codes.reshape(*shape[:-1], -1), words.reshape(*shape[:-1], -1)
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


def _starts(case, room):
    """Per sequence a first row that leaves `room` rows behind it."""
    return [n - 1 for n in reversed(_lengths(case, case["rows"] - room + 1))]


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen, kind = _gen(seed), case["kind"]
    s = {"case": case, "kind": kind}
    n = case["seqs"]
    if kind == "sample":
        s["logits"] = _randn(gen, n, case["vocab"]) * 3.0
        s["uniform"] = torch.rand(n, generator=gen, device="cuda")
        # each row's settings near the case's; a filter that is off stays off
        near = 0.9 + 0.2 * torch.rand((3, n), generator=gen, device="cuda")
        s["temperature"] = case["temperature"] * near[0]
        s["top_k"] = None if case["top_k"] == 0 else _ints([case["top_k"] + i % 3 for i in range(n)])
        s["top_p"] = None if case["top_p"] >= 1.0 else (case["top_p"] * near[1]).clamp(max=0.999)
        s["min_p"] = None if case["min_p"] <= 0.0 else case["min_p"] * near[2]
        return s
    h, kvh, d, rows = case["heads"], case["kv_heads"], case["dim"], case["rows"]
    kv = case.get("kv", "int4")
    if kind == "prefix":
        s["k_prefix"], s["k_prefix_scale"] = _cache(gen, kv, kvh, case["prefix"], d)
        s["v_prefix"], s["v_prefix_scale"] = _cache(gen, kv, kvh, case["prefix"], d)
    s["k"], s["k_scale"] = _cache(gen, kv, n, kvh, rows, d)
    s["v"], s["v_scale"] = _cache(gen, kv, n, kvh, rows, d)
    if kind == "append":
        s["qkv"] = _randn(gen, n * case["tokens"], (h + 2 * kvh) * d)
        s["pos"] = _ints(_starts(case, case["tokens"]))
        half = case["rotary"] // 2
        freq = 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
        s["offset"] = 100
        angle = torch.arange(rows + s["offset"], device="cuda", dtype=torch.float64)[:, None] * freq
        s["cos"], s["sin"] = torch.cos(angle).float(), torch.sin(angle).float()
    elif kind == "read":
        s["pos"] = _ints(_starts(case, case["take"]))
    elif kind == "prefix":
        s["q"] = _randn(gen, n, h, d)
        s["pos"] = _ints(_own_positions(case))
    else:
        s["q"] = _randn(gen, n, case["tokens"], h, d)
        first = _first_positions(case)
        s["pos"] = _ints(first)
        # the cache rows from which any token of the call sees, per sequence, and how many there are at most
        w, t = case["window"], case["tokens"]
        low = [max(case["sinks"], p - w + 1) if w else 0 for p in first]
        s["low"] = torch.tensor(low, device="cuda")
        s["span"] = max([p + t - a for p, a in zip(first, low)] + [0])
    return s


# -------------------------------------------------------------- plain forms
def _rows_of(cache, scale, *at):
    """The rows `at` of a cache in 32 bits (all without `at`)."""
    x, scale = (cache[at], scale[at]) if at else (cache, scale)
    if cache.dtype == torch.int8:
        x = x.float()
        return (x.reshape(*x.shape[:-1], -1, KV_BLOCK) * scale[..., None]).reshape(x.shape)
    codes = torch.stack((x & 15, x >> 4), dim=-1).to(torch.float32)
    codes = codes.reshape(*x.shape[:-1], -1, GROUP)
    step = (scale & ~15).view(torch.float16).float()
    return ((codes - (scale & 15).float()[..., None]) * step[..., None]).reshape(*x.shape[:-1], -1)


def _plain_append(s):
    c = s["case"]
    n, t, h, kvh, d, half = c["seqs"], c["tokens"], c["heads"], c["kv_heads"], c["dim"], c["rotary"] // 2
    x = s["qkv"].reshape(n, t, h + 2 * kvh, d)
    rows = s["pos"].long()[:, None] + torch.arange(t, device=x.device)
    cos, sin = s["cos"][rows + s["offset"]][:, :, None], s["sin"][rows + s["offset"]][:, :, None]

    def turn(x, cos, sin):
        a, b = x[..., :half], x[..., half:2 * half]
        return torch.cat((a * cos - b * sin, a * sin + b * cos, x[..., 2 * half:]), dim=3)

    seq = torch.arange(n, device=x.device)[:, None]
    # in 64 bits, so that a code next to a border is the definition's
    keys = turn(x[:, :, h:h + kvh].double(), cos.double(), sin.double())
    s["k"][seq, :, rows], s["k_scale"][seq, :, rows] = _pack4(keys)
    s["v"][seq, :, rows], s["v_scale"][seq, :, rows] = _pack4(x[:, :, h + kvh:].double())
    return {"q": turn(x[:, :, :h], cos, sin).reshape(n * t, h * d),
            "k": _rows_of(s["k"], s["k_scale"]).half(), "v": _rows_of(s["v"], s["v_scale"]).half()}


def _plain_read(s):
    c = s["case"]
    seq = torch.arange(c["seqs"], device="cuda")[:, None, None]
    head = torch.arange(c["kv_heads"], device="cuda")[:, None]
    at = s["pos"].long()[:, None, None] + torch.arange(c["take"], device="cuda")
    to = torch.float16 if c["to"] == "fp16" else torch.float32
    return {"k": _rows_of(s["k"], s["k_scale"], seq, head, at).to(to),
            "v": _rows_of(s["v"], s["v_scale"], seq, head, at).to(to)}


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


def _plain_sample(s):
    """Weights and their sums in 64 bits: a running sum decides the token."""
    x = s["logits"]
    n, v = x.shape
    ranked, order = torch.sort(x, dim=1, descending=True, stable=True)
    w = torch.exp((ranked.double() - ranked[:, :1].double()) / s["temperature"].double()[:, None])
    rank = torch.arange(v, device=x.device)
    if s["top_k"] is not None:
        w = torch.where(rank < s["top_k"][:, None], w, 0.0)
    if s["top_p"] is not None:
        before = torch.cumsum(w, dim=1) - w
        w = torch.where((before < s["top_p"].double()[:, None] * w.sum(dim=1, keepdim=True)) | (rank == 0), w, 0.0)
    if s["min_p"] is not None:
        w = torch.where((w >= s["min_p"].double()[:, None]) | (rank == 0), w, 0.0)
    kept = torch.zeros_like(w).scatter_(1, order, w)
    total = torch.cumsum(kept, dim=1)
    past = total > s["uniform"].double()[:, None] * total[:, -1:]
    token = torch.where(past, rank, v - 1).amin(dim=1)
    chance = kept.gather(1, token[:, None])[:, 0] / total[:, -1]
    return {"tokens": token.to(torch.int32), "probs": chance.float()}


def _own_run(s):
    from asdsl import kernels

    kind, c = s["kind"], s["case"]
    if kind == "append":
        q = kernels.kv_append(s["qkv"], s["k"], s["v"], s["cos"], s["sin"], s["pos"], n_heads=c["heads"],
                              pos_offset=s["offset"], k_scale=s["k_scale"], v_scale=s["v_scale"])
        k, v = kernels.kv_read(s["k"], s["v"], k_scale=s["k_scale"], v_scale=s["v_scale"])
        return {"q": q, "k": k, "v": v}
    if kind == "read":
        k, v = kernels.kv_read(s["k"], s["v"], pos=s["pos"], n_rows=c["take"], k_scale=s["k_scale"],
                               v_scale=s["v_scale"], dtype=torch.float16 if c["to"] == "fp16" else torch.float32)
        return {"k": k, "v": v}
    if kind == "window":
        return kernels.attention_window(s["q"], s["k"], s["v"], s["pos"], window=c["window"], sinks=c["sinks"],
                                        k_scale=s["k_scale"], v_scale=s["v_scale"])
    if kind == "prefix":
        return kernels.attention_prefix(s["q"], s["k_prefix"], s["v_prefix"], s["k"], s["v"], s["pos"],
                                        k_prefix_scale=s["k_prefix_scale"], v_prefix_scale=s["v_prefix_scale"],
                                        k_scale=s["k_scale"], v_scale=s["v_scale"])
    tokens, probs = kernels.sample_logits(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"],
                                          top_p=s["top_p"], min_p=s["min_p"])
    return {"tokens": tokens, "probs": probs}


def run(state):
    if own:
        return _own_run(state)
    return {"append": _plain_append, "read": _plain_read, "window": _plain_window, "prefix": _plain_prefix,
            "sample": _plain_sample}[state["kind"]](state)


# ------------------------------------------------------------- what it takes
def _row_bytes(c):
    """Bytes of one position's K and V rows over all KV heads."""
    return 2 * c["kv_heads"] * c["dim"] * (0.5 + 2.0 / GROUP if c.get("kv", "int4") == "int4" else 1.0 + 4.0 / KV_BLOCK)


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
    if kind == "sample":
        return {"bytes": 4 * n * c["vocab"] + 28 * n, "flops": 4 * n * c["vocab"]}
    width, values = c["heads"] * c["dim"], 2 * c["kv_heads"] * c["dim"]
    if kind == "append":
        t = n * c["tokens"]
        table = 4 * c["rotary"] * min(t, c["rows"])
        back = n * c["rows"] * (_row_bytes(c) + 2 * values)  # the caches read back as fp16
        return {"bytes": t * (4 * (width + values) + 4 * width + _row_bytes(c)) + table + back,
                "flops": 3 * t * (width + 2 * values) + 2 * n * c["rows"] * values}
    if kind == "read":
        t = n * c["take"]
        return {"bytes": t * (_row_bytes(c) + (2 if c["to"] == "fp16" else 4) * values), "flops": 2 * t * values}
    if kind == "window":
        rows, pairs = _visible(c)
        return {"bytes": rows * _row_bytes(c) + 8 * n * c["tokens"] * width, "flops": 4 * pairs * width}
    own_rows = sum(p + 1 for p in _own_positions(c))
    return {"bytes": (c["prefix"] + own_rows) * _row_bytes(c) + 8 * n * width,
            "flops": 4 * (n * c["prefix"] + own_rows) * width}


# ------------------------------------------------------------------ 64 bits
def _wide(cache, scale):
    """A cache's values, from its bits."""
    if cache.dtype == torch.int8:
        return cache.double() * scale.double().repeat_interleave(KV_BLOCK, dim=-1)
    dims = torch.arange(2 * cache.shape[-1], device=cache.device)
    code = (cache[..., dims // 2].int() >> (4 * (dims % 2)).int()) % 16
    word = scale.int()[..., dims // GROUP] & 0xFFFF
    power, part, zero = word // 1024, word // 16 % 64, word % 16  # scales are positive
    step = torch.where(power > 0, (64 + part).double() * torch.exp2((power - 21).double()), part * 2.0 ** -20)
    return (code - zero).double() * step


def _quantised(x):
    """The values for which 4 bits stand, of x [..., dim] in 64 bits, on the host."""
    x = np.clip(x, -MOST, MOST)
    g = x.reshape(-1, GROUP)
    lo, hi = np.minimum(g.min(axis=1), 0.0), np.maximum(g.max(axis=1), 0.0)
    step = (hi - lo) / 15.0
    _, e = np.frexp(step)  # step in [2^(e-1), 2^e)
    unit = np.ldexp(1.0, np.maximum(e - 7, -20))
    step = np.maximum(np.ceil(step / unit) * unit, 2.0 ** -20)[:, None]
    zero = np.rint(-lo[:, None] / step)
    return ((np.clip(np.rint(g / step) + zero, 0, 15) - zero) * step).reshape(x.shape)


def _attend(q, k, v, seen):
    """softmax(q k' / sqrt(d)) v over the rows that `seen` (tokens x rows) leaves; q (tokens, heads of one KV head, d)."""
    out = torch.zeros_like(q)
    for h in range(q.shape[1]):
        w = torch.where(seen, torch.exp((q[:, h] @ k.T / math.sqrt(q.shape[2])).clamp(-600, 600)), 0.0)
        total = w.sum(dim=1, keepdim=True)
        out[:, h] = (w @ v) / torch.where(total > 0, total, torch.ones_like(total))
    return out


def _exact_sample(s, n):
    x = s["logits"].cpu().numpy().astype(np.float64)
    host = {name: None if s[name] is None else s[name].cpu().numpy() for name in ("uniform", "temperature", "top_k",
                                                                                  "top_p", "min_p")}
    tokens, probs = [], []
    for i in range(n):
        order = np.argsort(-x[i], kind="stable")
        w = np.exp((x[i][order] - x[i][order[0]]) / np.float64(host["temperature"][i]))
        if host["top_k"] is not None:
            order, w = order[:host["top_k"][i]], w[:host["top_k"][i]]
        if host["top_p"] is not None:
            run_sum = np.cumsum(w)
            most = int(np.searchsorted(run_sum, np.float64(host["top_p"][i]) * run_sum[-1], side="left")) + 1
            order, w = order[:most], w[:most]
        if host["min_p"] is not None:
            most = max(1, int((w >= np.float64(host["min_p"][i])).sum()))
            order, w = order[:most], w[:most]
        by_id = np.argsort(order)
        run_sum = np.cumsum(w[by_id])
        at = min(int(np.searchsorted(run_sum, np.float64(host["uniform"][i]) * run_sum[-1], side="right")),
                 len(order) - 1)
        tokens.append(int(order[by_id[at]]))
        probs.append(float(w[by_id[at]] / run_sum[-1]))
    return {"tokens": _ints(tokens), "probs": torch.tensor(probs, dtype=torch.float64, device="cuda")}


def exact(case, seed):
    s, kind, n = prepare(case, seed), case["kind"], case["seqs"]
    if kind == "sample":
        return _exact_sample(s, n)
    h, kvh, d = case["heads"], case["kv_heads"], case["dim"]
    g = h // kvh
    if kind == "append":
        t, half = case["tokens"], case["rotary"] // 2
        k, v = _wide(s["k"], s["k_scale"]), _wide(s["v"], s["v_scale"])
        q = torch.zeros((n, t, h, d), dtype=torch.float64, device="cuda")
        x = s["qkv"].double().reshape(n, t, h + 2 * kvh, d)
        for i in range(n):
            p = int(s["pos"][i])
            cos, sin = (s[name][p + s["offset"]:p + s["offset"] + t].double()[:, None] for name in ("cos", "sin"))
            turned = x[i, :, :h + kvh].clone()
            a, b = x[i, :, :h + kvh, :half], x[i, :, :h + kvh, half:2 * half]
            turned[..., :half], turned[..., half:2 * half] = a * cos - b * sin, b * cos + a * sin
            q[i] = turned[:, :h]
            for cache, new in ((k, turned[:, h:]), (v, x[i, :, h + kvh:])):
                cache[i, :, p:p + t] = torch.from_numpy(_quantised(new.transpose(0, 1).cpu().numpy())).cuda()
        return {"q": q.reshape(n * t, h * d), "k": k, "v": v}
    if kind == "read":
        at = [int(p) for p in s["pos"]]
        return {name: torch.stack([_wide(s[name][i, :, p:p + case["take"]], s[name + "_scale"][i, :, p:p + case["take"]])
                                   for i, p in enumerate(at)]) for name in ("k", "v")}
    q = s["q"].double()
    out = torch.zeros_like(q)
    if kind == "prefix":
        for j in range(kvh):
            kp, vp = _wide(s["k_prefix"][j], s["k_prefix_scale"][j]), _wide(s["v_prefix"][j], s["v_prefix_scale"][j])
            for i in range(n):
                m = int(s["pos"][i]) + 1
                ko, vo = _wide(s["k"][i, j, :m], s["k_scale"][i, j, :m]), _wide(s["v"][i, j, :m], s["v_scale"][i, j, :m])
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
            k, v = (_wide(s[name][i, j, :len(key)], s[name + "_scale"][i, j, :len(key)]) for name in ("k", "v"))
            out[i, :, j * g:(j + 1) * g] = _attend(q[i, :, j * g:(j + 1) * g], k, v, seen)
    return out
