"""Plain implementations in 64 bits (numpy, on the host) of the operators of
many sequences, written from their definitions, and bounds on what fp32
arithmetic may be off from them."""

from __future__ import annotations

import numpy as np

EPS = 2.0 ** -24  # half a step of fp32


def wide(cache, scale=None):
    """A cache as the values it stands for."""
    x = np.asarray(cache, np.float64)
    if scale is not None:
        x = x * np.repeat(np.asarray(scale, np.float64), 64, axis=-1)
    return x


def attend_row(q, k, v):
    """(out, bound) of one query row over the rows k, v it sees.

    The bound counts, for each weight: the score's fp32 products and sums
    (n terms: n EPS times the sum of magnitudes, and 2^-22 of it where the
    query is held as two 11-bit parts), the rounding of the scaled score and of
    its distance from the maximum (4 EPS of the largest), the exponential
    (2 EPS) and its two-part form (2^-22); then the sums over the keys
    (one EPS a key).  Numerator and denominator may each be off by that."""
    d = q.shape[-1]
    if len(k) == 0:
        return np.zeros(d), np.zeros(d)
    with np.errstate(all="ignore"):
        s = k @ q / np.sqrt(d)
        mags = np.max(np.abs(k) @ np.abs(q)) / np.sqrt(d)
        w = np.exp(s - s.max())
        p = w / w.sum()
        off = (d * EPS + 2.0 ** -22) * mags + 4 * EPS * np.max(np.abs(s)) + 2 * EPS + 2.0 ** -22 + len(k) * EPS
        return p @ v, 2 * off * (p @ np.abs(v)) + 1e-37


def seen_rows(p, rows, window, sinks):
    """The cache rows that a token at position p sees."""
    if p < 0 or p >= rows:
        return np.zeros(0, np.int64)
    j = np.arange(p + 1)
    return j if window == 0 else j[(j < sinks) | (j > p - window)]


def window(q, k, v, pos, win, sinks):
    """q [n_seq, tokens, heads, d]; k, v [n_seq, kv_heads, rows, d] (wide); (out, bound)."""
    n, t, h, d = q.shape
    g = h // k.shape[1]
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for i in range(n):
        for j in range(t):
            at = seen_rows(int(pos[i]) + j, k.shape[2], win, sinks)
            for a in range(h):
                out[i, j, a], bound[i, j, a] = attend_row(q[i, j, a].astype(np.float64), k[i, a // g, at],
                                                          v[i, a // g, at])
    return out, bound


def prefix(q, kp, vp, prefix_len, ko, vo, own_pos):
    """q [n_seq, heads, d]; kp, vp [kv_heads, rows, d]; ko, vo [n_seq, kv_heads, rows, d] (wide); (out, bound)."""
    n, h, d = q.shape
    g = h // ko.shape[1]
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for i in range(n):
        m = int(own_pos[i]) + 1
        if m < 0 or m > ko.shape[2]:
            continue
        for a in range(h):
            k = np.concatenate([kp[a // g, :prefix_len], ko[i, a // g, :m]])
            v = np.concatenate([vp[a // g, :prefix_len], vo[i, a // g, :m]])
            out[i, a], bound[i, a] = attend_row(q[i, a].astype(np.float64), k, v)
    return out, bound


def rotate(x, cos, sin, half):
    """Heads x [..., heads, d] rotated by the angles of their token, cos/sin [..., half]."""
    x = np.asarray(x, np.float64)
    a, b = x[..., :half], x[..., half:2 * half]
    c, s = np.asarray(cos, np.float64)[..., None, :], np.asarray(sin, np.float64)[..., None, :]
    return np.concatenate([a * c - b * s, a * s + b * c, x[..., 2 * half:]], axis=-1)


def control(logits, history=None, prompt_len=None, history_len=None, repetition=None, frequency=None, presence=None,
            bias=None, allowed=None):
    """(out, tokens): each step in 32 bits, as the definition rounds."""
    f = np.float32
    rows, vocab = logits.shape
    out, tokens = np.empty_like(logits), []
    with np.errstate(all="ignore"):
        for r in range(rows):
            y = logits[r].astype(f)
            if history is not None:
                cap = history.shape[1]
                told = min(max(int(history_len[r]) if history_len is not None else cap, 0), cap)
                start = int(prompt_len[r]) if prompt_len is not None else 0
                ids = history[r, :told]
                ok = (ids >= 0) & (ids < vocab)
                seen = np.zeros(vocab, bool)
                seen[ids[ok]] = True
                made = ok & (np.arange(told) >= start)
                times = np.bincount(ids[made], minlength=vocab).astype(f)
                rep = f(1) if repetition is None else f(repetition[r])
                y = np.where(seen, np.where(y > 0, y / rep, y * rep), y).astype(f)
                if frequency is not None:
                    y = (y - f(frequency[r]) * times).astype(f)
                if presence is not None:
                    y = np.where(times > 0, y - f(presence[r]), y).astype(f)
            if bias is not None:
                y = (y + (bias if bias.ndim == 1 else bias[r])).astype(f)
            may = np.ones(vocab, bool)
            if allowed is not None:
                words = (allowed if allowed.ndim == 1 else allowed[r]).astype(np.uint32)
                v = np.arange(vocab)
                may = (words[v // 32] >> (v % 32).astype(np.uint32)) & 1 != 0
            out[r] = np.where(may, y, f(-np.inf))
            best = np.where(may & ~np.isnan(y), y, f(-np.inf))
            can = np.flatnonzero(may & ~np.isnan(y))
            tokens.append(int(can[np.argmax(best[can])]) if len(can) else -1)
    return out, np.array(tokens, np.int32)
