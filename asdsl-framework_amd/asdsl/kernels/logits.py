"""The choice of the next token on the HIP library: penalties for tokens that
occurred, biases, a grammar's mask, and the greedy token of what is left; or a
token drawn with temperature, top-k, top-p and min-p.  No counterpart in the
reference, whose decoding is plain greedy
(asdsl/kernels/native/unified_engine.cpp:207-233)."""

from __future__ import annotations

import functools

from asdsl import _hip
from asdsl.kernels._buffers import _Tensor
from asdsl.kernels.attention import _addr, _device, _empty_like, _f32, _i32, _stream, _work


@functools.lru_cache(maxsize=4096)
def _control_bytes(rows: int, vocab: int) -> int:
    return _hip.LIB.asdsl_logits_control_work_bytes(rows, vocab)


def control_logits(logits, *, history=None, prompt_len=None, history_len=None, repetition=None, frequency=None,
                   presence=None, bias=None, allowed=None, out=None, pick: bool = True):
    """Controlled logits and the greedy token of each row: (out, tokens).

    logits: fp32 [rows, vocab] (or one row's [vocab]).  history: int32 token
    ids [rows, most]; a row's first history_len (int32 [rows]; default: all)
    count, and the first prompt_len (int32 [rows]; default: none) of those are
    its prompt; ids outside the vocabulary (a padding of -1) are skipped.
    repetition, frequency, presence: fp32 [rows].  Per row, each step rounded
    to fp32:

        y = x / repetition if x > 0 else x * repetition    for tokens of the history
        y -= frequency * n, then y -= presence             for tokens that occur
                                                           n > 0 times past the prompt
        y += bias                                          fp32 [vocab] or [rows, vocab]
        y = -inf                                           where allowed's bit is clear

    allowed: int32 words [words] or [rows, words], words = (vocab + 31) // 32,
    bit v % 32 of word v // 32 for token v (compute_activation_bitmask's form).
    Returns out (a new tensor unless given; may be logits itself) and int32
    tokens [rows]: the first largest allowed value, -1 where nothing is
    allowed; a NaN is never taken.  pick=False: (out, None)."""
    fn = "control_logits"
    if not isinstance(logits, _Tensor) or logits.dim() not in (1, 2) or logits.numel() == 0:
        raise ValueError(f"{fn}: logits must be a device tensor [rows, vocab] or [vocab]")
    vocab = logits.shape[-1]
    n = logits.numel()
    rows = n // vocab
    cap = 0
    if history is None:
        for name, t in (("prompt_len", prompt_len), ("history_len", history_len), ("repetition", repetition),
                        ("frequency", frequency), ("presence", presence)):
            if t is not None:
                raise ValueError(f"{fn}: {name} without a history")
    elif not isinstance(history, _Tensor) or history.dim() not in (1, 2) \
            or (history.shape[0] if history.dim() == 2 else 1) != rows:
        raise ValueError(f"{fn}: history must be a device tensor [{rows}, ids]")
    else:
        cap = history.shape[-1]
        if cap > 1 << 30:
            raise ValueError(f"{fn}: a history of at most 2^30 ids a row")
    words = (vocab + 31) // 32
    strides = []
    for name, t, width in (("bias", bias, vocab), ("allowed", allowed, words)):
        if t is None:
            strides.append(0)
        elif isinstance(t, _Tensor) and t.dim() in (1, 2) and t.shape[-1] == width and t.numel() in (width, rows * width):
            strides.append(0 if t.numel() == width else width)
        else:
            raise ValueError(f"{fn}: {name} must be a device tensor [{width}] or [{rows}, {width}]")

    dev = _device(logits)
    a_logits = _addr(fn, dev, "logits", logits, _f32, n)
    a_history = a_prompt = a_len = a_rep = a_freq = a_pres = None
    if cap:
        a_history = _addr(fn, dev, "history", history, _i32, rows * cap)
        if prompt_len is not None:
            a_prompt = _addr(fn, dev, "prompt_len", prompt_len, _i32, rows)
        if history_len is not None:
            a_len = _addr(fn, dev, "history_len", history_len, _i32, rows)
        if repetition is not None:
            a_rep = _addr(fn, dev, "repetition", repetition, _f32, rows)
        if frequency is not None:
            a_freq = _addr(fn, dev, "frequency", frequency, _f32, rows)
        if presence is not None:
            a_pres = _addr(fn, dev, "presence", presence, _f32, rows)
    a_bias = None if bias is None else _addr(fn, dev, "bias", bias, _f32, bias.numel())
    a_allowed = None if allowed is None else _addr(fn, dev, "allowed", allowed, _i32, allowed.numel())
    if out is None:
        out = _empty_like(logits)
    a_out = _addr(fn, dev, "out", out, _f32, n)
    tokens = work = None
    nbytes = 0
    if pick:
        tokens = logits.new_empty(rows, dtype=_i32)
        nbytes = _control_bytes(rows, vocab)
        work = _work(nbytes, logits)
    _hip.call("asdsl_logits_control", a_logits, a_out, None if tokens is None else tokens.data_ptr(), a_history,
              a_prompt, a_len, cap, a_rep, a_freq, a_pres, a_bias, strides[0], a_allowed, strides[1], rows, vocab,
              None if work is None else work.data_ptr(), nbytes, _stream(dev))
    return out, tokens


@functools.lru_cache(maxsize=4096)
def _sample_bytes(rows: int, vocab: int, cuts: bool) -> int:
    return _hip.LIB.asdsl_sample_logits_work_bytes_cuts(rows, vocab, cuts)


def sample_logits(logits, uniform, *, temperature=None, top_k=None, top_p=None, min_p=None):
    """A token of each row drawn by its weights, and the share it had: (tokens, probs).

    logits: fp32 [rows, vocab] (or one row's [vocab]), vocab at most 2^20, as
    control_logits leaves them (pick=False).  uniform: fp32 [rows], the random
    numbers, in [0, 1).  temperature, top_p, min_p: fp32 [rows]; top_k: int32
    [rows]; each may be left out.  Per row, with the tokens ranked by logit and
    equal ones by index:

        w(v) = exp((x(v) - max x) / temperature)   (temperature left out: 1)
        kept are the first top_k                   (0 or less: all)
        of those the shortest part of the ranking that comes to
            top_p of their total                   (1 or more: all; 0 or less: the first)
        of those the ones with w >= min_p          (and always the first)
        token = in index order the first whose running sum of kept weights
            exceeds uniform * their sum

    Weights are whole multiples of 2^-43, so sums are exact and a call gives the
    same each time.  -inf and NaN are never taken; where the largest is +inf,
    those share evenly.  A temperature that is not above 0 takes the first of the
    ranking.  Returns int32 tokens [rows], -1 where no token has a weight, and
    fp32 probs [rows], the token's share of the kept weights (0 for -1)."""
    fn = "sample_logits"
    if not isinstance(logits, _Tensor) or logits.dim() not in (1, 2) or logits.numel() == 0:
        raise ValueError(f"{fn}: logits must be a device tensor [rows, vocab] or [vocab]")
    vocab = logits.shape[-1]
    n = logits.numel()
    rows = n // vocab
    if vocab > 1 << 20:
        raise ValueError(f"{fn}: a vocabulary of at most 2^20 tokens")
    dev = _device(logits)
    at = (_addr(fn, dev, "logits", logits, _f32, n), _addr(fn, dev, "uniform", uniform, _f32, rows),
          None if temperature is None else _addr(fn, dev, "temperature", temperature, _f32, rows),
          None if top_k is None else _addr(fn, dev, "top_k", top_k, _i32, rows),
          None if top_p is None else _addr(fn, dev, "top_p", top_p, _f32, rows),
          None if min_p is None else _addr(fn, dev, "min_p", min_p, _f32, rows))
    tokens, probs = logits.new_empty(rows, dtype=_i32), logits.new_empty(rows)
    nbytes = _sample_bytes(rows, vocab, top_k is not None or top_p is not None)
    work = _work(nbytes, logits)
    _hip.call("asdsl_sample_logits", *at, tokens.data_ptr(), probs.data_ptr(), rows, vocab,
              None if work is None else work.data_ptr(), nbytes, _stream(dev))
    return tokens, probs
