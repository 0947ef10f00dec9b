"""Control of the next token on the HIP library: penalties for tokens that
occurred, biases, a grammar's mask, and the greedy token of what is left.  No
counterpart in the reference, whose decoding is plain greedy
(asdsl/kernels/native/unified_engine.cpp:207-233)."""

from __future__ import annotations

from asdsl import _hip
from asdsl.kernels._buffers import _Tensor
from asdsl.kernels.attention import _addr, _empty, _f32, _i32, _work


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
    words = (vocab + 31) // 32
    strides = []
    for name, t, width in (("bias", bias, vocab), ("allowed", allowed, words)):
        if t is None:
            strides.append(0)
        elif isinstance(t, _Tensor) and t.dim() in (1, 2) and t.shape[-1] == width and t.numel() in (width, rows * width):
            strides.append(0 if t.numel() == width else width)
        else:
            raise ValueError(f"{fn}: {name} must be a device tensor [{width}] or [{rows}, {width}]")

    def opt(name, t, dtype, count):
        return None if t is None else _addr(fn, name, t, dtype, count)

    a_logits = _addr(fn, "logits", logits, _f32, n)
    a_history = opt("history", history, _i32, rows * cap) if cap else None
    a_prompt = opt("prompt_len", prompt_len, _i32, rows) if cap else None
    a_len = opt("history_len", history_len, _i32, rows) if cap else None
    a_rep = opt("repetition", repetition, _f32, rows) if cap else None
    a_freq = opt("frequency", frequency, _f32, rows) if cap else None
    a_pres = opt("presence", presence, _f32, rows) if cap else None
    a_bias = None if bias is None else _addr(fn, "bias", bias, _f32, bias.numel())
    a_allowed = None if allowed is None else _addr(fn, "allowed", allowed, _i32, allowed.numel())
    if out is None:
        out = _empty(logits.shape, dtype=_f32, device=logits.device)
    a_out = _addr(fn, "out", out, _f32, n)
    tokens = work = None
    nbytes = 0
    if pick:
        tokens = _empty(rows, dtype=_i32, device=logits.device)
        nbytes = _hip.LIB.asdsl_logits_control_work_bytes(rows, vocab)
        work = _work(nbytes, logits)
    _hip.call("asdsl_logits_control", a_logits, a_out, None if tokens is None else tokens.data_ptr(), a_history,
              a_prompt, a_len, cap, a_rep, a_freq, a_pres, a_bias, strides[0], a_allowed, strides[1], rows, vocab,
              None if work is None else work.data_ptr(), nbytes, _hip.stream_handle())
    return out, tokens
