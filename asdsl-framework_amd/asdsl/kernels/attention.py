"""Attention of many tokens and sequences over KV caches, on the HIP library.

``kv_append`` rotates queries and keys and writes the new cache rows,
``kv_read`` reads rows of quantized caches back, ``attention_window`` attends
with a sliding window and first tokens that stay visible, ``attention_prefix``
attends for sequences that share a prefix.  The caches are the decode engine's
(fp16, or int8 codes with one fp32 scale per 64 dims) or hold 4 bits a value,
with a leading sequence dimension where there are several.

A 4-bit cache is uint8 [..., rows, head_dim / 2], two codes a byte, the low
nibble the even dim's, with int16 scale words [..., rows, head_dim / 32]: a word
is an fp16 scale of 7 significant bits whose 4 low bits hold a zero point z, and
a value is (code - z) * scale, which is exactly an fp16 number.  0.5625 bytes a
value, where int8 takes 1.0625 and fp16 2.  Every tensor
is a contiguous device tensor of the current device, used as it is; calls are
queued on the current stream and can be captured.  No counterpart in the
reference, which decodes one sequence (asdsl/kernels/native/unified_engine.cpp:1339-1688).
"""

from __future__ import annotations

import functools

from asdsl import _hip
from asdsl.kernels._buffers import _Tensor

try:
    from torch import cuda as _cuda
    from torch import empty_like as _empty_like
    from torch import float16 as _f16
    from torch import float32 as _f32
    from torch import int8 as _i8
    from torch import int16 as _i16
    from torch import int32 as _i32
    from torch import uint8 as _u8
    from torch._C import _cuda_getCurrentRawStream as _raw_stream  # without a Stream object
except ImportError:  # no tensors without torch: every call is refused
    _cuda = _empty_like = _f16 = _f32 = _i8 = _i16 = _i32 = _u8 = _raw_stream = None

KV_BLOCK = 64  # dims per scale of an int8 cache
KV_GROUP = 32  # dims per scale word of a 4-bit cache


def _stream(dev: int) -> int:
    """The current stream of the current device dev."""
    return _raw_stream(dev) if _raw_stream is not None else _hip.stream_handle()


def _device(t) -> int:
    """The current device, which the call's tensors have to be on (no device where t, one of them, is on none)."""
    return _cuda.current_device() if isinstance(t, _Tensor) and t.is_cuda else -2


def _addr(fn: str, dev: int, name: str, t, dtype, n: int) -> int:
    """The address of a contiguous tensor of n elements on device dev.  A call
    of small sizes is bound by its host time, most of which is these checks:
    the good case is one expression."""
    if isinstance(t, _Tensor) and t.dtype is dtype and t.numel() == n and t.get_device() == dev and t.is_contiguous():
        return t.data_ptr()
    if not isinstance(t, _Tensor):
        raise ValueError(f"{fn}: {name} must be a device tensor")
    if t.dtype is not dtype:
        raise ValueError(f"{fn}: {name} must be {dtype}, got {t.dtype}")
    if t.numel() != n:
        raise ValueError(f"{fn}: {name} has {t.numel()} elements, needs {n}")
    if not t.is_cuda:
        raise ValueError(f"{fn}: {name} must be a device tensor")
    if t.get_device() != dev:
        raise ValueError(f"{fn}: {name} is on device {t.get_device()}, the current one is {dev}")
    raise ValueError(f"{fn}: {name} must be contiguous")


def _cache_dims(fn: str, name: str, k, v, dims: int = 4) -> tuple:
    """(n_seq, n_kv_heads, rows, head_dim) of a pair of caches; three dimensions are one sequence."""
    if not isinstance(k, _Tensor) or not isinstance(v, _Tensor):
        raise ValueError(f"{fn}: {name} caches must be device tensors")
    shape = tuple(k.shape)
    if tuple(v.shape) != shape or v.dtype is not k.dtype:
        raise ValueError(f"{fn}: the {name} caches differ in shape or type")
    if len(shape) != dims and len(shape) != 3:
        raise ValueError(f"{fn}: a {name} cache has {len(shape)} dimensions, {3 if dims == 3 else '3 or 4'} are wanted")
    d = shape[-1]
    if k.dtype is _u8:
        d *= 2
    elif k.dtype is not _f16 and k.dtype is not _i8:
        raise ValueError(f"{fn}: a {name} cache is fp16 or int8 or uint8 (4-bit codes), got {k.dtype}")
    if 0 in shape[:-2] or d not in (64, 128):
        raise ValueError(f"{fn}: {name} cache of shape {shape}; head_dim must be 64 or 128")
    return (*shape[:-1], d) if len(shape) == 4 else (1, *shape[:-1], d)


def _caches(fn: str, dev: int, name: str, k, v, k_scale, v_scale, head_dim: int) -> tuple:
    """Addresses of a pair of caches (k, v), and of their scales for the int8 and 4-bit forms (k, v, k_scale, v_scale)."""
    dtype, n = k.dtype, k.numel()
    if dtype is _f16:
        if k_scale is not None or v_scale is not None:
            raise ValueError(f"{fn}: {name} caches take scales exactly where they are int8 or 4-bit")
        return _addr(fn, dev, f"{name} keys", k, dtype, n), _addr(fn, dev, f"{name} values", v, dtype, n)
    if k_scale is None or v_scale is None:
        raise ValueError(f"{fn}: {name} caches take scales exactly where they are int8 or 4-bit")
    scale, m = (_f32, n // KV_BLOCK) if dtype is _i8 else (_i16, 2 * n // KV_GROUP)
    return (_addr(fn, dev, f"{name} keys", k, dtype, n), _addr(fn, dev, f"{name} values", v, dtype, n),
            _addr(fn, dev, f"{name} key scales", k_scale, scale, m),
            _addr(fn, dev, f"{name} value scales", v_scale, scale, m))


# The entry points' names end in the caches' form.
_APPEND = {_f16: "asdsl_kv_append_f16", _i8: "asdsl_kv_append_q8", _u8: "asdsl_kv_append_q4"}
_WINDOW = {_f16: "asdsl_attention_window_f16kv", _i8: "asdsl_attention_window_q8kv",
           _u8: "asdsl_attention_window_q4kv"}
_PREFIX = {_f16: "asdsl_attention_prefix_f16kv", _i8: "asdsl_attention_prefix_q8kv",
           _u8: "asdsl_attention_prefix_q4kv"}
_READ = {_i8: "asdsl_kv_read_q8", _u8: "asdsl_kv_read_q4"}


def _heads(fn: str, q, head_dim: int, n_rows: int, what: str = "q") -> int:
    """Heads of a tensor with n_rows rows of whole heads."""
    if not isinstance(q, _Tensor):
        raise ValueError(f"{fn}: {what} must be a device tensor")
    n = q.numel()
    if n == 0 or n % (n_rows * head_dim):
        raise ValueError(f"{fn}: {what} of shape {tuple(q.shape)} does not hold {n_rows} rows of heads of {head_dim}")
    return n // (n_rows * head_dim)


def _count(fn: str, name: str, v) -> int:
    """A length that the C ABI takes as an int."""
    n = int(v)
    if not 0 <= n < 1 << 31:
        raise ValueError(f"{fn}: {name} must be in [0, 2^31), got {n}")
    return n


def _work(nbytes: int, like):
    """A work buffer of this call on its stream (None where it needs none)."""
    return like.new_empty(nbytes, dtype=_u8) if nbytes else None


@functools.lru_cache(maxsize=4096)
def _work_bytes(entry: str, *dims) -> int:
    """Bytes of work that a call of an entry point, and so over its form of caches, needs."""
    return getattr(_hip.LIB, entry + "_work_bytes")(*dims)


def kv_append(qkv, k_cache, v_cache, rope_cos, rope_sin, pos, *, n_heads: int, pos_offset: int = 0, k_scale=None,
              v_scale=None, q_out=None):
    """Rotated queries and new cache rows of the tokens of one or more sequences.

    qkv: fp32, per token [q | k | v] of n_heads + 2 * kv_heads heads; its
    tokens are shared evenly by the cache's sequences, sequence by sequence.
    k_cache, v_cache: [n_seq, kv_heads, rows, head_dim] (or one sequence's
    [kv_heads, rows, head_dim]), fp16, or int8 with k_scale and v_scale fp32
    [..., rows, head_dim / 64], or uint8 [..., rows, head_dim / 2] with int16
    [..., rows, head_dim / 32] (4 bits).  Token t of sequence s is written to cache row
    pos[s] + t (pos: int32 [n_seq]) and rotated for position pos[s] + t +
    pos_offset of the tables rope_cos and rope_sin [positions, rotary_dim / 2].
    Returns the rotated queries, fp32 [tokens, n_heads * head_dim] (in q_out if
    given).  A token outside the cache or the tables writes nothing, and its
    queries are zero.

    4 bits: per 32 dims, held to +-2^15, with lo = min(0, x) and hi = max(0, x),
    scale = (hi - lo) / 15 rounded up to 7 significant bits (below 2^-14 to a
    multiple of 2^-20, at least 2^-20), z = round(-lo / scale) and code =
    clamp(round(x / scale) + z, 0, 15), half to even, in 64-bit arithmetic on
    rotated keys and values; 32 dims with a value that is not finite read as
    NaN."""
    fn = "kv_append"
    n_seq, n_kv, rows, d = _cache_dims(fn, "kv", k_cache, v_cache)
    n_heads, pos_offset = int(n_heads), _count(fn, "pos_offset", pos_offset)
    if n_heads <= 0 or n_heads % n_kv:
        raise ValueError(f"{fn}: n_heads must be a multiple of the caches' {n_kv} heads")
    if not isinstance(qkv, _Tensor) or qkv.numel() == 0 or qkv.numel() % (n_seq * (n_heads + 2 * n_kv) * d):
        raise ValueError(f"{fn}: qkv does not hold tokens of {n_heads + 2 * n_kv} heads of {d} for {n_seq} sequences")
    tokens = qkv.numel() // ((n_heads + 2 * n_kv) * d)
    if not isinstance(rope_cos, _Tensor) or not isinstance(rope_sin, _Tensor) or rope_cos.dim() != 2 \
            or rope_cos.shape != rope_sin.shape:
        raise ValueError(f"{fn}: rope_cos and rope_sin must be tensors [positions, rotary_dim / 2] of one shape")
    rope_rows, half = rope_cos.shape
    dev = _device(qkv)
    at = (_addr(fn, dev, "qkv", qkv, _f32, qkv.numel()), *_caches(fn, dev, "kv", k_cache, v_cache, k_scale, v_scale, d),
          _addr(fn, dev, "rope_cos", rope_cos, _f32, rope_rows * half),
          _addr(fn, dev, "rope_sin", rope_sin, _f32, rope_rows * half), _addr(fn, dev, "pos", pos, _i32, n_seq))
    if q_out is None:
        q_out = qkv.new_empty((tokens, n_heads * d))
    _hip.call(_APPEND[k_cache.dtype], *at,
              _addr(fn, dev, "q_out", q_out, _f32, tokens * n_heads * d), n_seq, tokens // n_seq, n_heads, n_kv, d,
              2 * half, rows, pos_offset, rope_rows, _stream(dev))
    return q_out


def kv_read(k_cache, v_cache, *, pos=None, n_rows: int | None = None, k_scale=None, v_scale=None, dtype=None,
            out=None):
    """Rows of int8 or 4-bit caches as the values they stand for: (k, v).

    Caches and scales as in kv_append.  Rows pos[s] .. pos[s] + n_rows - 1 of
    each sequence (pos: int32 [n_seq], default the first row; n_rows default:
    all of a cache's) come as [n_seq, kv_heads, n_rows, head_dim] (without the
    first dimension for one sequence's caches of three) of dtype float16 (the
    default) or float32, in the pair out if given.  int8 values are code * scale
    in fp32, rounded once more to fp16; 4-bit values are exact.  Rows outside
    the cache read as zero."""
    fn = "kv_read"
    n_seq, n_kv, rows, d = _cache_dims(fn, "kv", k_cache, v_cache)
    if k_cache.dtype is _f16:
        raise ValueError(f"{fn}: fp16 caches hold their values; int8 or 4-bit ones are wanted")
    n_rows = rows if n_rows is None else _count(fn, "n_rows", n_rows)
    if n_rows == 0:
        raise ValueError(f"{fn}: n_rows must be positive")
    if out is not None and (not isinstance(out, (tuple, list)) or len(out) != 2
                            or not all(isinstance(t, _Tensor) for t in out)):
        raise ValueError(f"{fn}: out must be a pair of device tensors")
    dtype = (out[0].dtype if out is not None else _f16) if dtype is None else dtype
    if dtype is not _f16 and dtype is not _f32:
        raise ValueError(f"{fn}: values are float16 or float32, not {dtype}")
    dev = _device(k_cache)
    at = (*_caches(fn, dev, "kv", k_cache, v_cache, k_scale, v_scale, d),
          None if pos is None else _addr(fn, dev, "pos", pos, _i32, n_seq))
    if out is None:
        shape = (*k_cache.shape[:-2], n_rows, d)
        out = k_cache.new_empty(shape, dtype=dtype), k_cache.new_empty(shape, dtype=dtype)
    k, v = out
    n = n_seq * n_kv * n_rows * d
    _hip.call(_READ[k_cache.dtype], *at, _addr(fn, dev, "k out", k, dtype, n), _addr(fn, dev, "v out", v, dtype, n),
              int(dtype is _f32), n_seq, n_kv, d, rows, n_rows, _stream(dev))
    return k, v


def attention_window(q, k_cache, v_cache, pos, *, n_heads: int | None = None, window: int = 0, sinks: int = 0,
                     k_scale=None, v_scale=None, out=None):
    """Attention over KV caches with a sliding window and first tokens that stay visible.

    q: fp32, the tokens of the caches' sequences, sequence by sequence, each
    n_heads heads of head_dim: [..., n_heads, head_dim] of three dimensions or
    more, or [tokens, n_heads * head_dim], or with n_heads given any shape.
    (Rows of one head_dim over one KV head could be tokens of one head or one
    token's heads: without n_heads they are refused.)  Caches as in kv_append.  Token t of sequence s
    is at position p = pos[s] + t and sees cache rows j <= p with j < sinks or
    j > p - window (window 0: all j <= p).  Returns softmax(q.K /
    sqrt(head_dim)) V in q's shape (in out if given); a token whose position
    is outside the cache sees nothing and gets zero."""
    fn = "attention_window"
    n_seq, n_kv, rows, d = _cache_dims(fn, "kv", k_cache, v_cache)
    per_seq = _heads(fn, q, d, n_seq)  # tokens * heads
    if n_heads is not None:
        n_heads = int(n_heads)
    elif q.dim() == 2 and n_kv == 1 and q.shape[-1] == d and per_seq > 1:
        raise ValueError(f"{fn}: q of shape {tuple(q.shape)} over one KV head is tokens or heads: give n_heads")
    else:
        n_heads = q.shape[-2] if q.dim() >= 3 and q.shape[-1] == d else q.shape[-1] // d if q.shape[-1] % d == 0 else 0
    if n_heads <= 0 or per_seq % n_heads or n_heads % n_kv:
        raise ValueError(f"{fn}: q must be [..., n_heads, {d}] or [tokens, n_heads * {d}], n_heads a multiple of {n_kv}")
    n = q.numel()
    tokens = per_seq // n_heads
    dims = (n_seq, tokens, n_heads, n_kv, d, rows, _count(fn, "window", window), _count(fn, "sinks", sinks))
    dev = _device(q)
    at = (_addr(fn, dev, "q", q, _f32, n), *_caches(fn, dev, "kv", k_cache, v_cache, k_scale, v_scale, d),
          _addr(fn, dev, "pos", pos, _i32, n_seq))
    if out is None:
        out = _empty_like(q)
    entry = _WINDOW[k_cache.dtype]
    nbytes = _work_bytes(entry, *dims)
    work = _work(nbytes, q)
    _hip.call(entry, *at,
              _addr(fn, dev, "out", out, _f32, n), *dims, None if work is None else work.data_ptr(), nbytes,
              _stream(dev))
    return out


def attention_prefix(q, k_prefix, v_prefix, k_own, v_own, own_pos, *, prefix_len: int | None = None,
                     k_prefix_scale=None, v_prefix_scale=None, k_scale=None, v_scale=None, out=None):
    """Attention of one token each of sequences that share a prefix.

    q: fp32 [n_seq, n_heads, head_dim] or [n_seq, n_heads * head_dim].
    Sequence s sees the first prefix_len rows (default: all) of the prefix
    caches [kv_heads, prefix rows, head_dim], which are read once for all
    sequences, and rows 0 .. own_pos[s] (int32; -1: none) of its own caches
    [n_seq, kv_heads, rows, head_dim]; both fp16, or both int8 or 4-bit with
    their scales, as in kv_append.  Returns softmax(q.K / sqrt(head_dim)) V
    in q's shape (in out if given); zero for a sequence that sees nothing or
    whose own_pos is outside [-1, rows)."""
    fn = "attention_prefix"
    n_seq, n_kv, rows, d = _cache_dims(fn, "own", k_own, v_own)
    _, p_kv, prefix_rows, p_d = _cache_dims(fn, "prefix", k_prefix, v_prefix, 3)
    if (p_kv, p_d) != (n_kv, d) or k_prefix.dtype is not k_own.dtype:
        raise ValueError(f"{fn}: the prefix and own caches differ in heads, head_dim or type")
    n_heads = _heads(fn, q, d, n_seq)
    if n_heads % n_kv:
        raise ValueError(f"{fn}: q has {n_heads} heads, no multiple of the caches' {n_kv}")
    prefix_len = prefix_rows if prefix_len is None else int(prefix_len)
    if not 0 <= prefix_len <= prefix_rows:
        raise ValueError(f"{fn}: prefix_len must be in [0, {prefix_rows}], got {prefix_len}")
    n = q.numel()
    dev = _device(q)
    at = (_addr(fn, dev, "q", q, _f32, n),
          *_caches(fn, dev, "prefix", k_prefix, v_prefix, k_prefix_scale, v_prefix_scale, d),
          *_caches(fn, dev, "own", k_own, v_own, k_scale, v_scale, d), _addr(fn, dev, "own_pos", own_pos, _i32, n_seq))
    if out is None:
        out = _empty_like(q)
    entry = _PREFIX[k_own.dtype]
    nbytes = _work_bytes(entry, n_seq, n_heads, n_kv, d, prefix_len, rows)
    work = _work(nbytes, q)
    _hip.call(entry, *at,
              _addr(fn, dev, "out", out, _f32, n), n_seq, n_heads, n_kv, d, prefix_len, prefix_rows, rows,
              None if work is None else work.data_ptr(), nbytes, _stream(dev))
    return out
