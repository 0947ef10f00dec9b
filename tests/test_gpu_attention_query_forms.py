"""The shapes in which attention_window takes its queries give one result."""

from __future__ import annotations

import numpy as np
import ops_reference as ref
import pytest
from test_gpu_attention_ops import check, dev, make_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,tokens", [(3, 1), (1, 3), (3, 5)])
def test_query_shapes_over_one_kv_head(gpu, heads, tokens):
    import torch

    from asdsl.kernels import attention_window

    rng = np.random.default_rng(heads * 10 + tokens)
    n, d, rows, pos = 2, 128, 40, [20, 7]
    q = rng.standard_normal((n, tokens, heads, d)).astype(np.float32)
    k, _, kw = make_cache(rng, "fp16", n, 1, rows, d)
    v, _, vw = make_cache(rng, "fp16", n, 1, rows, d)
    want, bound = ref.window(q, kw, vw, pos, 0, 0)
    p = dev(np.array(pos, np.int32))
    got = attention_window(dev(q), k, v, p)
    check(got, want, bound)
    for shape in ((n * tokens * heads, d), (n * tokens, heads * d), (n, tokens * heads, d), (n * tokens * heads * d,)):
        again = attention_window(dev(q.reshape(shape)), k, v, p, n_heads=heads)
        assert again.shape == shape and torch.equal(again.reshape(q.shape), got)
