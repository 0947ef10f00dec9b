"""How attention_window reads its queries' shape: before any HIP call here."""

from __future__ import annotations

import pytest


def test_which_heads_a_flat_query_holds():
    import torch

    from asdsl.kernels import attention_window

    one = torch.zeros((2, 1, 8, 128), dtype=torch.float16)  # two sequences, one KV head
    pos = torch.zeros(2, dtype=torch.int32)

    def refused(text, *shape, k=one, **args):
        with pytest.raises(ValueError, match=text):
            attention_window(torch.zeros(shape), k, k, pos, **args)
    # three tokens of one head, or one token of three heads
    refused("n_heads", 6, 128)
    refused("n_heads", 4, 128)
    # these say it, and are refused later, as they are on no device
    for shape, args in (((6, 128), {"n_heads": 1}), ((6, 128), {"n_heads": 3}), ((2, 128), {}), ((6, 256), {}),
                        ((2, 3, 128), {}), ((2, 3, 1, 128), {}), ((2, 3, 128), {"n_heads": 1})):
        refused("device", *shape, **args)
    for n in (0, -1, 2, 7):
        refused("must be", 6, 128, n_heads=n)
    four = torch.zeros((2, 4, 8, 128), dtype=torch.float16)
    refused("must be", 6, 128, k=four, n_heads=1)
    refused("must be", 8, 128, k=four)  # no multiple of the KV heads
    refused("device", 8, 128, k=four, n_heads=4)
