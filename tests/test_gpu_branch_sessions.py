"""BranchDecoder between its calls: a start that fails, tokens that a caller
forces, masks that raise, an engine whose rows change under it."""

from __future__ import annotations

import numpy as np
import pytest
from test_gpu_branches import VOCAB, engine, prompt_of

pytestmark = pytest.mark.gpu


def test_a_start_that_fails_leaves_nothing_to_step(gpu):
    """Refused by the engine behind its reset (as a chunk, and as a verify
    pass), or by the control: no step over what is left of the rows."""
    from asdsl.inference.branches import BranchDecoder, TokenControl

    b = BranchDecoder(engine(), 2, 8)
    for bad in (([VOCAB],), ([1, 2, 3, 4, VOCAB],), ([1, 2], TokenControl(repetition=0.0)),
                ([1, 2], TokenControl(bias={3: "x"}))):
        b.start(prompt_of(20))
        b.step()
        b.step()
        with pytest.raises(ValueError):
            b.start(*bad)
        for call in (b.step, b.forward):
            with pytest.raises(RuntimeError, match="start"):
                call()
    # refused before the engine is touched: the prompt is still there
    b.start(prompt_of(20))
    b.step()
    for bad in ([], [1] * 249):
        with pytest.raises(ValueError):
            b.start(bad)
    b.step()
    assert [len(r) for r in b.continuations()] == [3, 3]
