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


def test_forwarded_tokens_are_the_history(gpu):
    """Tokens given to forward() are the continuations that control and masks
    see; a step() behind a forward() chooses from that pass and runs none."""
    import torch

    from asdsl.inference.branches import BranchDecoder, TokenControl

    n, steps = 3, 4
    own = np.random.default_rng(4).permutation(VOCAB)[:n * steps].reshape(steps, n)
    asked = []

    def mask(rows):
        asked.append([list(r) for r in rows])
    eng, other, ids = engine(), engine(), prompt_of(30)
    b = BranchDecoder(eng, n, steps + 1)
    b.start(ids, TokenControl(frequency=1000.0, bias={int(t): 500.0 for t in own.flat}, allowed=mask))
    for i in range(steps):
        logits = b.forward(own[i])
        assert b.continuations() == own[:i + 1].T.tolist()
    raw = logits.cpu().numpy()
    with pytest.raises(RuntimeError, match="chosen"):
        b.forward()
    b.step()
    y = raw.copy()
    y[:, own.reshape(-1)] += np.float32(500)
    for j in range(n):
        y[j, own[:, j]] = raw[j, own[:, j]] - np.float32(1000) + np.float32(500)
    chosen = y.argmax(axis=1)
    assert asked[-1] == own.T.tolist() and b.own_pos.tolist() == [steps] * n
    assert b.continuations() == [[*own[:, j].tolist(), int(chosen[j])] for j in range(n)]
    # that token is passed once, in the next row
    b.step()
    assert b.own_pos.tolist() == [steps + 1] * n and [len(r) for r in b.continuations()] == [steps + 2] * n
    other.prefill(ids)
    for i, t in enumerate([*own[:, 1].tolist(), int(chosen[1])]):
        other.forward_token(t, len(ids) + i)
    at = len(ids)
    assert torch.equal(b.k[0, 1], other.layers[0]["k_cache"][:, at:at + steps + 1])
    # full: nothing more is passed or chosen
    for call in (b.step, lambda: b.forward([1] * n)):
        with pytest.raises(ValueError, match="stepped"):
            call()


def test_forward_between_steps(gpu):
    """Steps (queued, then replayed), a pass over the chosen tokens or over
    others in their place, and the choice behind it: the plain steps' run."""
    import torch

    from asdsl.inference.branches import BranchDecoder, TokenControl

    control = TokenControl(repetition=1.3, frequency=0.5, presence=0.1)
    plain, mixed = (BranchDecoder(engine("int8"), 4, 12) for _ in range(2))
    for b in (plain, mixed):
        b.start(prompt_of(25), control)
    for _ in range(12):
        plain.step()
    for i in range(6):
        mixed.step()
        mixed.forward() if i % 2 else mixed.forward(mixed.tokens.tolist())
        mixed.step()
    assert mixed.continuations() == plain.continuations() and mixed.own_pos.tolist() == plain.own_pos.tolist()
    assert torch.equal(mixed.k, plain.k) and torch.equal(mixed.logits, plain.logits)
    # a token in place of the chosen one
    mixed.start(prompt_of(25), control)
    first = mixed.continuations()
    mixed.forward([7, 8, 9, 10])
    assert mixed.continuations() == [[7], [8], [9], [10]] != first


@pytest.mark.parametrize("words", [None, 3, "text"])
def test_a_mask_that_fails_leaves_the_step_undone(gpu, words):
    """A mask that raises once, or gives what is no mask: the step can be
    taken again."""
    import torch

    from asdsl.inference.branches import BranchDecoder, TokenControl

    failed = []

    def mask(rows):
        if len(rows[0]) == 3 and not failed:
            failed.append(True)
            if words is None:
                raise KeyError("grammar")
            return torch.zeros(words, dtype=torch.int32) if words == 3 else words
        return None
    plain, b = (BranchDecoder(engine(), 3, 6) for _ in range(2))
    plain.start(prompt_of(20))
    b.start(prompt_of(20), TokenControl(allowed=mask))
    for i in range(6):
        plain.step()
        if i == 2:
            with pytest.raises((KeyError, ValueError)):
                b.step()
        b.step()
    assert failed and b.continuations() == plain.continuations()
    assert b.own_pos.tolist() == plain.own_pos.tolist() and torch.equal(b.k, plain.k)


def test_the_engines_rows_changed_under_the_decoder(gpu):
    """The prompt's rows are the engine's.  Whatever changes them ends the
    decoder's run with an error; what leaves them alone does not."""
    from asdsl.inference.branches import BranchDecoder

    eng, ids = engine(), prompt_of(30)
    b, second = BranchDecoder(eng, 2, 12), BranchDecoder(eng, 3, 4)
    want = b.generate(ids, eos=())
    for change in (eng.reset_session, lambda: eng.prefill(prompt_of(5)), lambda: eng.prefill([1, 2]),
                   lambda: eng.forward_token(5, 29), lambda: eng.forward_batch_all_logits([1, 2, 3], 28),
                   lambda: eng.truncate_kv(29), lambda: eng.prefill_kv_random(7),
                   lambda: (eng.truncate_kv(29), eng.step()), lambda: second.start(prompt_of(6))):
        b.start(ids)
        b.step()
        change()
        for call in (b.step, b.forward):
            with pytest.raises(RuntimeError, match="rows"):
                call()
    second.step()  # the newer one goes on, also behind a change of rows that only the older one had
    eng.step()
    second.step()
    b.start(ids)
    for harmless in (lambda: eng.forward_token(5, 30), lambda: eng.truncate_kv(30), eng.step, eng.verify_next_tokens,
                     lambda: eng.forward_batch_all_logits([1, 2, 3], 40), eng.snapshot_kv, eng.capture, eng.next_token):
        b.step()
        harmless()
    while len(b.continuations()[0]) < 12:
        b.step()
    assert b.continuations() == want


def test_buffers_outlive_their_launches(gpu, monkeypatch):
    """A start() replaces buffers that steps queued on another stream may still
    use: their memory is not handed out again on the stream that allocated
    them while those steps have not run."""
    import torch

    from asdsl.inference.branches import BranchDecoder, TokenControl

    eng = engine()
    eng.graph_calls = False  # to drop a graph waits for its replays
    b = BranchDecoder(eng, 4, 8)
    control = TokenControl(repetition=1.2)
    b.start(prompt_of(40), control)
    torch.cuda.synchronize()
    sizes = {t.data_ptr(): t.numel() * t.element_size()
             for t in (b._work, b.history, b.history_len, *b._control.values())}
    for stream in (torch.cuda.current_stream(), side := torch.cuda.Stream()):
        with torch.cuda.stream(stream):  # room in the allocator: to ask the driver for more waits
            room = [torch.empty(n, dtype=torch.uint8, device="cuda") for n in (1 << 20, *sizes.values()) for _ in range(40)]
            del room
    main = torch.cuda.current_stream()
    got, kept, full = [], [], torch.full

    def later(*a, **k):
        """Called by start() behind each buffer that it has replaced."""
        with torch.cuda.stream(main):
            kept.extend(torch.empty(n, dtype=torch.uint8, device="cuda") for n in sizes.values())
        got.extend(t.data_ptr() for t in kept)
        return full(*a, **k)

    ids = torch.tensor(prompt_of(41), dtype=torch.int32, device="cuda")  # an upload would wait for the work queued
    with torch.cuda.stream(side):
        b.step()
        b.step()
        torch.cuda._sleep(1_500_000_000)
        with monkeypatch.context() as m:
            m.setattr(eng, "prefill", lambda tokens: None)
            m.setattr(torch, "full", later)
            m.setattr(torch, "tensor", lambda *a, **k: ids)
            b.start(prompt_of(41), control)
    assert len(got) > 3 * len(sizes) and not set(got) & set(sizes)
    torch.cuda.synchronize()


def test_first_tokens_by_the_rule_of_every_choice(gpu):
    """The largest controlled logits, ties to the lower token, a NaN never, as
    control_logits takes them one by one; one mask for all, or a row each."""
    import torch

    from asdsl.inference.branches import BranchDecoder, TokenControl

    tied = [1500, 700, 41, 9, 3, 2047]
    level = torch.zeros(VOCAB)
    level[tied] = 1e9  # the logits beside it are less than half a step
    level[5] = float("nan")
    for rows in (False, True):
        words = torch.full((4, VOCAB // 32) if rows else (VOCAB // 32,), -1, dtype=torch.int32)
        for n, want in ((1, [3]), (4, [3, 9, 41, 700])):
            b = BranchDecoder(engine(), n, 2)
            b.start(prompt_of(20), TokenControl(bias=level, allowed=words[:n] if rows else words))
            assert b.tokens.tolist() == want and b.continuations() == [[t] for t in want]
    level[8] = float("inf")
    b = BranchDecoder(engine(), 3, 2)
    b.start(prompt_of(20), TokenControl(bias=level))
    assert b.tokens.tolist() == [8, 3, 9]
    # a row whose only token an earlier one took
    may = np.zeros((2, VOCAB // 32), np.int32)
    may[0, 0], may[1, 0] = 0b11, 0b01
    b = BranchDecoder(engine(), 2, 2)
    with pytest.raises(ValueError, match="fewer than 2 .*continuation 1"):
        b.start(prompt_of(20), TokenControl(bias={0: 1e6}, allowed=torch.from_numpy(may)))
    b.start(prompt_of(20), TokenControl(bias={1: 1e6}, allowed=torch.from_numpy(may)))
    assert b.tokens.tolist() == [1, 0]
