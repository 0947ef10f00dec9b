"""Several continuations of one prompt, decoded together.

``BranchDecoder`` prefills the prompt once on a ``DecodeEngine`` and then steps
n continuations in one pass (asdsl_decode_branches): the weights stream once
for all of them, the prompt's K/V rows are read once for all, and every
continuation keeps its own rows in a cache of its own.  The next tokens are
the greedy ones of the controlled logits (asdsl.kernels.control_logits:
penalties, biases, a grammar's mask).  No counterpart in the reference, which
decodes one sequence (asdsl/inference/unified_bridge.py:360-421).
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Any

from asdsl import _hip
from asdsl.inference.unified_bridge import PHI4_EOS, _engine_of
from asdsl.kernels import control_logits


class _BranchLayer(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("k", "v", "k_scale", "v_scale")]


@dataclass
class TokenControl:
    """What bears on the choice of the next token (asdsl.kernels.control_logits).

    repetition, frequency, presence: penalties for tokens of the prompt and the
    continuation (repetition) and of the continuation alone.  bias: {token: value}
    or a float tensor [vocab].  allowed: int32 mask words [words] or [n, words],
    or a callable that takes the continuations so far (a list of n token lists)
    and returns such words (or None: everything is allowed) before each choice."""

    repetition: float = 1.0
    frequency: float = 0.0
    presence: float = 0.0
    bias: Any = None
    allowed: Any = None


class BranchDecoder:
    """n continuations of one prompt of at most max_new_tokens tokens each.

    store: a weight store or a DecodeEngine, whose caches hold the prompt's
    rows.  An engine call that changes any of them between start() and the
    last step(), another decoder's start() among them, ends the run: the next
    step() or forward() raises RuntimeError."""

    CHUNK = 16  # steps between two reads of the device's tokens in generate()

    def __init__(self, store: Any, n: int, max_new_tokens: int):
        import torch

        eng = self.engine = _engine_of(store)
        c = eng.cfg
        self.n, self.own_rows = int(n), int(max_new_tokens)
        if not 1 <= self.n <= 256:
            raise ValueError("BranchDecoder: 1..256 continuations")
        if not 1 <= self.own_rows <= c.max_seq:
            raise ValueError(f"BranchDecoder: max_new_tokens must be in [1, {c.max_seq}]")
        dev = eng.token.device
        shape = (c.n_layers, self.n, c.n_kv_heads, self.own_rows, c.head_dim)
        self.k = torch.zeros(shape, dtype=torch.int8 if eng.kv_int8 else torch.float16, device=dev)
        self.v = torch.zeros_like(self.k)
        self.k_scale = self.v_scale = None
        if eng.kv_int8:
            self.k_scale = torch.ones(shape[:-1] + (c.head_dim // 64,), dtype=torch.float32, device=dev)
            self.v_scale = torch.ones_like(self.k_scale)
        self._own = (_BranchLayer * c.n_layers)()
        for i in range(c.n_layers):
            for name in ("k", "v", "k_scale", "v_scale"):
                t = getattr(self, name)
                setattr(self._own[i], name, None if t is None else _hip.ptr(t[i]))
        self.logits = torch.empty((self.n, c.vocab), dtype=torch.float32, device=dev)
        self.tokens = torch.zeros(self.n, dtype=torch.int32, device=dev)
        self.own_pos = torch.zeros(self.n, dtype=torch.int32, device=dev)
        self.prefix_len = -1  # nothing started
        self._steps = 0  # passes run
        self._passed = False  # whether self.tokens have been through one
        self._graph = None

    # ------------------------------------------------------------ one prompt
    def start(self, prompt_ids, control: TokenControl | None = None):
        """Prefill the prompt; the first tokens are the n best of its controlled
        logits (device int32 [n], also in self.tokens), all different: each
        continuation in turn takes the best (as control_logits chooses) that
        its mask allows and no earlier one has taken, and where none is left
        ValueError is raised.  If it raises, the next call has to be
        another start(), unless it refused the prompt's length (nothing was
        touched then)."""
        import torch

        eng, c = self.engine, self.engine.cfg
        prompt = [int(t) for t in prompt_ids]
        if not prompt:
            raise ValueError("BranchDecoder.start: empty prompt")
        if len(prompt) + self.own_rows > c.max_seq:
            raise ValueError("BranchDecoder.start: prompt and continuation out of kv-cache range")
        self.prefix_len, self._steps, self._graph = -1, 0, None  # nothing to step from until all of this is done
        eng.reset_session()
        eng.prefill(prompt)
        self._rows = eng.hold_rows(len(prompt))
        nbytes = _hip.LIB.asdsl_decode_branches_work_bytes(ctypes.byref(eng._model), self.n, len(prompt),
                                                           self.own_rows)
        if nbytes == 0:
            raise ValueError(f"BranchDecoder: {_hip.last_error()}")
        dev = self.tokens.device
        self._stream = _hip.stream_handle()  # which allocates what follows
        self._work = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        self.own_pos.zero_()
        self.history = torch.full((self.n, len(prompt) + self.own_rows + 1), -1, dtype=torch.int32, device=dev)
        self.history[:, :len(prompt)] = torch.tensor(prompt, dtype=torch.int32, device=dev)
        self.history_len = torch.full((self.n,), len(prompt), dtype=torch.int32, device=dev)
        try:
            self.prefix_len = len(prompt)
            self._set_control(control or TokenControl())
            self._note(self._first_tokens())
        except BaseException:
            self.prefix_len = -1
            raise
        return self.tokens

    def _first_tokens(self):
        """Each continuation in turn takes the token that control_logits
        chooses among those that its mask allows and no earlier one has taken."""
        import torch

        vocab = self.engine.cfg.vocab
        logits = self.engine.logits.reshape(1, -1)
        if self._allowed is None or self._allowed.numel() == (vocab + 31) // 32:  # one mask for all
            rows, _ = control_logits(logits, pick=False, **self._control_args(1))
            rows = rows.expand(self.n, -1)
        else:
            rows, _ = control_logits(logits.expand(self.n, -1).contiguous(), pick=False, **self._control_args(self.n))
        open_ = torch.ones(vocab, dtype=torch.bool, device=rows.device)
        tokens = torch.empty(self.n, dtype=torch.int64, device=rows.device)
        values = torch.empty(self.n, device=rows.device)
        for i in range(self.n):
            left = rows[i].masked_fill(~open_, float("-inf"))
            _, token = control_logits(left)
            tokens[i:i + 1] = token.clamp(min=0)
            values[i:i + 1] = left.index_select(0, tokens[i:i + 1])
            open_.index_fill_(0, tokens[i:i + 1], False)
        taken = (values > float("-inf")).tolist()
        if not all(taken):
            raise ValueError(f"BranchDecoder.start: fewer than {self.n} tokens to begin with: none is left for "
                             f"continuation {taken.index(False)}")
        return tokens.to(torch.int32)

    def _set_control(self, control: TokenControl) -> None:
        import torch

        vocab, dev = self.engine.cfg.vocab, self.tokens.device
        self._control = {}
        if (control.repetition, control.frequency, control.presence) != (1.0, 0.0, 0.0):
            if not control.repetition > 0:
                raise ValueError("TokenControl: repetition must be positive")
            self._control = {name: torch.full((self.n,), float(getattr(control, name)), device=dev)
                             for name in ("repetition", "frequency", "presence")}
            self._control["prompt_len"] = torch.full_like(self.history_len, self.prefix_len)
        bias = control.bias
        if isinstance(bias, dict):
            if any(not 0 <= int(t) < vocab for t in bias):
                raise ValueError("TokenControl: bias of a token out of vocab range")
            ids = [int(t) for t in bias]
            bias = torch.zeros(vocab, dtype=torch.float32)
            bias[ids] = torch.tensor([float(v) for v in control.bias.values()])
        self._bias = None if bias is None else bias.to(dev, torch.float32).contiguous()
        self._mask = control.allowed if callable(control.allowed) else None
        self._allowed = None if self._mask or control.allowed is None else \
            control.allowed.to(dev, torch.int32).contiguous()
        self._ask()

    def _ask(self) -> None:
        """A callable mask's words for the next choice."""
        if self._mask is not None:
            import torch

            words = self._mask(self.continuations())
            if words is not None and not isinstance(words, torch.Tensor):
                raise ValueError("TokenControl: allowed must give int32 mask words or None")
            self._allowed = None if words is None else words.to(self.tokens.device).contiguous()

    def _control_args(self, rows: int) -> dict:
        args = {name: t[:rows] for name, t in self._control.items()}
        if args:
            args |= {"history": self.history[:rows], "history_len": self.history_len[:rows]}
        allowed = self._allowed
        if allowed is not None and allowed.dim() == 2:
            allowed = allowed[:rows]
        return args | {"bias": self._bias, "allowed": allowed}

    def _note(self, tokens) -> None:
        """The chosen tokens into the history; what the next step takes."""
        self.tokens.copy_(tokens)
        self.history.scatter_(1, self.history_len.long().unsqueeze(1), self.tokens.unsqueeze(1))
        self.history_len.add_(1)
        self._passed = False

    # -------------------------------------------------------------- stepping
    def _forward(self) -> None:
        eng = self.engine
        _hip.check(_hip.LIB.asdsl_decode_branches(ctypes.byref(eng._model), self._own, self.n, self.prefix_len,
                                                  self.own_rows, _hip.ptr(self.tokens), _hip.ptr(self.own_pos),
                                                  _hip.ptr(self.logits), _hip.ptr(self._work), self._work.numel(),
                                                  _hip.stream_handle()),
                   "asdsl_decode_branches")
        self.own_pos.add_(1)

    def _choose(self) -> None:
        _, tokens = control_logits(self.logits, out=self.logits, **self._control_args(self.n))
        self._note(tokens)

    def _started(self) -> None:
        if self.prefix_len < 0:
            raise RuntimeError("BranchDecoder: start() has not been called")
        if self._rows != self.engine._rows_version:
            raise RuntimeError("BranchDecoder: the engine's prompt rows have changed since start()")
        if _hip.stream_handle() != self._stream:
            import torch

            # The next start() replaces these while launches queued here may
            # still use them: their memory must not go to the next tensor of
            # the stream that allocated them before those are done.
            for t in (self._work, self.history, self.history_len, self._bias, self._allowed, *self._control.values()):
                if t is not None:
                    t.record_stream(torch.cuda.current_stream())

    def _room(self) -> None:
        self._started()
        if self._steps >= self.own_rows:
            raise ValueError(f"BranchDecoder: {self.own_rows} tokens a continuation are stepped")

    def forward(self, tokens=None):
        """One pass over self.tokens, or over the given n tokens: the n rows of
        logits (device [n, vocab]), nothing chosen.  Given tokens take the
        place of chosen ones that no pass has had; behind another forward()
        they go on from its tokens.  All of them are part of the continuations,
        as control and masks see them.  A step() behind it chooses from these
        logits and runs no pass of its own."""
        import torch

        self._room()
        if tokens is not None:
            ids = [int(t) for t in tokens]
            if len(ids) != self.n or any(not 0 <= t < self.engine.cfg.vocab for t in ids):
                raise ValueError(f"BranchDecoder.forward: {self.n} tokens of the vocabulary are wanted")
            if not self._passed:
                self.history_len.sub_(1)
            self._note(torch.tensor(ids, dtype=torch.int32))
        elif self._passed:
            raise RuntimeError("BranchDecoder.forward: no tokens were given or chosen since the last pass")
        self._forward()
        self._steps, self._passed = self._steps + 1, True
        return self.logits

    def step(self) -> None:
        """One pass over self.tokens (unless forward() has run it) and the
        choice of the next ones (then in self.tokens; self.logits are the
        controlled ones).  Queued eagerly the first time and replayed from a
        HIP graph from the second on, as the engine's steps are; token,
        position and history advance on the device.  Where a mask raises or
        gives no mask the pass has run, and another step() asks again."""
        import torch

        self._started()
        if self._passed:
            self._ask()
            self._choose()
            return
        self._room()
        graphs = self._mask is None and self.engine.graph_calls and not torch.cuda.is_current_stream_capturing()
        if graphs and self._graph is not None:
            self._graph.replay()
            self._steps += 1
            return
        self.forward()  # if the choice fails, the next step() has only that left to do
        self._ask()
        self._choose()
        if not graphs:
            return
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            self._forward()
            self._choose()
        self._graph = graph

    def continuations(self) -> list[list[int]]:
        """The tokens chosen or given so far, per continuation (one device
        read); -1 where nothing was allowed."""
        return self.history[:, self.prefix_len:int(self.history_len[0])].tolist()

    def generate(self, prompt_ids, max_new_tokens: int | None = None, control: TokenControl | None = None,
                 eos=PHI4_EOS) -> list[list[int]]:
        """n continuations, each up to max_new_tokens (default: the decoder's),
        an end-of-sequence token, which is not returned, or a place where
        nothing is allowed.  The first tokens are
        the n best after the prompt, the others each continuation's own greedy
        ones under control.  A continuation that has ended is stepped on with
        the others and cut."""
        most = self.own_rows if max_new_tokens is None else int(max_new_tokens)
        if not 0 <= most <= self.own_rows:
            raise ValueError(f"BranchDecoder.generate: max_new_tokens must be in [0, {self.own_rows}]")
        if most == 0:
            return [[] for _ in range(self.n)]
        ends = {int(t) for t in eos} | {-1}
        self.start(prompt_ids, control)
        while True:
            out = self.continuations()
            if len(out[0]) >= most or all(any(t in ends for t in row) for row in out):
                break
            for _ in range(min(self.CHUNK, most - len(out[0]))):
                self.step()
        return [row[:next((i for i, t in enumerate(row) if t in ends), most)] for row in out]
