"""Beam search as a loop: the tables, scores, pool and logits that it carries from step to step, and the calls
of `Sampler` that make a step, in their order.

    search = BeamSearch(sampler, groups, beams, max_steps, vocab, config, head=Head(weight))
    search.begin()
    while not finished:
        hidden = model(search.tokens, caches)              # [groups * beams, hidden] bfloat16
        search.step(hidden, states=caches, lens=used, position_dim=2)
    found = search.result()

The reference has no generation at all; its nearest call site is the per-batch loop of
examples/mnist/main.go:229-245.  Everything stays on the device; nothing synchronises but the making of a search
with a history, which waits until its memory is zeroed.  A search runs on the stream that its calls are given (None: the
default stream), whichever it was made on; its caller orders calls on different streams.
"""
import ctypes as C
import math
from dataclasses import dataclass

from .sampler import BeamConfig, BeamPool, InvalidArgument

try:
    import torch
except Exception:  # pragma: no cover
    torch = None


@dataclass
class Head:
    """The layer that makes logits of hidden states (`Sampler.linear`)."""
    weight: "torch.Tensor"             # [vocab, hidden] bfloat16
    bias: "torch.Tensor" = None        # [vocab] float32
    activation: str = "none"
    scale: float = 1.0


_parked = []  # tables of searches that went while their stream was being captured, which cannot wait for anything


class BeamSearch:
    """One search at a time over groups * beams rows of `vocab` tokens, at most max_steps of them.

    With `history` (a capacity) the penalties of `config` go over the device-resident history of the sampler,
    which the search owns until its end; without it penalties are off."""

    def __init__(self, sampler, groups, beams, max_steps, vocab, config=None, head=None, history=0):
        self.sampler, self.groups, self.beams, self.vocab = sampler, int(groups), int(beams), int(vocab)
        self.max_steps, self.config, self.head, self.history = int(max_steps), config or BeamConfig(), head, int(history)
        if self.groups < 1 or self.beams < 1 or self.max_steps < 1:
            raise InvalidArgument("groups, beams and max_steps must be positive")
        c = self.config
        if not history and (c.repetition_penalty not in (0.0, 1.0) or c.frequency_penalty or c.presence_penalty):
            raise InvalidArgument("penalties need a history")
        if head is not None and int(head.weight.shape[0]) != self.vocab:
            raise InvalidArgument(f"head has {int(head.weight.shape[0])} features, not {self.vocab}")
        rows, dev = self.groups * self.beams, f"cuda:{sampler.device}"
        i32 = dict(dtype=torch.int32, device=dev)
        self.token_table = torch.empty((self.max_steps, rows), **i32)
        self.parent_table = torch.empty((self.max_steps, rows), **i32)
        self.scores = torch.empty(rows, dtype=torch.float32, device=dev)
        self.status = torch.empty(rows, **i32)
        self.pool = BeamPool(self.groups, self.beams, dev)  # (begin() empties it, on its own stream)
        # (held here: the kernel writes them after the step's call has returned, on whatever stream it was given)
        self.ends = {n: torch.empty((self.groups, self.beams), dtype=d, device=dev) for n, d in
                     (("end_parent", torch.int32), ("end_token", torch.int32), ("end_score", torch.float32))}
        self.logits = torch.empty((rows, self.vocab), dtype=torch.float32, device=dev) if head is not None else None
        self.steps = None
        # What the tables' memory was last used for is done on this stream at this point; begin() waits for it.
        self._home = torch.cuda.current_stream(dev)
        self._made = torch.cuda.Event()
        self._made.record(self._home)
        self._used = None  # event behind the last call on another stream
        self._at = None    # the last call's stream
        if self.history:
            sampler.history_create(self.history)

    def begin(self, prompts=None, lens=None, stream=None):
        """Start a search: one empty beam per group.  prompts [groups, n] (int32) with optional lens fill the
        histories of all its beams."""
        if self.history and prompts is not None:
            self._check_prompts(prompts, lens)
        self.steps = 0
        with self._on(stream):
            # (a capture may not wait for what is outside it: its replays come behind whatever the caller puts before them)
            if (stream or 0) != self._home.cuda_stream and not torch.cuda.is_current_stream_capturing():
                self._made.wait()
            self.scores.fill_(-math.inf)
            self.scores[::self.beams] = 0.0
        self.sampler.beam_pool_reset(self.pool, stream=stream)
        if self.history:
            with self._on(stream):
                if prompts is None:
                    prompts = torch.empty((self.groups, 0), dtype=torch.int32, device=self.scores.device)
                rows = prompts.to(self.scores.device).repeat_interleave(self.beams, 0).contiguous()
                lens = None if lens is None else lens.to(self.scores.device).repeat_interleave(self.beams).contiguous()
            self._prompts = (rows, lens)  # (kept until the copy on the stream has read them)
            self.sampler.history_reset(rows, lens, stream=stream)
        self._mark(stream)

    def _check_prompts(self, prompts, lens):
        # (their elements are read as they lie in memory)
        if prompts.ndim != 2 or int(prompts.shape[0]) != self.groups or prompts.dtype != torch.int32:
            raise InvalidArgument(f"prompts must be [{self.groups}, n] int32, not {tuple(prompts.shape)} {prompts.dtype}")
        if lens is not None and (tuple(lens.shape) != (self.groups,) or lens.dtype != torch.int32):
            raise InvalidArgument(f"lens must be [{self.groups}] int32, not {tuple(lens.shape)} {lens.dtype}")

    def _on(self, stream):
        return torch.cuda.stream(self._stream(stream))

    def _stream(self, stream):
        if self._at is None or self._at.cuda_stream != (stream or 0):
            dev = self.scores.device
            self._at = torch.cuda.ExternalStream(stream, device=dev) if stream else torch.cuda.default_stream(dev)
        return self._at

    def _mark(self, stream):
        # (the replays of a capture need the search itself)
        if (stream or 0) != self._home.cuda_stream and not torch.cuda.is_current_stream_capturing():
            self._used = self._used or torch.cuda.Event()
            self._used.record(self._stream(stream))

    def __del__(self):
        """The tables' memory goes back to the stream on which the search was made: that stream waits for the calls on others."""
        if getattr(self, "_used", None) is None:
            return
        try:
            with torch.cuda.stream(self._home):
                if torch.cuda.is_current_stream_capturing():
                    _parked.append(self.__dict__)
                else:
                    self._used.wait()
        except Exception:  # (the interpreter ends, or the device is gone)
            pass

    @property
    def tokens(self):
        """The last step's token of every row, [groups * beams] int32; -1 where no beam goes on."""
        if not self.steps:
            raise InvalidArgument("no step has been made")
        return self.token_table[self.steps - 1]

    def step(self, x, states=(), lens=None, position_dim=None, mask=None, stream=None):
        """One step: with a head the logits of hidden states x, the beams that go on, and `states` after them (see
        `Sampler.beam_reorder`; a list, or a list of lists where layouts differ).  Returns the rows' tokens."""
        if self.steps is None:
            raise InvalidArgument("begin() comes first")
        if self.steps >= self.max_steps:
            raise InvalidArgument(f"the search was made for {self.max_steps} steps")
        s, h, t = self.sampler, self.head, self.steps
        logits = x
        if h is not None:
            logits = s.linear(x, h.weight, bias=h.bias, activation=h.activation, scale=h.scale, out=self.logits, stream=stream)
        if tuple(logits.shape) != (self.groups * self.beams, self.vocab):
            raise InvalidArgument(f"logits are {tuple(logits.shape)}, not {(self.groups * self.beams, self.vocab)}")
        states = list(states)
        moves = [s.prepare_beam_reorder(part, self.parent_table[t], self.beams, lens=lens, position_dim=position_dim)
                 for part in (states if states and isinstance(states[0], (list, tuple)) else [states] if states else [])]
        make = s.beam_next if self.history else s.beam_step
        make(logits, self.scores, self.beams, config=self.config, mask=mask, pool=self.pool, step=t, stream=stream,
             out={"token": self.token_table[t], "parent": self.parent_table[t], "score": self.scores, "status": self.status,
                  **self.ends})
        self.steps = t + 1
        for move in moves:
            move.run(stream)
        self._mark(stream)
        return self.token_table[t]

    def _norm(self, length):
        try:
            return float(length) ** C.c_float(self.config.length_penalty).value
        except OverflowError:  # (infinite, as the step's is)
            return math.inf

    def result(self, stream=None):
        """The best `beams` hypotheses of every group, best first: those of the pool and, in groups that are not
        done, the beams that are still going, all by score / length ** length_penalty.  A dict of tokens [groups,
        beams, steps] padded with -1, lens and scores [groups, beams] (length 0 and -inf: none)."""
        if not self.steps:
            raise InvalidArgument("no step has been made")
        N, K, T, p = self.groups, self.beams, self.steps, self.pool
        i32 = dict(dtype=torch.int32, device=self.scores.device)
        with self._on(stream):
            going = (p.done == 0)[:, None] & (self.tokens.view(N, K) >= 0)
            # (as the pool's: in 64 bits, by a division; a Python divisor would be a multiplication by its rounded inverse)
            norm = torch.full((), self._norm(T), dtype=torch.float64, device=self.scores.device)
            score = torch.where(going, (self.scores.view(N, K).double() / norm).float(), -math.inf)
            scores, order = torch.sort(torch.cat([p.score, score], 1), dim=1, descending=True, stable=True)
            scores, order = scores[:, :K].contiguous(), order[:, :K]
            last = torch.where(going, T - 1, -1).to(torch.int32)
            ends = [torch.cat(pair, 1).gather(1, order).contiguous() for pair in
                    ((p.step, last), (p.parent, self.parent_table[T - 1].view(N, K)), (p.token, self.tokens.view(N, K)))]
            out = {"tokens": torch.empty((N, K, T), **i32), "lens": torch.empty((N, K), **i32)}
        self.sampler.beam_sequences(self.token_table[:T], self.parent_table[:T], *ends, K, out=out, stream=stream)
        self._mark(stream)
        return {"tokens": out["tokens"], "lens": out["lens"], "scores": scores}
