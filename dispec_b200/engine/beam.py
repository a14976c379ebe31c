"""Beam search: the likeliest continuations of every prompt.

A step runs one token of every beam of every prompt.  The beams of a prompt share the pages that their common tokens fill, which
the attention reads once a prompt (``ModelRunner.beam_step``); the best continuations are chosen on the device over all
beams and the vocabulary (``ops.beam_select``); beams that go on in more than one way fork, and only the page in which they
part and the recurrent states are copied (``ModelRunner.fork``).  The host reads twice as many candidates as there are beams
once a step, so that enough are left where some end.  (The reference decodes greedily, by sampling and speculatively:
puneethgv/DiSpec dispec/sampling.py, dispec/spec/speculative.py.)"""
from __future__ import annotations

import itertools
import math
from dataclasses import dataclass, field

import torch

from dispec_b200 import ops
from dispec_b200.config.engine_config import KVConfig
from dispec_b200.engine.batch import SeqEntry
from dispec_b200.engine.runner import ModelRunner


@dataclass
class Hypothesis:
    tokens: list   # new tokens, the end token among them where there is one
    score: float   # the sum of their log-probabilities over their number to the power of the length penalty


@dataclass
class Beam:
    req_id: object
    tokens: list   # new tokens
    total: float   # the sum of their log-probabilities


@dataclass
class BeamSet:
    """What the host keeps of one prompt's search."""
    width: int
    max_new_tokens: int
    length_penalty: float
    eos: int | None
    beams: list = field(default_factory=list)      # Beam, the best first
    finished: list = field(default_factory=list)   # Hypothesis, the best first, at most ``width``
    done: bool = False

    def _finish(self, tokens: list, total: float) -> None:
        self.finished.append(Hypothesis(tokens, total / len(tokens) ** self.length_penalty))
        self.finished.sort(key=lambda h: -h.score)
        del self.finished[self.width:]

    def advance(self, candidates: list) -> list:
        """Takes a step's candidates (number of the beam, token, total), the best first; returns those of them that go on.  One that
        ends among the first ``width`` is finished.  The search is done when ``width`` are finished and no beam could still
        be ranked before the worst of them were it to end now, or when the beams are as long as they may be."""
        going = []
        for rank, (parent, token, total) in enumerate(candidates):
            if token == self.eos:
                if rank < self.width:
                    self._finish(self.beams[parent].tokens + [token], total)
            else:
                going.append((parent, token, total))
                if len(going) == self.width:
                    break
        length = len(self.beams[0].tokens) + 1
        if not going:
            self.done = True
        elif length >= self.max_new_tokens:
            for parent, token, total in going:
                self._finish(self.beams[parent].tokens + [token], total)
            self.done = True
        elif len(self.finished) == self.width and going[0][2] / length ** self.length_penalty <= self.finished[-1].score:
            self.done = True
        return [] if self.done else going


class BeamSearchEngine:
    """``BeamSearchEngine(model, kv, num_blocks, beam_width).generate(prompts, max_new_tokens, length_penalty, eos_token_id,
    num_return) -> list of lists of Hypothesis``, the best first, for each prompt.  At most ``max_num_seqs`` beams run at a time;
    prompts beyond them wait."""

    _seq_counter = itertools.count()

    def __init__(self, model, kv: KVConfig | None = None, num_blocks: int | None = None, beam_width: int = 4, max_num_seqs: int = 64):
        if not 1 <= beam_width <= 128:
            raise ValueError(f"beam_width={beam_width}: 1 to 128")
        if max_num_seqs < beam_width:
            raise ValueError(f"max_num_seqs={max_num_seqs}: room for one prompt's {beam_width} beams is needed")
        kv = kv or KVConfig()
        self.runner = ModelRunner(model, page_size=kv.block_size, num_pages=kv.max_blocks if num_blocks is None else num_blocks,
                                  max_num_seqs=max_num_seqs)
        self.beam_width, self.max_num_seqs = beam_width, max_num_seqs
        self.num_steps = 0  # steps of beams

    def generate(self, prompts: list, max_new_tokens: int, length_penalty: float = 1.0, eos_token_id: int | None = None,
                 num_return: int = 1) -> list:
        if any(not len(p) for p in prompts):
            raise ValueError("a prompt needs at least one token")
        if not math.isfinite(length_penalty):
            raise ValueError(f"length_penalty={length_penalty}")
        if max_new_tokens <= 0:
            return [[] for _ in prompts]
        try:
            max_new_tokens ** abs(length_penalty)
        except OverflowError:
            raise ValueError(f"length_penalty={length_penalty}: {max_new_tokens} tokens to this power cannot be counted") from None
        at_once = self.max_num_seqs // self.beam_width
        out = []
        for i in range(0, len(prompts), at_once):
            out += self._search([list(p) for p in prompts[i:i + at_once]], max_new_tokens, length_penalty, eos_token_id)
        return [found[:max(0, num_return)] for found in out]

    def _new_id(self):
        return ("beam", next(self._seq_counter))

    def _search(self, prompts: list, max_new_tokens: int, length_penalty: float, eos) -> list:
        run = self.runner
        sets = [BeamSet(self.beam_width, max_new_tokens, length_penalty, eos) for _ in prompts]
        shared = [[0] * len(run.cache.groups) for _ in prompts]
        live = []  # requests held
        try:
            logits = []
            for s, p in zip(sets, prompts):
                s.beams = [Beam(self._new_id(), [], 0.0)]
                run.admit(s.beams[0].req_id)
                live.append(s.beams[0].req_id)
                logits.append(run.step([SeqEntry(s.beams[0].req_id, p, 0, [len(p) - 1])]))
            starts = torch.arange(len(prompts) + 1, dtype=torch.int32, device=run.device)
            self._choose(sets, torch.cat(logits), starts, live)
            while True:
                going = [i for i, s in enumerate(sets) if not s.done]
                if not going:
                    break
                groups = [[SeqEntry(b.req_id, [b.tokens[-1]], len(prompts[i]) + len(b.tokens) - 1) for b in sets[i].beams] for i in going]
                logits, starts = run.beam_step(groups, [shared[i] for i in going])
                self.num_steps += 1
                self._choose([sets[i] for i in going], logits, starts, live)
            return [s.finished for s in sets]
        finally:
            for r in live:
                run.release(r)

    def _choose(self, sets: list, logits: torch.Tensor, starts: torch.Tensor, live: list) -> None:
        """Chooses every prompt's continuations by the logits behind its beams, and forks beams that go on in several ways."""
        totals = torch.tensor([b.total for s in sets for b in s.beams], dtype=torch.float32).to(logits.device)
        got = ops.beam_select(logits, totals, starts, count=2 * self.beam_width)
        read = torch.stack([got.parent, got.token, got.score.view(torch.int32)]).cpu()  # the step's only wait
        ops.raise_on_device_error("a step of beams")
        parents, tokens = read[0].tolist(), read[1].tolist()
        scores = read[2].view(torch.float32).tolist()
        first, forks = 0, []
        for s, of_parent, of_token, of_score in zip(sets, parents, tokens, scores):
            candidates = [(p - first, t, x) for p, t, x in zip(of_parent, of_token, of_score) if p >= 0]
            first += len(s.beams)
            going = s.advance(candidates)
            beams, taken = [], set()
            for parent, token, total in going:
                old = s.beams[parent]
                # the first that goes on keeps the request
                req_id = self._new_id() if parent in taken else old.req_id
                if parent in taken:
                    forks.append((old.req_id, req_id))
                taken.add(parent)
                beams.append(Beam(req_id, old.tokens + [token], total))
            for i, b in enumerate(s.beams):
                if i not in taken:
                    self.runner.release(b.req_id)
                    live.remove(b.req_id)
            s.beams = beams
        for _, new in forks:
            live.append(new)
        try:
            self.runner.fork(forks)
        except Exception:
            live[:] = [r for r in live if self.runner.cache.has(r)]
            raise
