"""Speculative decoding: several drafted tokens a request are checked in one pass of the model.

A step takes one tree of drafts per request.  The model runs once over all nodes (``ModelRunner.tree_step``), the drafts
are accepted against its distributions (``ops.verify_tree``), and the accepted branch's keys and values are put into
line in the cache (``ops.keep_path``); the host reads the accepted nodes and the drawn token once a step.  A request
gets at least one token a step, and the tokens are distributed as if they had been sampled one by one; at temperature 0
they are the same.  Drafts come from a ``draft(tokens, max_nodes)`` function; the one here looks the last tokens up in
what the request has already seen.  (The reference drafts a chain with a second model and truncates the cache behind a
refused draft: puneethgv/DiSpec dispec/spec/speculative.py, dispec/spec/rejection.py.)"""
from __future__ import annotations

import itertools
from dataclasses import dataclass, field

import torch

from dispec_b200 import ops
from dispec_b200.config.engine_config import KVConfig
from dispec_b200.engine.batch import SeqEntry, TreeEntry
from dispec_b200.engine.runner import ModelRunner
from dispec_b200.sampling.sampler import _BELOW_ONE, Sampler, SamplingParams, make_rng


def look_up(tokens: list, max_nodes: int, longest: int = 3, branches: int = 3) -> tuple[list, list]:
    """Drafts by looking the last tokens up: (tokens, parents) of a tree whose node 0 is the last token.  What followed
    earlier occurrences of the last ``longest`` tokens (then of fewer) is drafted, the latest occurrences
    first, at most ``branches`` of them, each once however many of the last tokens it shares; continuations that begin
    alike share their nodes."""
    nodes, parents = [tokens[-1]], [-1]
    children: list[dict] = [{}]
    found = set()  # places in ``tokens`` where a continuation begins
    for n in range(min(longest, len(tokens) - 1), 0, -1):
        tail = tokens[-n:]
        for at in range(len(tokens) - n - 1, -1, -1):
            if len(found) >= branches or len(nodes) >= max_nodes:
                return nodes, parents
            if tokens[at:at + n] != tail or at + n in found:
                continue
            found.add(at + n)
            node = 0
            for t in tokens[at + n:at + n + max(1, (max_nodes - 1) // branches)]:
                nxt = children[node].get(t)
                if nxt is None:
                    if len(nodes) >= max_nodes:
                        break
                    nxt = len(nodes)
                    nodes.append(t)
                    parents.append(node)
                    children.append({})
                    children[node][t] = nxt
                node = nxt
    return nodes, parents


@dataclass
class _Request:
    req_id: object
    tokens: list  # prompt and output
    prompt_len: int
    params: SamplingParams
    rng: object
    out: list = field(default_factory=list)
    done: bool = False


class SpeculativeEngine:
    """``SpeculativeEngine(model, kv, num_blocks, max_nodes).generate(prompts, max_new_tokens, params, eos_token_id) ->
    list of token lists``.  ``params``: one ``SamplingParams`` for all or one per prompt (temperature and seed; top-k
    and top-p are refused)."""

    _seq_counter = itertools.count()

    def __init__(self, model, kv: KVConfig | None = None, num_blocks: int | None = None, max_nodes: int = 16,
                 max_num_seqs: int = 64, draft=look_up):
        if max_nodes < 1:
            raise ValueError(f"max_nodes={max_nodes}: a tree has at least its root")
        kv = kv or KVConfig()
        self.runner = ModelRunner(model, page_size=kv.block_size, num_pages=kv.max_blocks if num_blocks is None else num_blocks,
                                  max_num_seqs=max_num_seqs)
        self.sampler = Sampler(model.device)
        self.max_nodes, self.draft = max_nodes, draft
        self.num_steps = self.num_accepted = 0  # steps over trees; tokens that they gave

    def generate(self, prompts: list, max_new_tokens: int, params=None, eos_token_id: int | None = None) -> list:
        params = params if isinstance(params, (list, tuple)) else [params or SamplingParams()] * len(prompts)
        if len(params) != len(prompts):
            raise ValueError(f"{len(prompts)} prompts with {len(params)} sampling parameters")
        for p in params:
            if p.top_k or p.top_p < 1.0:
                raise ValueError("speculative decoding verifies against the whole distribution: top-k and top-p are not supported")
        if any(not len(p) for p in prompts):
            raise ValueError("a request needs at least one prompt token")
        requests = [_Request(("spec", next(self._seq_counter)), list(p), len(p), q, make_rng(q)) for p, q in zip(prompts, params)]
        admitted = []
        try:
            for r in requests:
                self.runner.admit(r.req_id)
                admitted.append(r)
            for r in requests:
                if max_new_tokens <= 0:
                    r.done = True
                    continue
                logits = self.runner.step([SeqEntry(r.req_id, r.tokens, 0, [r.prompt_len - 1])])
                self._take(r, self.sampler.sample(logits, [r.params], [r.rng]), max_new_tokens, eos_token_id)
            while True:
                live = [r for r in requests if not r.done]
                if not live:
                    break
                self._step(live, max_new_tokens, eos_token_id)
            return [r.out for r in requests]
        finally:
            for r in admitted:
                self.runner.release(r.req_id)

    def _take(self, r: _Request, tokens: list, max_new_tokens: int, eos) -> None:
        for t in tokens:
            if r.done:
                return
            r.tokens.append(t)
            r.out.append(t)
            r.done = len(r.out) >= max_new_tokens or t == eos

    def _step(self, live: list, max_new_tokens: int, eos) -> None:
        entries, uniforms = [], []
        for r in live:
            # (no more drafts than the request may still emit beside the drawn token)
            nodes, parents = self.draft(r.tokens, max(1, min(self.max_nodes, max_new_tokens - len(r.out))))
            if not nodes or nodes[0] != r.tokens[-1]:
                raise ValueError(f"a draft begins with {nodes[:1]}, not with the request's last token {r.tokens[-1]}")
            entries.append(TreeEntry(r.req_id, nodes, parents, len(r.tokens) - 1))
            uniforms += [min(r.rng.random(), _BELOW_ONE) for _ in nodes]
        draws = [min(r.rng.random(), _BELOW_ONE) for r in live]
        ctx, logits = self.runner.tree_step(entries)
        numbers = torch.tensor([r.params.temperature for r in live] + draws + uniforms, dtype=torch.float32).to(logits.device)
        S, tree = len(live), ctx.tree
        got = ops.verify_tree(logits, ctx.token_ids, tree.parents, tree.node_start, numbers[:S], numbers[2 * S:],
                              numbers[S:2 * S], max_nodes=tree.max_nodes)
        self.runner.move_accepted(ctx, got)
        read = torch.cat([got.count[:, None], got.token[:, None], got.path], dim=1).tolist()  # the step's only wait
        ops.raise_on_device_error("a step of drafted trees")
        self.runner.keep(entries, [row[0] for row in read])
        self.num_steps += 1
        for r, e, (count, token, *path) in zip(live, entries, read):
            before = len(r.out)
            self._take(r, [e.tokens[i] for i in path[1:count]] + [token], max_new_tokens, eos)
            self.num_accepted += len(r.out) - before
