"""The step function: runs a batch of (request, its next tokens) from the cache and returns
the logits at the wanted places.

``ModelRunner`` owns the cache manager, the device pools and the state buffers of one model.
``step(entries)`` runs only the tokens it is given, as one flat batch (portions of prompts
beside single decoded tokens), and leaves their keys and values in the pages.  It plays the
role of ``ModelRunner.forward`` + ``ModelRunner.logits`` of the reference (puneethgv/DiSpec
dispec/engine/model_runner.py:188-231) with the bookkeeping its callers do by hand
(dispec/sched/scheduler.py:132-197) moved behind one call.
"""
from __future__ import annotations

import functools
import math

import torch

from dispec_b200 import ops
from dispec_b200.cache.manager import CacheManager
from dispec_b200.cache.storage import CacheStorage, StateStorage
from dispec_b200.engine.batch import (HostStaging, SeqEntry, SharedStep, StepPlanLayout, TreeEntry, build_context,
                                      build_tree_context)
from dispec_b200.ops import library as _library
from dispec_b200.ops.beams import ON_FMA_UNITS
from dispec_b200.models.model import DecoderModel

# Context lengths for which a captured decode step is laid out (the last class is the engine's
# own maximum): few enough that little is captured, far enough apart that a short context does
# not pay for the key sharing that a long one needs.
GRAPH_CONTEXT_CLASSES = (2048, 8192, 32768, 131072, 524288)


# Bytes of keys and values that reading shared pages once has to save in a layer: the attention of shared pages is three launches and
# one of the rotation where that of single tokens is one.  A layer of a step as the engine runs it, eagerly and read back (models of 8 to
# 14 layers, layer by layer both), shared and each its own, us: 28 heads of 128 on 4, 4 beams behind 16,384 tokens (101 MB) 160 and
# 160, 8 behind 16,384 (235 MB) 174 and 184, 32 behind 16,384 (1 GB) 272 and 380, 32 groups of 4 behind 500 (98 MB) 259 and 243, 8 of 5
# behind 4,101 (268 MB) 220 and 254; 12 on 2, 8 groups of 5 (134 MB) 169 and 159; 40 on 8, 8 behind 4,096 (117 MB) 175 and 170, 4
# behind 16,384 (201 MB) 187 and 192; 28 heads of 32 on 4, 32 behind 16,384 (260 MB) 196 and 237.  In 32 bits the attention of single
# tokens is bound by its arithmetic, and the products of shared pages are of tiles of rows: 12 on 2, 2 beams behind 64 tokens (0.1 MB) 154
# and 155, behind 256 (0.5 MB) 155 and 167, 8 behind 4,096 173 and 457.
# Where single tokens have a tensor-core kernel and shared pages the 32-bit one (bfloat16 heads other than 32, 64 and 128, pages of other
# than 8 to 64 tokens), a tile of 32 rows takes as long with five of them.  28 heads of 96 on 4 never gain, 64 beams behind 32,768
# tokens 1,931 and 1,225; one or two heads a key head do from 16 rows on: 8 of 96 on 8, 8 groups of 5 behind 4,101 (403 MB) 430 and 305, 8
# beams behind 32,768 (705 MB) 362 and 297, 16 behind 16,384 (755 MB) 279 and 305, 32 (1.6 GB) 375 and 540; 16 of 80 on 8, 32 behind 4,096
# (325 MB) 228 and 210, 16 behind 16,384 (629 MB) 275 and 294; 8 of 16 on 4, 64 behind 32,768 (528 MB) 899 and 1,115; 16 of 128 on 8, pages
# of 128 tokens, 32 behind 4,096 (520 MB) 203 and 189.  Narrower heads take longer a byte, here and below.
# (What is not listed counts as the model's type.)
SHARED_BYTES = {torch.bfloat16: 150_000_000, torch.float32: 500_000, ON_FMA_UNITS: 600_000_000}
FILLED_ROWS = 16
# A step that reads shared pages once runs layer by layer, which takes the host 105 us a layer; others of a dense decoder run behind one
# call (ops/dense_chain.py), and take as long as the device does.  So such a step has to read so many times SHARED_BYTES a layer, or the
# device waits for the host: weights, and keys and values by what a byte of them takes (1.4 times a weight's with heads of 128).  Behind one call and shared: 12 heads of 128 on 2, 8 beams behind 16,384 tokens (0.28 GB so counted) 98
# and 152, 32 behind 16,384 (0.85 GB) 214 and 206; 16 of 64 on 4, 8 behind 16,384 (0.30 GB) 99 and 153, 16 groups of 8 behind 4,101 (1.1 GB)
# 291 and 252; 28 on 4, 8 behind 16,384 (0.84 GB) 190 and 174.
CHAIN_SHARED_BYTES, KEY_BYTE = 4, 1.4


def _time_of_a_byte(dim: int) -> float:
    """Of keys and values, beside heads of 128: a fit to the figures above."""
    return math.sqrt(128 / dim)


def _least_saved(by: tuple, dtype: torch.dtype, dim: int, sequences: float) -> float:
    """Bytes that reading shared pages once has to save, for a mixer that does so "by" (``Part.takes_shared``) and so many sequences a
    group."""
    kernel, heads = by
    least = SHARED_BYTES.get(kernel, SHARED_BYTES[dtype])
    if kernel != ON_FMA_UNITS:
        return least
    return least / _time_of_a_byte(dim) * (FILLED_ROWS / min(FILLED_ROWS, heads * sequences)) ** 4


MAX_SHARED_GROUPS = 1024  # of a call (ops/beams.py)


class ModelRunner:
    def __init__(self, model: DecoderModel, page_size: int = 16, num_pages=4096,
                 max_num_seqs: int = 256, poison: bool = False, cuda_graph: bool = False,
                 max_model_len: int | None = None):
        if model.device is None:
            raise ValueError("the model has no weights yet (load it first)")
        self.model = model
        self.dtype = model.dtype
        self.device = model.device
        self.page_size = page_size
        groups = model.cache_groups
        counts = [num_pages] * len(groups) if isinstance(num_pages, int) else list(num_pages)
        self.cache = CacheManager(groups, page_size, counts, max_num_seqs)
        self.storage = CacheStorage(groups, page_size, counts, self.dtype, self.device, poison=poison)
        self.states = StateStorage(model.state_needs, max_num_seqs, self.device)
        self.staging = HostStaging(self.device)
        self.poison = poison  # tests: pages given back are filled with NaN
        self.vocab_size = model.spec.vocab_size
        self.num_steps = 0
        self.cuda_graph = (bool(cuda_graph) and self.dtype == torch.bfloat16
                           and all(getattr(p, "graph_safe", True) for p in model._parts))
        # captured decode steps, one per padded batch size; the page tables of a captured step
        # have room for the longest sequence the pools or the model allow
        # (powers of two, and the largest batch itself so that every batch has a bucket)
        self.graph_buckets = [1 << i for i in range(13) if (1 << i) < max_num_seqs]
        self.graph_buckets.append(max_num_seqs)
        # the longest request: the configuration's max_position_embeddings unless the caller says
        # otherwise (angles are computed from the position, so no table stands in the way of more)
        limit = max_model_len or model.spec.max_position or (1 << 30)
        self.max_model_len = min(limit, self.cache.capacity_tokens())
        self._group_windows = [g.window for g in groups]
        self._group_pages = list(counts)
        self._graphs: dict = {}

    # ---------------------------------------------------------------- request lifecycle
    def admit(self, req_id, prompt_len: int = 0, max_total_len: int = 0, max_chunk: int = 1) -> None:
        slot = self.cache.admit(req_id, prompt_len, max_total_len, max_chunk)
        if self.states.buffers:
            self.states.reset_slot(slot)

    def release(self, req_id) -> None:
        self._poison(self.cache.free(req_id))

    def _poison(self, released) -> None:
        if self.poison and released:
            for g in range(len(self.cache.groups)):
                self.storage.poison_pages(g, [p for gg, p in released if gg == g])

    # ----------------------------------------------------------------------- the step
    @torch.inference_mode()
    def step(self, entries: list[SeqEntry], feed_tokens: torch.Tensor | None = None) -> torch.Tensor:
        """Logits [number of wanted places, vocab] in float32, in the order of ``entries`` and
        of each entry's ``want``.  ``feed_tokens`` (int32, on the device): the tokens sampled in
        the previous step; an entry with ``feed_row`` r takes its single token from row r of it
        on the device, so the host need not have seen that token yet."""
        if not entries:
            return torch.empty((0, self.vocab_size), dtype=torch.float32, device=self.device)
        seen = set()
        for e in entries:
            if e.req_id in seen:
                raise ValueError(f"request {e.req_id!r} appears twice in one step")
            seen.add(e.req_id)
            if not self.cache.has(e.req_id):
                raise KeyError(f"request {e.req_id!r} was not admitted")
            if len(e.tokens) == 0:
                raise ValueError(f"request {e.req_id!r} brings no tokens")
            stored = self.cache.num_tokens(e.req_id)
            if e.start != stored:
                raise ValueError(f"request {e.req_id!r}: tokens start at position {e.start} but "
                                 f"{stored} tokens are stored")
        if any(e.feed_row >= 0 for e in entries) and feed_tokens is None:
            raise ValueError("an entry is fed from the previous step but feed_tokens is missing")
        for e in entries:  # may raise OutOfPagesError before anything ran
            self.cache.extend(e.req_id, e.start + len(e.tokens))
        if (self.cuda_graph and self.graph_buckets and len(entries) <= self.graph_buckets[-1]
                and all(len(e.tokens) == 1 for e in entries)):
            return self._graph_step(entries, feed_tokens)
        ctx, _ = build_context(entries, self.cache, self.storage, self.states, self.staging,
                               self.dtype, self.device, self.model.attention_tile_tokens,
                               self.vocab_size)
        if ctx.num_fed:
            ops.feed_tokens(ctx.token_ids, ctx.feed_src, feed_tokens)
        x, pending = self.model.forward(ctx)
        n_rows = ctx.logit_rows.shape[0]
        if n_rows:
            logits = self.model.logits(ctx, x, pending, ctx.logit_rows)
        else:
            logits = torch.empty((0, self.vocab_size), dtype=torch.float32, device=self.device)
        for e in entries:
            self._poison(self.cache.commit(e.req_id, e.start + len(e.tokens)))
        self.num_steps += 1
        return logits

    # ------------------------------------------------------------------ drafted trees
    @torch.inference_mode()
    def tree_step(self, entries: list[TreeEntry]):
        """One pass over the requests' drafted trees: the context of the step and the logits behind every node, in
        float32, tree after tree.  The nodes' keys and values lie behind the stored tokens; nothing is stored for
        good until ``keep`` has been told which branch was accepted."""
        if not all(self.model.layers[c.layer].mixer.takes_trees for c in self.model.schedule):
            raise ValueError("this model has layers that cannot be run on drafted trees")
        if not entries or len({e.req_id for e in entries}) != len(entries):
            raise ValueError("a step of drafted trees needs requests, each of them once")
        for e in entries:
            if not self.cache.has(e.req_id):
                raise KeyError(f"request {e.req_id!r} was not admitted")
            if not e.tokens or len(e.tokens) != len(e.parents):
                raise ValueError(f"request {e.req_id!r}: {len(e.tokens)} nodes with {len(e.parents)} parents")
            if e.start != self.cache.num_tokens(e.req_id):
                raise ValueError(f"request {e.req_id!r}: the tree starts at position {e.start} but "
                                 f"{self.cache.num_tokens(e.req_id)} tokens are stored")
        for e in entries:  # may raise OutOfPagesError before anything ran
            self.cache.extend(e.req_id, e.start + len(e.tokens))
        ctx = build_tree_context(entries, self.cache, self.storage, self.staging, self.dtype, self.device, self.vocab_size)
        x, pending = self.model.forward(ctx)
        logits = self.model.logits(ctx, x, pending, ctx.logit_rows)
        self.num_steps += 1
        return ctx, logits

    @torch.inference_mode()
    def move_accepted(self, ctx, verified) -> None:
        """Puts the accepted branches' keys and values into line behind the stored tokens, on the device."""
        for g, named in enumerate(self.storage.pools):
            ops.keep_path(list(named.values()), ctx.page_tables[g], ctx.tree.ctx_len, verified.path, verified.count)

    def keep(self, entries: list[TreeEntry], counts: list) -> None:
        """Records that so many tokens of each tree's accepted branch are stored, once they are in line."""
        for e, n in zip(entries, counts):
            if not 1 <= n <= len(e.tokens):
                raise ValueError(f"request {e.req_id!r}: {n} accepted nodes of {len(e.tokens)}")
            self._poison(self.cache.commit(e.req_id, e.start + n))

    # ------------------------------------------------------------------------- beams
    @torch.inference_mode()
    def beam_step(self, groups: list[list[SeqEntry]], shared: list[list[int]]):
        """One token for every sequence of every group: the logits behind them in float32, group after group, and the first
        sequence of each group on the device ([groups + 1] int32).  ``shared``: per group and cache group, so many first pages
        are known to be the same for the group's sequences; counted on in place.  They are read once a group by mixers that
        can (``takes_shared``)."""
        entries = [e for of in groups for e in of]
        if not entries or not all(groups) or len({e.req_id for e in entries}) != len(entries):
            raise ValueError("a step of beams needs groups of requests, each of them once")
        for e in entries:
            if not self.cache.has(e.req_id):
                raise KeyError(f"request {e.req_id!r} was not admitted")
            if len(e.tokens) != 1:
                raise ValueError(f"request {e.req_id!r}: a step of beams takes one token each")
            if e.start != self.cache.num_tokens(e.req_id):
                raise ValueError(f"request {e.req_id!r}: its token is at position {e.start} but {self.cache.num_tokens(e.req_id)} "
                                 "tokens are stored")
        for e in entries:  # may raise OutOfPagesError before anything ran
            self.cache.extend(e.req_id, e.start + 1)
        ctx, _ = build_context([SeqEntry(e.req_id, e.tokens, e.start, [0]) for e in entries], self.cache, self.storage, self.states,
                               self.staging, self.dtype, self.device, self.model.attention_tile_tokens, self.vocab_size)
        n, starts, prefixes, worth, reads = len(groups), [0], [], [], []
        for of in groups:
            starts.append(starts[-1] + len(of))
        for c, spec in enumerate(self.cache.groups):
            saved = seen = 0  # tokens that need not be read, and that are seen
            for of, known in zip(groups, shared):
                if len(of) > 1:
                    known[c] = self.cache.shared_pages([e.req_id for e in of], c, known[c])
                prefixes.append(known[c] * self.page_size if len(of) > 1 else 0)
                of_window = prefixes[-1] if spec.window <= 0 else max(0, min(prefixes[-1], prefixes[-1] + spec.window - of[0].start - 1))
                saved += (len(of) - 1) * of_window
                seen += sum(e.start + 1 if spec.window <= 0 else min(e.start + 1, spec.window) for e in of)
            token = sum(t.num_heads * t.width for t in spec.tensors) * self.dtype.itemsize
            dim = max(t.width for t in spec.tensors)
            reads.append(spec.num_slots * seen * token * _time_of_a_byte(dim))
            least = max((_least_saved(by, self.dtype, dim, len(entries) / n) for by in self._shared_by[c]), default=math.inf)
            worth.append(n <= MAX_SHARED_GROUPS and saved * token >= least)
        if self.model.dense_chain:
            a_layer = self._layer_bytes() + KEY_BYTE * sum(reads) / sum(spec.num_slots for spec in self.cache.groups)
            if a_layer < CHAIN_SHARED_BYTES * SHARED_BYTES[self.dtype]:
                worth = [False] * len(worth)
        numbers = torch.tensor(starts + prefixes, dtype=torch.int32).to(self.device)
        if any(worth):
            ctx.shared = SharedStep(numbers[:n + 1], [numbers[n + 1 + c * n:n + 1 + (c + 1) * n] if w else None for c, w in enumerate(worth)])
        x, pending = self.model.forward(ctx)
        logits = self.model.logits(ctx, x, pending, ctx.logit_rows)
        for e in entries:
            self._poison(self.cache.commit(e.req_id, e.start + 1))
        self.num_steps += 1
        return logits, numbers[:n + 1]

    @functools.cached_property
    def _shared_by(self) -> list:
        """Per cache group: how its mixers read pages that sequences share."""
        of = [set() for _ in self.cache.groups]
        for call, label in zip(self.model.schedule, self.model.call_cache):
            takes = getattr(self.model.layers[call.layer].mixer, "takes_shared", None)  # (a mixer need not know of it)
            by = takes(self.page_size, self.dtype) if takes is not None and label is not None else None
            if by is not None:
                of[self.model.placement[label].group].add(by)
        return of

    def _layer_bytes(self) -> int:
        """Weights of a layer of a dense decoder."""
        block = self.model.layers[self.model.schedule[0].layer]
        return sum(w.numel() * w.element_size() for w in (block.mixer.w_qkv, block.mixer.w_o, block.feed_forward.w_gate_up,
                                                          block.feed_forward.w_down))

    @torch.inference_mode()
    def fork(self, pairs: list) -> None:
        """For each (request, new one): the new one goes on from where the request is, with pages in common and a copy of the
        page that both will write to and of the states.  Where one cannot, none is there."""
        pages = [[] for _ in self.cache.groups]
        slots, there, origin = [], [], {}
        for req_id, new_id in pairs:
            try:
                slot, copies = self.cache.fork(req_id, new_id)
            except Exception:
                for r in there:
                    self.release(r)
                raise
            there.append(new_id)
            # (what is itself new here is copied from where it comes from: all is read before anything is written)
            old = self.cache.state_slot(req_id)
            origin[slot] = origin.get(old, old)
            slots.append((slot, origin[slot]))
            for g, page, copy in copies:
                origin[g, copy] = origin.get((g, page), page)
                pages[g].append((copy, origin[g, copy]))
        for named, moves in zip(self.storage.pools, pages):
            self._copy_slots(list(named.values()), moves)
        self._copy_slots([b.view(1, b.shape[0], -1) for b in self.states.buffers], slots)

    def _copy_slots(self, pools: list, moves: list) -> None:
        """(destination, source) pairs, in pools [layers, slots, ...]."""
        if not pools or not moves:
            return
        moves = sorted(moves)
        numbers = torch.tensor([d for d, _ in moves] + [s for _, s in moves], dtype=torch.int32).to(self.device)
        dst, src = numbers[:len(moves)], numbers[len(moves):]
        for i in range(0, len(pools), 64):
            for k in range(0, len(moves), 8192):  # (copies are new: none of them is read)
                ops.reorder_slots(pools[i:i + 64], src[k:k + 8192], dst[k:k + 8192])

    # -------------------------------------------------------- captured all-decode steps
    def _context_class(self, entries: list) -> int:
        """The context length a captured step is laid out for: the smallest class that holds the
        step's longest request.  How the keys of a row are shared among CTAs is decided on the
        host from this bound, so a graph serves one class."""
        longest = max(e.start + len(e.tokens) for e in entries)
        for bound in GRAPH_CONTEXT_CLASSES:
            if longest <= bound < self.max_model_len:
                return bound
        # beyond the listed classes (a model whose groups all have windows has no longest request of
        # its own): powers of two, so that the page tables of a captured step stay near the context
        bound = GRAPH_CONTEXT_CLASSES[-1]
        while bound < longest:
            bound *= 2
        return min(bound, self.max_model_len)

    def _graph_pages(self, ctx_bound: int) -> list:
        """Page-table width per group of a step captured for contexts up to ``ctx_bound``: a full
        group never holds more pages than its pool has; a window group's table is indexed by
        logical page (holes behind the window), so its length follows the context, not the pool."""
        longest = max(1, -(-min(ctx_bound, self.max_model_len) // self.page_size))
        return [longest if w > 0 else max(1, min(c, longest))
                for w, c in zip(self._group_windows, self._group_pages)]

    def _capture(self, bucket: int, ctx_bound: int) -> dict:
        """Captures one decode step of ``bucket`` single-token rows, none longer than
        ``ctx_bound``, as a CUDA graph.  Every
        integer input lives in one device buffer of fixed address and layout; a replay copies
        the step's values there first.  Rows beyond the live requests carry position -1 and
        length 0, which the kernels skip."""
        plan = StepPlanLayout([], self.cache, self.model.attention_tile_tokens, self.vocab_size,
                              pad_seqs=bucket, fixed_pages=self._graph_pages(ctx_bound))
        buffer = torch.empty(plan.total, dtype=torch.int32, device=self.device)
        self.staging.upload(plan.total, plan.fill, into=buffer)
        ctx = plan.context(buffer, self.storage, self.states, self.dtype, self.device)
        ctx.max_ctx_len = ctx_bound  # choices made on the host must not vary per step
        ctx.graph_capture = True

        def run():
            x, pending = self.model.forward(ctx)
            return self.model.logits(ctx, x, pending, ctx.logit_rows)

        side = torch.cuda.Stream(device=self.device)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                run()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        before = _library.LaunchCounter.n
        with torch.cuda.graph(graph):
            logits = run()
        entry = dict(graph=graph, buffer=buffer, total=plan.total, logits=logits,
                     launches=_library.LaunchCounter.n - before)
        self._graphs[(bucket, ctx_bound)] = entry
        return entry

    def _graph_step(self, entries: list, feed_tokens=None) -> torch.Tensor:
        bucket = next(b for b in self.graph_buckets if b >= len(entries))
        ctx_bound = self._context_class(entries)
        g = self._graphs.get((bucket, ctx_bound)) or self._capture(bucket, ctx_bound)
        plan = StepPlanLayout(entries, self.cache, self.model.attention_tile_tokens, self.vocab_size,
                              pad_seqs=bucket, fixed_pages=self._graph_pages(ctx_bound))
        assert plan.total == g["total"]
        self.staging.upload(plan.total, plan.fill, into=g["buffer"])
        if plan.num_fed:
            (o_ids, n_ids), (o_src, n_src) = plan.layout["token_ids"], plan.layout["feed_src"]
            ops.feed_tokens(g["buffer"][o_ids:o_ids + n_ids], g["buffer"][o_src:o_src + n_src], feed_tokens)
        g["graph"].replay()
        _library.LaunchCounter.n += g["launches"]
        for e in entries:
            self._poison(self.cache.commit(e.req_id, e.start + len(e.tokens)))
        self.num_steps += 1
        # rows of the padded batch follow the sorted (= given) order of the single-token entries
        wanted = [i for i, e in enumerate(entries) if e.want]
        logits = g["logits"][:len(entries)]
        if len(wanted) != len(entries):
            logits = logits[torch.tensor(wanted, dtype=torch.long, device=self.device)]
        return logits

    def check_device(self, where: str = "step") -> None:
        """Raises if a kernel recorded a bad page or token id (synchronises)."""
        ops.raise_on_device_error(where)
