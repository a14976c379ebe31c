"""Drafted trees over the paged cache: what a step of speculative decoding adds to a step of the engine.

Three operators, timed one call at a time:

``attention``  the nodes of one tree of drafted tokens per request attend to the request's cache and to
               their own ancestors (``ops.tree_attention``);
``verify``     the walk from a tree's root along accepted drafts, and the token drawn where it ends
               (``ops.verify_tree``);
``keep``       the accepted branch's keys and values moved into line in the cache (``ops.keep_path``).

Node 0 of a tree is the token that the previous step drew; every other node's parent comes before it.
Head counts, head sizes, layers, vocabularies and pages of 16 tokens are those of the Qwen2.5 sizes
that ``bench.py`` runs and of the tiny configurations of the tests.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda:0"
SPREAD, RAISE = 2.0, 14.0  # logits: their standard deviation, and what a raised one is raised by
MASS_ONE = 2.0 ** 40  # the mass of the likeliest token: distributions are held in whole numbers
CAP = {"bytes": 9e8, "flops": 2.0e11}  # no drawn attention costs more than the largest listed one


def listed():
    return [
        # one user, a short conversation, a small tree: the time of a launch counts
        dict(name="attention one tree", op="attention", seqs=1, nodes=8, ctx=1000, heads=12, kv_heads=2, dim=128, window=0,
             dtype="bfloat16", page=16, pages="runs", shape="tree"),
        # a small server: eight ragged requests
        dict(name="attention 8 trees", op="attention", seqs=8, nodes=16, ctx=4101, heads=28, kv_heads=4, dim=128, window=0,
             dtype="bfloat16", page=16, pages="runs", shape="tree"),
        # long documents on pages in no order
        dict(name="attention long context", op="attention", seqs=2, nodes=24, ctx=32768, heads=28, kv_heads=4, dim=128,
             window=0, dtype="bfloat16", page=16, pages="scattered", shape="tree"),
        # a full server with wide trees: 320 query rows a key/value head
        dict(name="attention 64 wide trees", op="attention", seqs=64, nodes=64, ctx=2050, heads=40, kv_heads=8, dim=128,
             window=0, dtype="bfloat16", page=16, pages="runs", shape="tree"),
        # the 32-bit path, a chain of drafts
        dict(name="attention float32", op="attention", seqs=4, nodes=7, ctx=701, heads=12, kv_heads=2, dim=128, window=0,
             dtype="float32", page=16, pages="scattered", shape="chain"),
        # layers with a sliding window, smaller heads
        dict(name="attention window", op="attention", seqs=16, nodes=13, ctx=3001, heads=16, kv_heads=4, dim=64, window=1024,
             dtype="bfloat16", page=16, pages="runs", shape="tree"),
        # one user, drafts looked up in the prompt (certain drafts, no probabilities)
        dict(name="verify one chain", op="verify", seqs=1, nodes=6, vocab=151936, drafted=False, temperature=0.8, accept=0.7,
             shape="chain"),
        # a small server, drafts drawn from a draft model's distribution
        dict(name="verify 8 drawn trees", op="verify", seqs=8, nodes=16, vocab=152064, drafted=True, temperature=1.0, accept=0.6,
             shape="tree"),
        # a full server, some requests greedy
        dict(name="verify 64 trees", op="verify", seqs=64, nodes=64, vocab=151936, drafted=False, temperature=0.7, accept=0.6,
             shape="tree"),
        # tiny model, 32-bit cache, pages of 8
        dict(name="keep tiny", op="keep", seqs=4, nodes=9, ctx=40, layers=3, kv_heads=1, dim=32, dtype="float32", page=8,
             shape="tree"),
        dict(name="keep 8 trees", op="keep", seqs=8, nodes=16, ctx=333, layers=28, kv_heads=4, dim=128, dtype="bfloat16",
             page=16, shape="tree"),
        dict(name="keep 64 wide trees", op="keep", seqs=64, nodes=64, ctx=97, layers=48, kv_heads=8, dim=128, dtype="bfloat16",
             page=16, shape="tree"),
    ]


def _log(rng, low, high):
    return int(round(low * (high / low) ** rng.random()))


def draw(rng):
    op = rng.choice(["attention", "attention", "verify", "keep"])
    shape = rng.choice(["tree", "tree", "chain"])
    while True:
        if op == "attention":
            heads, kv_heads = rng.choice([(12, 2), (28, 4), (40, 8), (16, 4), (3, 1), (8, 8)])
            case = dict(op=op, seqs=_log(rng, 1, 64), nodes=_log(rng, 1, 64), ctx=_log(rng, 1, 32768), heads=heads,
                        kv_heads=kv_heads, dim=rng.choice([128, 128, 64, 32]), window=rng.choice([0, 0, 0, _log(rng, 16, 4096)]),
                        dtype=rng.choice(["bfloat16"] * 5 + ["float32"]), page=rng.choice([16, 16, 8, 32]),
                        pages=rng.choice(["runs", "scattered"]), shape=shape)
            padded = case["seqs"] * (case["ctx"] + case["nodes"])
            w = work(case)
            if case["dtype"] == "float32" and w["flops"] > CAP["flops"] / 32:
                continue
            if (w["bytes"] <= CAP["bytes"] and w["flops"] <= CAP["flops"] and padded * kv_heads * case["dim"] <= 2e8
                    and padded * case["nodes"] * heads <= 4e8):
                return case
        elif op == "verify":
            case = dict(op=op, seqs=_log(rng, 1, 64), nodes=_log(rng, 2, 64), vocab=_log(rng, 200, 152064),
                        drafted=rng.random() < 0.5, temperature=rng.choice([0.0, 0.6, 1.0, 1.3]),
                        accept=rng.choice([0.3, 0.6, 0.8]), shape=shape)
            if case["seqs"] * case["nodes"] * case["vocab"] <= (3.2e8 if case["drafted"] else 6.3e8):
                return case
        else:
            case = dict(op=op, seqs=_log(rng, 1, 64), nodes=_log(rng, 5, 64), ctx=_log(rng, 1, 400), layers=_log(rng, 2, 48),
                        kv_heads=rng.choice([1, 2, 4, 8]), dim=rng.choice([128, 64, 32]),
                        dtype=rng.choice(["bfloat16", "bfloat16", "float32"]), page=rng.choice([16, 8, 32]), shape="tree")
            if case["seqs"] * (case["ctx"] + 2 * case["nodes"]) * case["layers"] * case["kv_heads"] * case["dim"] <= 5e8:
                return case


# ------------------------------------------------------------------------------------------ sizes
def _lengths(case):
    """Stored tokens of every request: between half of ``ctx`` and all of it, odd ones among them."""
    s = case["seqs"]
    return [max(0, case["ctx"] - (i * case["ctx"]) // (2 * s) - (i % 5 if case["ctx"] > 64 else 0)) for i in range(s)]


def _counts(case):
    """Nodes of every tree, the root among them."""
    return [max(1, case["nodes"] - i % 3) for i in range(case["seqs"])]


def _parents(case, rng):
    """Parents inside each tree (-1: the root)."""
    trees = []
    for n in _counts(case):
        if case["shape"] == "chain":
            trees.append([i - 1 for i in range(n)])
        else:
            trees.append([-1] + [rng.randint(max(0, (i - 1) // 2 - 2), max(0, min(i - 1, i // 2 + 1))) for i in range(1, n)])
    return trees


def _depths(parents):
    depths = []
    for p in parents:
        depths.append(0 if p < 0 else depths[p] + 1)
    return depths


def _visible(parents):
    """Bit j of node i: node j is i or one of its ancestors."""
    bits = []
    for i, p in enumerate(parents):
        bits.append((bits[p] if p >= 0 else 0) | 1 << i)
    return bits


def _rows_visited(case):
    """Expected nodes of a walk: a node's raised token is one of its children's with probability ``accept``, and the
    target draws the raised token with about this probability (see ``_prepare_verify``)."""
    t = case["temperature"]
    p = case["accept"]
    if t > 0:
        p /= 1.0 + case["vocab"] * math.exp(0.5 * (SPREAD / t) ** 2 - RAISE / t)
    depth = max(max(_depths(tree)) for tree in _parents(case, random.Random(1)))
    return sum(p ** k for k in range(depth + 1))


def work(case):
    size = 2 if case.get("dtype") == "bfloat16" else 4
    if case["op"] == "attention":
        w = case["window"]
        seen = [min(c, w) if w else c for c in _lengths(case)]
        nodes = _counts(case)
        kv = sum(c + n for c, n in zip(seen, nodes)) * case["kv_heads"] * case["dim"] * 2 * size
        rows = sum(nodes) * case["heads"] * case["dim"] * 2 * size
        return {"bytes": kv + rows, "flops": 4 * case["heads"] * case["dim"] * sum((c + 1) * n for c, n in zip(seen, nodes))}
    if case["op"] == "verify":  # the rows of the nodes on the walk, and of draft probabilities the last one's
        rows = case["seqs"] * (_rows_visited(case) + case["drafted"])
        return {"bytes": rows * case["vocab"] * 4, "flops": rows * case["vocab"] * 4}
    moved = sum(1 for t in _parents(case, random.Random(1)) for j, i in enumerate(_path(t)[:-1]) if i != j)
    return {"bytes": 2 * 2 * moved * case["layers"] * case["kv_heads"] * case["dim"] * size, "flops": 1}


def _path(parents):
    """The nodes from the root to the last node."""
    path, i = [], len(parents) - 1
    while i >= 0:
        path.append(i)
        i = parents[i]
    return path[::-1]


# ----------------------------------------------------------------------------------------- inputs
def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _page_table(case, rng):
    """Pages of every request: one after the other, or in no order; entries behind a window are -1."""
    page, w = case["page"], case.get("window", 0)
    need = [-(-(c + n) // page) for c, n in zip(_lengths(case), _counts(case))]
    ids = list(range(sum(need) + 1))
    if case.get("pages", "scattered") == "scattered":
        rng.shuffle(ids)
    table, at = [], 0
    for n, c in zip(need, _lengths(case)):
        row = ids[at:at + n]
        at += n
        if w:
            for j in range(min(n, max(0, c - w + 1) // page)):
                row[j] = -1
        table.append(row + [-1] * (max(need) - n))
    return _i32(table), sum(need) + 1


def prepare(case, seed):
    rng = random.Random(seed)
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    counts = _counts(case)
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    trees = _parents(case, rng)
    state = dict(case=dict(case), node_start=_i32(starts), max_nodes=max(counts))
    if case["op"] == "verify":
        return _prepare_verify(case, state, trees, starts, rng, gen)
    dtype = getattr(torch, case["dtype"])
    state["page_table"], pages = _page_table(case, rng)
    state["ctx_len"] = _i32(_lengths(case))
    normal = lambda *shape: torch.empty(shape, dtype=dtype, device=DEVICE).normal_(generator=gen)
    if case["op"] == "keep":
        paths = [_path(t) for t in _parents(case, random.Random(1))]
        shape = (case["layers"], pages, case["kv_heads"], case["page"], case["dim"])
        state.update(k=normal(*shape), v=normal(*shape), count=_i32([max(1, len(p) - 1) for p in paths]),
                     path=_i32([(p + [-1] * state["max_nodes"])[:state["max_nodes"]] for p in paths]))
        return state
    words = -(-state["max_nodes"] // 64)
    bits = [[(v >> (64 * k)) & (2 ** 64 - 1) for k in range(words)] for t in trees for v in _visible(t)]
    signed = [[b - 2 ** 64 if b >= 2 ** 63 else b for b in row] for row in bits]
    rows = starts[-1]
    width = (case["heads"] + 2 * case["kv_heads"]) * case["dim"]
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    qkv = normal(rows, width)  # the rows of the fused projection: the queries come first
    state.update(q=qkv[:, :case["heads"] * case["dim"]], k=normal(*shape), v=normal(*shape), scale=1.5 * case["dim"] ** -0.5,
                 visible=torch.tensor(signed, dtype=torch.int64, device=DEVICE),
                 depth=_i32([d for t in trees for d in _depths(t)]))
    return state


def _prepare_verify(case, state, trees, starts, rng, gen):
    """Logits of a language model's spread, one raised token per node: one of the node's children's (the better the
    draft, the more often), or another."""
    s, rows, vocab = case["seqs"], starts[-1], case["vocab"]
    tokens = [rng.randrange(vocab) for _ in range(rows)]
    raised = []
    for tree, first in zip(trees, starts):
        children = [[] for _ in tree]
        for i, p in enumerate(tree):
            if p >= 0:
                children[p].append(i)
        for i in range(len(tree)):
            good = children[i] and rng.random() < case["accept"]
            raised.append(tokens[first + rng.choice(children[i])] if good else rng.randrange(vocab))
    at, top = torch.arange(rows, device=DEVICE), torch.tensor(raised, device=DEVICE)
    logits = torch.empty((rows, vocab), dtype=torch.float32, device=DEVICE).normal_(generator=gen).mul_(SPREAD)
    logits[at, top] += RAISE
    greedy = [case["temperature"] <= 0 or (s > 1 and i % 7 == 6) for i in range(s)]
    uniform = lambda n: torch.rand(n, dtype=torch.float32, device=DEVICE, generator=gen)
    state.update(logits=logits, tokens=_i32(tokens), parents=_i32([p for t in trees for p in t]), uniforms=uniform(rows),
                 draws=uniform(s), draft_probs=None,
                 temperature=torch.tensor([0.0 if g else case["temperature"] for g in greedy], device=DEVICE))
    if case["drafted"]:  # a draft model: the same distribution, more or less
        probs = torch.empty((rows, vocab), dtype=torch.float32, device=DEVICE).normal_(generator=gen).add_(logits, alpha=0.9)
        near = torch.tensor([[t] for t in tokens], device=DEVICE)
        parent_row = torch.tensor([f + max(p, 0) for f, t in zip(starts, trees) for p in t], device=DEVICE)
        probs[parent_row, near[:, 0]] += 6.0
        probs = torch.exp_(probs.sub_(probs.amax(1, keepdim=True)))
        state["draft_probs"] = probs.div_(probs.sum(1, keepdim=True))
    return state


# ----------------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if own:
        from dispec_b200 import ops

        if case["op"] == "attention":
            return ops.tree_attention(state["q"], state["k"], state["v"], state["page_table"], state["ctx_len"],
                                      state["node_start"], state["visible"], state["depth"], max_nodes=state["max_nodes"],
                                      scale=state["scale"], window=case["window"])
        if case["op"] == "verify":
            got = ops.verify_tree(state["logits"], state["tokens"], state["parents"], state["node_start"], state["temperature"],
                                  state["uniforms"], state["draws"], draft_probs=state["draft_probs"],
                                  max_nodes=state["max_nodes"])
            return {"count": got.count, "path": got.path, "token": got.token}
        ops.keep_path([state["k"], state["v"]], state["page_table"], state["ctx_len"], state["path"], state["count"])
        return {"key": state["k"], "value": state["v"]}
    return {"attention": _plain_attention, "verify": _plain_verify, "keep": _plain_keep}[case["op"]](state)


def _tree_rows(state):
    """Flat row of node i of tree s (a tree's last row where it has fewer), and which of them there are."""
    first, last = state["node_start"][:-1, None].long(), state["node_start"][1:, None].long()
    rows = first + torch.arange(state["max_nodes"], device=DEVICE)
    return torch.minimum(rows, last - 1), rows < last


def _plain_attention(state):
    case = state["case"]
    kv_heads, dim, page, w = case["kv_heads"], case["dim"], case["page"], case["window"]
    group, n = case["heads"] // kv_heads, state["max_nodes"]
    ctx = state["ctx_len"].long()[:, None]
    rows, there = _tree_rows(state)
    seqs, longest = ctx.shape[0], state["page_table"].shape[1] * page
    at = torch.arange(longest, device=DEVICE)
    pages = state["page_table"].long().clamp_min(0)[:, at // page]
    keys = state["k"][pages, :, at % page].float()  # [S, L, KVH, D]
    values = state["v"][pages, :, at % page].float()
    # which keys a node sees: stored ones, and of the tree those whose bit is set
    depth = state["depth"].long()[rows]  # [S, N]
    bit = at[None] - ctx  # [S, L]: a key's place in the tree
    in_tree = (bit >= 0) & (bit < there.sum(1, keepdim=True))
    place = torch.where(in_tree, bit, 0)
    words = state["visible"][rows]  # [S, N, words]
    word = torch.gather(words, 2, (place // 64)[:, None].expand(seqs, n, longest))
    seen = torch.where(in_tree[:, None], (word >> (place % 64)[:, None]) & 1 == 1, bit[:, None] < 0)
    if w:
        position = torch.where(in_tree, torch.gather(depth, 1, place.clamp_max(n - 1)), bit)  # relative to ctx
        seen = seen & (position[:, None] > depth[:, :, None] - w)
    seen = seen[:, None, :, None]  # [S, 1, N, 1, L]
    q = state["q"].float()[rows].view(seqs, n, kv_heads, group, dim).permute(0, 2, 1, 3, 4)
    scores = torch.matmul(q.reshape(seqs, kv_heads, n * group, dim), keys.permute(0, 2, 3, 1)) * state["scale"]
    scores = scores.view(seqs, kv_heads, n, group, longest).masked_fill_(~seen, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(top == float("-inf"), 0.0, top))
    total = weights.sum(-1, keepdim=True)
    values = torch.where((at[None] < ctx + there.sum(1, keepdim=True))[:, :, None, None], values, 0.0)
    out = torch.matmul(weights.view(seqs, kv_heads, n * group, longest), values.permute(0, 2, 1, 3))
    out = out.view(seqs, kv_heads, n, group, dim) / torch.where(total == 0, 1.0, total)
    out = out.permute(0, 2, 1, 3, 4).reshape(seqs * n, case["heads"] * dim)
    return out[there.view(-1)].to(state["q"].dtype)


def _masses(logits, temperature):
    """A distribution over the vocabulary in whole numbers, the likeliest token's being 2^40: sums of them do not
    depend on their order.  Temperature 0: all of it on the largest logit, ties to the lowest index."""
    vocab = logits.shape[1]
    t = temperature[:, None]
    x = torch.where(torch.isnan(logits), float("-inf"), logits) / torch.where(t > 0, t, 1.0)
    top = x.amax(1, keepdim=True)
    is_top = x == top
    e = torch.where(is_top, 1.0, torch.exp(x - top))
    at = torch.arange(vocab, device=DEVICE)
    first = torch.where(is_top, at, vocab).amin(1, keepdim=True)
    alone = (t <= 0) | (top == float("-inf"))
    e = torch.where(alone, (at == first).float(), e)
    return (e * MASS_ONE).to(torch.int64)


def _plain_verify(state):
    """Nodes in index order: a node is tried when the walk stands at its parent."""
    node_start, parents, tokens = state["node_start"].long(), state["parents"].long(), state["tokens"].long()
    first, n_nodes = node_start[:-1], node_start[1:] - node_start[:-1]
    seqs = first.shape[0]
    cur = torch.zeros_like(first)
    path = torch.full((seqs, state["max_nodes"]), -1, dtype=torch.int32, device=DEVICE)
    path[:, 0] = 0
    count = torch.ones_like(first)
    mass = _masses(state["logits"][first], state["temperature"])
    for i in range(1, state["max_nodes"]):
        row = torch.minimum(first + i, node_start[1:] - 1)
        tried = (i < n_nodes) & (parents[row] == cur)
        token = tokens[row][:, None]
        left = mass.sum(1, keepdim=True).float()
        u = state["uniforms"][row][:, None]
        if state["draft_probs"] is None:
            taken = u * left < torch.gather(mass, 1, token).float()
            less = mass.scatter(1, token, 0)
        else:
            q = state["draft_probs"][first + cur]
            taken = u * torch.gather(q, 1, token) * left < torch.gather(mass, 1, token).float()
            less = (mass - (q * left).to(torch.int64)).clamp_min(0)
        less = torch.where(less.sum(1, keepdim=True) > 0, less, mass)
        taken = taken[:, 0] & tried
        mass = torch.where(taken[:, None], _masses(state["logits"][row], state["temperature"]),
                           torch.where(tried[:, None], less, mass))
        cur = torch.where(taken, i, cur)
        path = path.scatter(1, torch.where(taken, count, 0)[:, None], torch.where(taken, i, 0)[:, None].int())
        count = count + taken.long()
    left = mass.sum(1)
    aim = torch.minimum((state["draws"] * left.float()).to(torch.int64), left - 1)
    at = torch.arange(mass.shape[1], device=DEVICE)
    token = torch.where(torch.cumsum(mass, 1) > aim[:, None], at, mass.shape[1]).amin(1)
    return {"count": count.int(), "path": path, "token": token.int()}


def _plain_keep(state):
    """All that moves is read before any of it is written."""
    page, path = state["case"]["page"], state["path"].long()
    to = torch.arange(path.shape[1], device=DEVICE).expand_as(path)
    seq, step = torch.nonzero((to < state["count"][:, None]) & (path != to), as_tuple=True)
    src = state["ctx_len"].long()[seq] + path[seq, step]
    dst = state["ctx_len"].long()[seq] + step
    table = state["page_table"].long()
    for pool in (state["k"], state["v"]):
        pool[:, table[seq, dst // page], :, dst % page] = pool[:, table[seq, src // page], :, src % page]
    return {"key": state["k"], "value": state["v"]}


# ---------------------------------------------------------------------------- the same in 64 bits
def exact(case, seed):
    """Request by request, in 64 bits.  A verified tree gives whole numbers only: nothing to say about them here."""
    if case["op"] == "verify":
        return None
    state = prepare(case, seed)
    table, page = state["page_table"].tolist(), case["page"]
    lens, counts = _lengths(case), _counts(case)
    place = lambda s, p: (table[s][p // page], p % page)
    if case["op"] == "keep":
        key, value = state["k"].double(), state["v"].double()
        paths, kept = state["path"].tolist(), state["count"].tolist()
        for s, (ctx, path, n) in enumerate(zip(lens, paths, kept)):
            for j in range(n):  # a node never moves forward, so none is overwritten before it has moved
                (a, b), (c, d) = place(s, ctx + path[j]), place(s, ctx + j)
                key[:, c, :, d], value[:, c, :, d] = key[:, a, :, b].clone(), value[:, a, :, b].clone()
        return {"key": key, "value": value}
    heads, group, dim, w = case["heads"], case["heads"] // case["kv_heads"], case["dim"], case["window"]
    trees = _parents(case, random.Random(seed))
    out, first = [], 0
    for s, (ctx, n, tree) in enumerate(zip(lens, counts, trees)):
        total = ctx + n
        pages = torch.tensor([max(p, 0) for p in table[s][:-(-total // page)]], device=DEVICE)
        flat = lambda pool: pool[pages].double().transpose(1, 2).reshape(-1, case["kv_heads"], dim)[:total]
        keys, values = flat(state["k"]), flat(state["v"])
        depths = _depths(tree)
        where = torch.tensor(list(range(ctx)) + [ctx + d for d in depths], device=DEVICE)
        mask = torch.zeros((n, total), dtype=torch.bool, device=DEVICE)
        mask[:, :ctx] = True
        mask[:, ctx:] = torch.tensor([[bool(v >> j & 1) for j in range(n)] for v in _visible(tree)], device=DEVICE)
        if w:
            mask &= where[None] > (ctx + torch.tensor(depths, device=DEVICE))[:, None] - w
        q = state["q"][first:first + n].double().view(n, case["kv_heads"], group, dim)
        scores = torch.einsum("ngid,lgd->gnil", q, keys) * state["scale"]
        scores = scores.masked_fill(~mask[None, :, None], float("-inf"))
        out.append(torch.einsum("gnil,lgd->ngid", torch.softmax(scores, -1), values).reshape(n, heads * dim))
        first += n
    return torch.cat(out)
