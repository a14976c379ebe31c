"""Several continuations of one prompt at a time: what a step of beam search adds to a step of the engine.

Three operators, timed one call at a time:

``attention``  single tokens of sequences that come in groups with a shared beginning, which is read once for
               all sequences of a group (``ops.shared_prefix_attention``);
``select``     the best continuations of every group of beams, over all its beams and the vocabulary
               (``ops.beam_select``);
``reorder``    caches and states follow the choice: slots of pools are copied to others
               (``ops.reorder_slots``).

Head counts, head sizes, layers, vocabularies and pages of 16 tokens are those of the Qwen2.5 sizes
that ``bench.py`` runs and of the tiny configurations of the tests; states are matrices of 128 x 128 a head.
"""
from __future__ import annotations

import random

import torch

own = False

DEVICE = "cuda:0"
SPREAD = 2.5  # standard deviation of the logits
CAP = {"bytes": 3e8, "flops": 4.2e10}  # no drawn attention costs more than the largest listed one


def listed():
    return [
        # one user, four beams over a short conversation: the time of a launch counts
        dict(name="attention 4 beams", op="attention", groups=1, beams=4, prefix=1000, suffix=20, heads=12, kv_heads=2, dim=128,
             window=0, dtype="bfloat16", page=16, pages="runs"),
        # a small server: eight ragged prompts
        dict(name="attention 8 groups", op="attention", groups=8, beams=5, prefix=4101, suffix=130, heads=28, kv_heads=4, dim=128,
             window=0, dtype="bfloat16", page=16, pages="runs"),
        # 64 answers to a question about a long document, on pages in no order
        dict(name="attention long document", op="attention", groups=1, beams=64, prefix=32768, suffix=300, heads=40, kv_heads=8,
             dim=128, window=0, dtype="bfloat16", page=16, pages="scattered"),
        # a full server: many users' requests behind a few instructions that they share
        dict(name="attention 256 sequences", op="attention", groups=8, beams=32, prefix=2050, suffix=700, heads=28, kv_heads=4,
             dim=128, window=0, dtype="bfloat16", page=16, pages="runs"),
        # the 32-bit path
        dict(name="attention float32", op="attention", groups=2, beams=5, prefix=701, suffix=33, heads=12, kv_heads=2, dim=128,
             window=0, dtype="float32", page=16, pages="scattered"),
        # layers with a sliding window, smaller heads
        dict(name="attention window", op="attention", groups=16, beams=8, prefix=3001, suffix=100, heads=16, kv_heads=4, dim=64,
             window=1024, dtype="bfloat16", page=16, pages="runs"),
        # one user's four beams
        dict(name="select 4 beams", op="select", groups=1, beams=4, vocab=151936, count=8, dtype="float32"),
        # a small server, logits in 16 bits (equal ones are common)
        dict(name="select 8 groups", op="select", groups=8, beams=5, vocab=152064, count=10, dtype="bfloat16"),
        # a full server
        dict(name="select 64 groups", op="select", groups=64, beams=8, vocab=151936, count=16, dtype="float32"),
        # tiny model, 32-bit cache, pages of 8
        dict(name="reorder tiny", op="reorder", kind="pages", groups=2, beams=3, layers=3, kv_heads=1, dim=32, page=8,
             dtype="float32"),
        # recurrent states of four beams each, in place
        dict(name="reorder states", op="reorder", kind="states", groups=8, beams=4, layers=12, kv_heads=8, dim=128, page=0,
             dtype="float32"),
        # a full server's beams that fork: their last pages, all layers
        dict(name="reorder pages", op="reorder", kind="pages", groups=32, beams=8, layers=48, kv_heads=8, dim=128, page=16,
             dtype="bfloat16"),
    ]


def _log(rng, low, high):
    return int(round(low * (high / low) ** rng.random()))


def draw(rng):
    op = rng.choice(["attention", "attention", "select", "reorder"])
    while True:
        if op == "attention":
            heads, kv_heads = rng.choice([(12, 2), (28, 4), (40, 8), (16, 4), (3, 1), (8, 8)])
            case = dict(op=op, groups=_log(rng, 1, 32), beams=_log(rng, 1, 64), prefix=_log(rng, 1, 32768),
                        suffix=_log(rng, 1, 1024), heads=heads, kv_heads=kv_heads, dim=rng.choice([128, 128, 64, 32]),
                        window=rng.choice([0, 0, 0, _log(rng, 16, 4096)]), dtype=rng.choice(["bfloat16"] * 5 + ["float32"]),
                        page=rng.choice([16, 16, 8, 32]), pages=rng.choice(["runs", "scattered"]))
            rows, longest = case["groups"] * case["beams"], case["prefix"] + case["suffix"]
            w = work(case)
            if case["dtype"] == "float32" and w["flops"] > CAP["flops"] / 16:
                continue
            stored = (case["groups"] * case["prefix"] + rows * (case["suffix"] + case["page"])) * kv_heads * case["dim"]
            if w["bytes"] <= CAP["bytes"] and w["flops"] <= CAP["flops"] and stored <= 3e8 and rows * longest * heads <= 3e8:
                return case
        elif op == "select":
            case = dict(op=op, groups=_log(rng, 1, 64), beams=_log(rng, 1, 32), vocab=_log(rng, 200, 152064),
                        count=_log(rng, 2, 64), dtype=rng.choice(["float32", "float32", "bfloat16"]))
            if case["groups"] * case["beams"] * case["vocab"] <= 6.7e7 and case["count"] <= case["vocab"]:
                return case
        else:
            kind = rng.choice(["pages", "states"])
            case = dict(op=op, kind=kind, groups=_log(rng, 1, 32), beams=_log(rng, 2, 16), layers=_log(rng, 2, 48),
                        kv_heads=rng.choice([1, 2, 4, 8]), dim=rng.choice([128, 64, 32]),
                        page=rng.choice([16, 8, 32]) if kind == "pages" else 0, dtype=rng.choice(["bfloat16", "float32"]))
            slots = case["groups"] * case["beams"] * (2 if kind == "pages" else 1)
            if slots * _slot_elements(case) <= 8e8 and work(case)["bytes"] <= 9e8:
                return case


# ------------------------------------------------------------------------------------------ sizes
def _rows(case):
    """Sequences of every group: ragged where there are many."""
    b = case["beams"]
    return [max(1, b - i % 3) if b > 4 else b for i in range(case["groups"])]


def _prefixes(case):
    """Shared tokens of every group: between half of ``prefix`` and all of it, odd ones among them."""
    p, n = case["prefix"], case["groups"]
    return [max(1, p - (i * p) // (2 * n) - (i % 5 if p > 64 else 0)) for i in range(n)]


def _lengths(case):
    """Stored tokens of every sequence, group by group."""
    s = case["suffix"]
    return [[p + max(1, s - (i * s) // (2 * case["groups"]) - j % 3) for j in range(n)]
            for i, (n, p) in enumerate(zip(_rows(case), _prefixes(case)))]


def _moves(case, rng):
    """Which slot goes where after a step: every beam of a group keeps or takes over another one's state; about half of
    them do.  Of pages a beam that takes over gets a fresh one (the second half of the slots)."""
    src, dst, first = [], [], 0
    total = case["groups"] * case["beams"]
    for _ in range(case["groups"]):
        for j in range(case["beams"]):
            parent = rng.randrange(case["beams"])
            if parent != j and rng.random() < 0.6:
                src.append(first + parent)
                dst.append(first + j + (total if case["kind"] == "pages" else 0))
        first += case["beams"]
    return (src, dst) if src else ([1], [total if case["kind"] == "pages" else 0])


def _slot_elements(case):
    """Elements of a slot: a page's keys and values, or a matrix a head, of all layers."""
    return case["layers"] * case["kv_heads"] * case["dim"] * (2 * case["page"] or case["dim"])


def work(case):
    size = 2 if case["dtype"] == "bfloat16" else 4
    if case["op"] == "attention":
        w, keys, pairs, rows = case["window"], 0, 0, 0
        for p, lengths in zip(_prefixes(case), _lengths(case)):
            first = [max(0, n - w) if w else 0 for n in lengths]
            keys += max(0, p - min(first)) + sum(n - max(p, f) for n, f in zip(lengths, first))
            pairs += sum(n - f for n, f in zip(lengths, first))
            rows += len(lengths)
        return {"bytes": (2 * keys * case["kv_heads"] + 2 * rows * case["heads"]) * case["dim"] * size,
                "flops": 4 * pairs * case["heads"] * case["dim"]}
    if case["op"] == "select":
        logits = sum(_rows(case)) * case["vocab"]
        return {"bytes": logits * size, "flops": 4 * logits}
    moved = len(_moves(case, random.Random(1))[0])
    return {"bytes": 2 * moved * _slot_elements(case) * size, "flops": 1}


# ----------------------------------------------------------------------------------------- inputs
def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def prepare(case, seed):
    rng = random.Random(seed)
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    dtype = getattr(torch, case["dtype"])
    normal = lambda *shape: torch.empty(shape, dtype=dtype, device=DEVICE).normal_(generator=gen)
    state = dict(case=dict(case))
    if case["op"] == "reorder":
        src, dst = _moves(case, random.Random(1))
        order = sorted(range(len(dst)), key=dst.__getitem__)
        n = case["groups"] * case["beams"]
        if case["kind"] == "pages":  # of the whole cache, keys and values
            shape = (case["layers"], 2 * n, case["kv_heads"], case["page"], case["dim"])
            state["pools"] = [normal(*shape), normal(*shape)]
        else:  # a buffer for every layer
            state["pools"] = [normal(1, n, case["kv_heads"], case["dim"], case["dim"]) for _ in range(case["layers"])]
        state.update(src=_i32([src[i] for i in order]), dst=_i32([dst[i] for i in order]))
        return state
    starts = [0]
    for n in _rows(case):
        starts.append(starts[-1] + n)
    state["group_start"] = _i32(starts)
    if case["op"] == "select":
        logits = torch.empty((starts[-1], case["vocab"]), dtype=torch.float32, device=DEVICE).normal_(generator=gen)
        state["logits"] = logits.mul_(SPREAD).to(dtype)
        state["scores"] = torch.rand(starts[-1], device=DEVICE, generator=gen) * -6.0 - 20.0
        return state
    # pages: a group's whole shared pages belong to all its sequences; the page in which the shared part ends is every
    # sequence's own copy
    page, prefixes, lengths = case["page"], _prefixes(case), _lengths(case)
    need = sum(p // page + sum(-(-n // page) - p // page for n in of) for p, of in zip(prefixes, lengths))
    ids = list(range(need + 1))
    if case["pages"] == "scattered":
        rng.shuffle(ids)
    width = max(-(-n // page) for of in lengths for n in of)
    table, at, copies = [], 0, []
    for p, of in zip(prefixes, lengths):
        shared = ids[at:at + p // page]
        at += p // page
        for j, n in enumerate(of):
            mine = ids[at:at + -(-n // page) - p // page]
            at += len(mine)
            table.append(shared + mine + [-1] * (width - len(shared) - len(mine)))
            if j == 0:
                leader = mine
            elif p % page:
                copies.append((leader[0], mine[0], p % page))
    shape = (need + 1, case["kv_heads"], page, case["dim"])
    qkv = normal(starts[-1], (case["heads"] + 2 * case["kv_heads"]) * case["dim"])  # the rows of the fused projection
    k, v = normal(*shape), normal(*shape)
    for off in sorted({c[2] for c in copies}):
        a, b = (torch.tensor([c[i] for c in copies if c[2] == off], device=DEVICE) for i in (0, 1))
        for pool in (k, v):
            pool[b, :, :off] = pool[a, :, :off]
    state.update(q=qkv[:, :case["heads"] * case["dim"]], k=k, v=v, scale=1.5 * case["dim"] ** -0.5, page_table=_i32(table),
                 ctx_len=_i32([n for of in lengths for n in of]), prefix_len=_i32(prefixes))
    return state


# ----------------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if own:
        from dispec_b200 import ops

        if case["op"] == "attention":
            return ops.shared_prefix_attention(state["q"], state["k"], state["v"], state["page_table"], state["ctx_len"],
                                               state["group_start"], state["prefix_len"], scale=state["scale"],
                                               window=case["window"])
        if case["op"] == "select":
            got = ops.beam_select(state["logits"], state["scores"], state["group_start"], count=case["count"])
            return {"parent": got.parent, "token": got.token, "score": got.score}
        ops.reorder_slots(state["pools"], state["src"], state["dst"])
        return state["pools"]
    return {"attention": _plain_attention, "select": _plain_select, "reorder": _plain_reorder}[case["op"]](state)


def _group_rows(state):
    """Row of beam j of group g (a group's last row where it has fewer), and which of them there are."""
    start = state["group_start"].long()
    rows = start[:-1, None] + torch.arange(state["case"]["beams"], device=DEVICE)
    return torch.minimum(rows, start[1:, None] - 1), rows < start[1:, None]


def _plain_attention(state):
    """The shared parts as one product a group and head, the rest row by row; one softmax over both."""
    case = state["case"]
    kv_heads, dim, page, w = case["kv_heads"], case["dim"], case["page"], case["window"]
    share, groups, beams = case["heads"] // kv_heads, case["groups"], case["beams"]
    rows, there = _group_rows(state)
    ctx = state["ctx_len"].long()
    prefix = state["prefix_len"].long()
    longest = torch.arange(min(case["prefix"], state["page_table"].shape[1] * page), device=DEVICE)
    rest = torch.arange(case["suffix"], device=DEVICE)
    table = state["page_table"].long().clamp_min(0)
    # keys and values of the shared places [groups, L, kv_heads, dim] and of each row's own [rows, L', kv_heads, dim]
    pages = table[rows[:, 0]][:, longest // page]
    k0, v0 = (state[n][pages, :, longest % page].float() for n in "kv")
    places = (prefix[:, None].expand(groups, beams)[there])[:, None] + rest  # [R, L']
    inside = places.clamp_max(table.shape[1] * page - 1)
    pages = torch.gather(table, 1, inside // page)
    k1, v1 = (state[n][pages, :, inside % page].float() for n in "kv")
    q = state["q"].float().view(-1, kv_heads, share, dim)
    q0 = q[rows].permute(0, 2, 1, 3, 4).reshape(groups, kv_heads, beams * share, dim)
    s0 = (torch.matmul(q0, k0.permute(0, 2, 3, 1)) * state["scale"]).view(groups, kv_heads, beams, share, -1)
    s0 = s0.permute(0, 2, 1, 3, 4)[there]  # [R, kv_heads, share, L]
    s1 = torch.matmul(q, k1.permute(0, 2, 3, 1)) * state["scale"]  # [R, kv_heads, share, L']
    first = (ctx - w if w else torch.zeros_like(ctx))[:, None]
    of_row = prefix[:, None].expand(groups, beams)[there][:, None]
    see0 = (longest[None] < torch.minimum(of_row, ctx[:, None])) & (longest[None] >= first)
    see1 = (places < ctx[:, None]) & (places >= first)
    s0 = s0.masked_fill_(~see0[:, None, None], float("-inf"))
    s1 = s1.masked_fill_(~see1[:, None, None], float("-inf"))
    top = torch.maximum(s0.amax(-1, keepdim=True), s1.amax(-1, keepdim=True))
    top = torch.where(top == float("-inf"), 0.0, top)
    s0, s1 = s0.sub_(top).exp_(), s1.sub_(top).exp_()
    total = s0.sum(-1, keepdim=True) + s1.sum(-1, keepdim=True)
    full = s0.new_zeros((groups, beams) + s0.shape[1:])
    full[there] = s0
    full = full.permute(0, 2, 1, 3, 4).reshape(groups, kv_heads, beams * share, -1)
    o0 = torch.matmul(full, v0.permute(0, 2, 1, 3)).view(groups, kv_heads, beams, share, dim).permute(0, 2, 1, 3, 4)[there]
    v1 = torch.where(see1[:, :, None, None], v1, 0.0)
    out = (o0 + torch.matmul(s1, v1.permute(0, 2, 1, 3))) / torch.where(total == 0, 1.0, total)
    return out.reshape(-1, case["heads"] * dim).to(state["q"].dtype)


def _plain_select(state):
    """Scores in 64 bits, the statistic of a row rounded to 32; the best one is taken out again and again."""
    logits, count = state["logits"].float(), state["case"]["count"]
    top = logits.amax(1, keepdim=True)
    away = logits.double() - top.double()
    log_sum = torch.log(torch.exp(away).sum(1, keepdim=True)).float()
    score = state["scores"].double()[:, None] + away - log_sum.double()
    rows, there = _group_rows(state)
    vocab = score.shape[1]
    left = torch.where(there[:, :, None], score[rows], float("-inf")).view(rows.shape[0], -1)
    at = torch.arange(left.shape[1], device=DEVICE)
    got = []
    for _ in range(count):
        best = left.amax(1, keepdim=True)
        place = torch.where(left == best, at, left.shape[1]).amin(1, keepdim=True)
        left.scatter_(1, place, float("-inf"))
        got.append((torch.gather(rows, 1, place // vocab), place % vocab, best))
    parent, token, best = (torch.cat(x, 1) for x in zip(*got))
    none = best == float("-inf")
    return {"parent": torch.where(none, -1, parent).int(), "token": torch.where(none, -1, token).int(), "score": best.float()}


def _plain_reorder(state):
    """All that moves is read before any of it is written."""
    src, dst = state["src"].long(), state["dst"].long()
    for pool in state["pools"]:
        pool[:, dst] = pool[:, src]
    return state["pools"]


# ---------------------------------------------------------------------------- the same in 64 bits
def exact(case, seed):
    """Row by row, in 64 bits.  A choice gives whole numbers beside its scores: nothing to say about those here."""
    state = prepare(case, seed)
    if case["op"] == "reorder":
        pools = [p.double() for p in state["pools"]]
        before = {s: [p[:, s].clone() for p in pools] for s in state["src"].tolist()}
        for s, d in zip(state["src"].tolist(), state["dst"].tolist()):
            for pool, old in zip(pools, before[s]):
                pool[:, d] = old
        return pools
    starts = state["group_start"].tolist()
    if case["op"] == "select":
        scores = []
        for a, b in zip(starts, starts[1:]):
            log_p = torch.log_softmax(state["logits"][a:b].double(), 1) + state["scores"][a:b, None].double()
            best = torch.sort(log_p.flatten(), descending=True).values[:case["count"]]
            pad = best.new_full((case["count"] - best.numel(),), float("-inf"))
            scores.append(torch.cat([best, pad]))
        return {"parent": None, "token": None, "score": torch.stack(scores)}
    kv_heads, dim, page = case["kv_heads"], case["dim"], case["page"]
    out = []
    for a, p, lengths in zip(starts, _prefixes(case), _lengths(case)):
        for r, n in enumerate(lengths, a):
            first = max(0, n - case["window"]) if case["window"] else 0
            at = torch.arange(first, n, device=DEVICE)
            pages = torch.where(at < p, state["page_table"][a, at // page], state["page_table"][r, at // page]).long()
            keys, values = (state[x][pages, :, at % page].double() for x in "kv")  # [n, kv_heads, dim]
            q = state["q"][r].double().view(kv_heads, -1, dim)
            weights = torch.softmax(torch.einsum("gid,lgd->gil", q, keys) * state["scale"], -1)
            out.append(torch.einsum("gil,lgd->gid", weights, values).reshape(-1))
    return torch.stack(out)
