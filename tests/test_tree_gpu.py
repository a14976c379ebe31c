"""Attention of drafted trees, their verification and keeping the accepted branch, against plain forms in 64 bits."""
import random

import pytest
import torch

from tree_util import AttentionCase, VerifyCase, paged, random_tree

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def trees(spec, seed=1, chain=False):
    rng = random.Random(seed)
    return [(ctx, random_tree(n, rng, chain)) for ctx, n in spec]


def no_device_error():
    from dispec_b200 import ops
    ops.raise_on_device_error("test")


# ------------------------------------------------------------------------------------- attention
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads,kv_heads,dim", [(12, 2, 128), (28, 4, 128), (8, 8, 64), (3, 1, 32), (5, 1, 8), (16, 4, 256),
                                                (40, 8, 128), (16, 4, 64)])
def test_attention_head_layouts(dtype, heads, kv_heads, dim):
    AttentionCase(trees([(100, 9), (0, 1), (63, 17), (64, 1), (201, 5)]), heads, kv_heads, dim, dtype).check()
    no_device_error()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("spec", [[(0, 1)], [(1, 1)], [(0, 64)], [(0, 65), (130, 130)], [(5000, 3)], [(62, 2), (63, 2), (64, 2)],
                                  [(10, 0), (20, 4), (30, 0)], [(700, 256)], [(40, 4)] * 70, [(3, 1)] * 200,
                                  [(130, 5), (64, 3), (190, 20)] * 40])
def test_attention_lengths(dtype, spec):
    AttentionCase(trees(spec), 12, 2, 128, dtype, seed=3).check()
    no_device_error()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kv_heads,window", [(8, 0), (3, 50), (5, 0), (7, 100)])
def test_attention_many_shares_a_cta(dim, kv_heads, window):
    """Work that is cut at every place: shares of one key tile and of many follow one another in a CTA."""
    spec = [(100 + 61 * i % 400, 1 + 7 * i % 40) for i in range(60)]
    AttentionCase(trees(spec), 4 * kv_heads, kv_heads, dim, BF16, window=window).check()
    no_device_error()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("page_size", [1, 8, 16, 24, 32, 64, 128])
@pytest.mark.parametrize("scatter", [False, True])
def test_attention_pages(dtype, page_size, scatter):
    AttentionCase(trees([(333, 12), (64, 3), (0, 40)]), 8, 2, 128, dtype, page_size=page_size, scatter=scatter).check()
    no_device_error()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window", [1, 2, 7, 64, 100, 1000])
def test_attention_window(dtype, dim, window):
    spec = [(300, 20), (0, 9), (5, 30), (129, 12)]
    AttentionCase(trees(spec), 8, 2, dim, dtype, window=window).check()
    AttentionCase(trees(spec, chain=True), 8, 2, dim, dtype, window=window).check()
    no_device_error()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim", [32, 128])
def test_attention_rows_that_see_nothing_or_not_themselves(dtype, dim):
    case = AttentionCase(trees([(0, 6), (70, 6), (0, 1)]), 8, 2, dim, dtype)
    case.visible[0] = 0       # a root without stored tokens that does not see itself: nothing
    case.visible[3] = 0
    case.visible[7] = 1 << 4  # sees a later node only, beside the stored tokens
    case.visible[12] = 0
    case.check()
    got = case.run()
    assert not got[0].any() and not got[3].any() and not got[12].any()
    no_device_error()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_all_bits_set_and_bits_beyond_the_tree(dtype):
    case = AttentionCase(trees([(20, 3), (0, 64), (9, 5)]), 4, 2, 64, dtype)
    case.visible[:] = -1  # every node sees the whole tree; bits of nodes that are not there mean nothing
    case.check()
    no_device_error()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_attention_hidden_keys_may_be_anything(dtype, bad):
    """A key that a row does not see does not reach it, whatever its numbers are."""
    case = AttentionCase([(50, [-1, 0, 0, 1, 2])], 4, 2, 128, dtype)
    want, bound = case.plain()
    p, o = int(case.table[0, 52 // 16]), 52 % 16
    case.k[p, :, o] = bad  # node 2: seen by itself and node 4
    got = case.run().double().cpu()
    for row in (0, 1, 3):
        assert ((got[row] - want[row]).abs() <= bound[row]).all()
    no_device_error()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("ctx,n,window", [(50, 6, 0), (64, 6, 0), (3000, 70, 0), (200, 9, 3), (1000, 40, 120)])
def test_attention_hidden_values_may_be_anything(dtype, bad, dim, ctx, n, window):
    """A value that a row does not see does not reach it, whatever its numbers are; one that it sees does."""
    case = AttentionCase([(ctx, random_tree(n, random.Random(2))), (90, [-1, 0])], 28, 4, dim, dtype, window=window)
    want, bound = case.plain()
    depth = [int(d) for d in case.depth[:n]]
    inside = lambda i, d: not window or d > depth[i] - window
    # a node, and another one or a stored token that the deeper nodes do not see
    last = ctx - window + 2 if window else ctx + n - 1
    for j in (ctx + 2, last):
        p, o = int(case.table[0, j // 16]), j % 16
        case.v[p, :, o] = bad
    hit = torch.tensor([case.sees(0, i, 2) and inside(i, depth[2]) or
                        (inside(i, 2 - window) if window else case.sees(0, i, n - 1)) for i in range(n)])
    assert 0 < int(hit.sum()) < n
    got = case.run().double().cpu()
    clear = torch.cat([~hit, torch.ones(2, dtype=torch.bool)])
    assert ((got - want).abs() <= bound)[clear].all()
    assert not torch.isfinite(got[:n][hit]).any()
    no_device_error()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("scale", [1e-4, 4.0])
def test_attention_flat_and_sharp_weights(dtype, scale):
    AttentionCase(trees([(400, 9), (31, 4)]), 4, 2, 128, dtype, scale=scale).check()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_rows_of_wider_matrices(dtype):
    case = AttentionCase(trees([(90, 7), (10, 3)]), 4, 2, 64, dtype, extra_columns=64)
    wide = torch.full((10, 4 * 64 + 32), 7.0, dtype=dtype, device="cuda:0")
    case.check(out=wide[:, 16:16 + 256])
    assert (wide[:, :16] == 7).all() and (wide[:, 272:] == 7).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_same_bits_again_and_on_another_stream(dtype):
    case = AttentionCase(trees([(900, 20), (35, 7)]), 12, 2, 128, dtype)
    first = case.run()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        second = case.run()
    side.synchronize()
    assert torch.equal(first, second) and torch.equal(first, case.run())


def test_attention_in_a_graph():
    case = AttentionCase(trees([(150, 9), (35, 7)]), 12, 2, 128, BF16)
    from dispec_b200 import ops
    dev = "cuda:0"
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    q, k, v, table = case.q.to(dev), case.k.to(dev), case.v.to(dev), case.table.to(dev)
    ctx, starts, vis = i32(case.ctx), i32(case.starts), case.visible.to(dev)
    call = lambda: ops.tree_attention(q, k, v, table, ctx, starts, vis, max_nodes=9, scale=case.scale)
    want = call()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        call()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    got.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    # lengths are the device's: the same graph with other lengths
    case.ctx[0] = 97
    ctx.copy_(i32(case.ctx))
    graph.replay()
    want = call()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_page_outside_the_pool_is_reported(dtype):
    from dispec_b200 import ops
    case = AttentionCase(trees([(100, 4)]), 4, 2, 64, dtype)
    case.v = torch.nan_to_num(case.v)
    case.table[0, 2] = case.k.shape[0] + 5
    case.run()
    assert ops.device_error() == 1
    case.table[0, 2] = -1
    got = case.run()
    assert ops.device_error() == 1 and torch.isfinite(got).all()


# ---------------------------------------------------------------------------------- verification
def verify_case(spec, vocab, temperature, drafted, seed, spread=2.0, good=0.6):
    rng = random.Random(seed)
    gen = torch.Generator().manual_seed(seed)
    forest = [random_tree(n, rng, rng.random() < 0.3) for n in spec]
    rows = sum(spec)
    logits = torch.randn(rows, vocab, generator=gen) * spread
    tokens, starts = [rng.randrange(vocab) for _ in range(rows)], [0]
    for n in spec:
        starts.append(starts[-1] + n)
    draft = torch.softmax(logits * 0.8 + torch.randn(rows, vocab, generator=gen), -1) if drafted else None
    for s, tree in enumerate(forest):
        for i, p in enumerate(tree):
            if i == 0:
                continue
            row = starts[s] + p
            if drafted:
                tokens[starts[s] + i] = int(torch.multinomial(draft[row], 1, generator=gen))
            elif rng.random() < good:
                logits[row, tokens[starts[s] + i]] = logits[row].max() + 1.0
    t = [temperature if temperature is not None else rng.choice([0.0, 0.5, 1.0, 1.7]) for _ in spec]
    return VerifyCase(forest, tokens, logits, t, torch.rand(rows, generator=gen), torch.rand(len(spec), generator=gen), draft)


@pytest.mark.parametrize("drafted", [False, True])
@pytest.mark.parametrize("vocab", [1, 2, 37, 256, 1024, 5003, 40000, 151936])
@pytest.mark.parametrize("temperature", [0.0, 0.7, None])
def test_verify_decisions(drafted, vocab, temperature):
    spec = [1, 2, 7, 16, 3, 12] if vocab > 10000 else [1, 2, 7, 0, 16, 33, 65] * 4
    case = verify_case(spec, vocab, temperature, drafted, seed=vocab)
    count, path, token = case.run()
    for s in range(len(spec)):
        case.follow(s, count[s], path[s], token[s])
    no_device_error()


@pytest.mark.parametrize("drafted", [False, True])
def test_verify_gives_the_targets_distribution(drafted):
    """The token behind the root, accepted or drawn, is distributed as the target's."""
    S, vocab, n = 40000, 6, 4
    gen = torch.Generator().manual_seed(11)
    logits = torch.tensor([[0.3, 1.2, -0.7, 0.0, 2.0, -3.0]])
    draft = torch.tensor([[0.35, 0.1, 0.2, 0.25, 0.05, 0.05]])
    tree = [-1, 0, 0, 0]
    if drafted:
        drawn = torch.multinomial(draft[0], 3 * S, replacement=True, generator=gen).view(S, 3).tolist()
    else:
        drawn = [[2, 4, 0]] * S
    tokens = [t for d in drawn for t in [0] + d]
    case = VerifyCase([tree] * S, tokens, logits.repeat(n * S, 1), [1.0] * S, torch.rand(n * S, generator=gen),
                      torch.rand(S, generator=gen), draft.repeat(n * S, 1) if drafted else None)
    count, path, token = case.run()
    seen = torch.zeros(vocab)
    for s in range(S):
        seen[token[s] if count[s] == 1 else tokens[n * s + path[s][1]]] += 1
    p = torch.softmax(logits[0].double(), 0)
    assert ((seen / S - p).abs() <= 5 * (p * (1 - p) / S).sqrt()).all(), (seen / S, p)


def test_verify_greedy_follows_the_largest_logit():
    V = 300
    logits = torch.zeros(5, V)
    logits[0, 7] = logits[0, 9] = 1.0   # a tie: the lower index
    logits[2, 3] = 5.0
    logits[4, 299] = 2.0
    # children of the root: 9 (refused), 7 (taken); of node 2: 4 (refused), 3 (taken)
    case = VerifyCase([[-1, 0, 0, 2, 2]], [0, 9, 7, 4, 3], logits, [0.0], [0.999] * 5, [0.999])
    assert case.run() == ([3], [[0, 2, 4, -1, -1]], [299])


def test_verify_rows_of_infinities_and_nan():
    V = 70
    nan, inf = float("nan"), float("inf")
    logits = torch.zeros(4, V)
    logits[0] = nan
    logits[1] = -inf
    logits[2, 5] = logits[2, 60] = inf  # the mass is shared by the two
    logits[3] = -inf
    logits[3, 33] = 1.0
    logits[3, 34] = nan
    case = VerifyCase([[-1]] * 4, [0] * 4, logits, [1.0] * 4, [0.0] * 4, [0.9, 0.9, 0.9, 0.0])
    assert case.run()[2] == [0, 0, 60, 33]


def test_verify_nothing_left_keeps_the_masses():
    """A draft distribution above the target's everywhere it has mass: the masses stay as they were."""
    logits = torch.full((2, 4), float("-inf"))
    logits[:, 1] = 0.0
    draft = torch.tensor([[0.0, 1.0, 0.0, 0.0]] * 2)
    case = VerifyCase([[-1, 0]], [0, 2], logits, [1.0], [0.5] * 2, [0.3], draft)
    assert case.run() == ([1], [[0, -1]], [1])


def test_verify_edges_of_the_uniform_numbers():
    logits = torch.zeros(2, 3)
    below_one = 1.0 - 2.0 ** -24
    case = VerifyCase([[-1, 0]], [0, 2], logits, [1.0], [0.0, 0.0], [0.0])
    assert case.run() == ([2], [[0, 1]], [0])
    case = VerifyCase([[-1, 0]], [0, 2], logits, [1.0], [0.0, below_one], [below_one])
    assert case.run() == ([1], [[0, -1]], [1])


def test_verify_bfloat16_logits():
    case = verify_case([5, 9, 2], 1000, 0.8, False, seed=4)
    case.logits = case.logits.bfloat16().float()
    assert case.run() == case.run(logits_dtype=BF16)


def test_verify_max_nodes_bounds_the_walk():
    case = verify_case([12], 50, 0.0, False, seed=8)
    case.trees = [[i - 1 for i in range(12)]]
    for i in range(1, 12):
        case.logits[i - 1] = 0
        case.logits[i - 1, case.tokens[i]] = 9.0
    assert case.run()[0] == [12]
    count, path, _ = case.run(max_nodes=5)
    assert count == [5] and path == [[0, 1, 2, 3, 4]]


def test_verify_token_outside_the_vocabulary_is_reported():
    from dispec_b200 import ops
    logits = torch.zeros(3, 8)
    logits[:, 6] = 9.0
    case = VerifyCase([[-1, 0, 0]], [0, 800, 6], logits, [0.0], [0.5] * 3, [0.5])
    assert case.run()[:2] == ([2], [[0, 2, -1]])
    assert ops.device_error() == 2


def test_verify_rows_of_a_wider_matrix():
    case = verify_case([6, 4], 100, 0.9, True, seed=3)
    want = case.run()
    case.logits = torch.nn.functional.pad(case.logits, (0, 28), value=50.0)[:, :100]
    assert case.logits.stride(0) == 128
    from dispec_b200 import ops
    assert case.run() == want and ops.device_error() == 0


# ------------------------------------------------------------------------------------------ keep
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("page_size,heads,dim,layers", [(16, 4, 128, 3), (8, 1, 32, 5), (24, 3, 8, 1), (1, 2, 64, 2), (64, 8, 128, 2)])
def test_keep_moves_the_branch(dtype, page_size, heads, dim, layers):
    from dispec_b200 import ops
    rng = random.Random(5)
    spec = [(0, 30), (17, 9), (64, 1), (5, 70), (33, 12)]
    table, pages = paged([c + n for c, n in spec], page_size, rng, True)
    gen = torch.Generator().manual_seed(2)
    pools = [torch.randn(layers, pages, heads, page_size, d, generator=gen).to(dtype) for d in (dim, 2 * dim)]
    width = 70
    path = torch.full((5, width), -1, dtype=torch.int32)
    count = []
    for s, (_, n) in enumerate(spec):
        nodes = sorted({0} | set(rng.sample(range(n), min(n, n // 2 + 1))))
        count.append(len(nodes) if s != 3 else len(nodes) - 2)
        path[s, :len(nodes)] = torch.tensor(nodes)
    want = [p.clone() for p in pools]
    for s, (ctx, _) in enumerate(spec):
        for j in range(count[s]):
            a, b = ctx + int(path[s, j]), ctx + j
            for w, p in zip(want, pools):
                w[:, table[s, b // page_size], :, b % page_size] = p[:, table[s, a // page_size], :, a % page_size]
    dev = "cuda:0"
    got = [p.to(dev) for p in pools]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    ops.keep_path(got, table.to(dev), i32([c for c, _ in spec]), path.to(dev), i32(count))
    for g, w in zip(got, want):
        assert torch.equal(g.cpu(), w)
    no_device_error()


def test_keep_reports_a_path_that_does_not_ascend_and_pages_outside():
    from dispec_b200 import ops
    dev = "cuda:0"
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    pool = torch.arange(2 * 4 * 1 * 4 * 8, dtype=torch.float32, device=dev).view(2, 4, 1, 4, 8)
    before = pool.clone()
    table = i32([[0, 1]])
    ops.keep_path([pool], table, i32([0]), i32([[0, 3, 2]]), i32([3]))
    assert ops.device_error() == 8
    want = before.clone()
    want[:, 0, :, 1] = before[:, 0, :, 3]
    assert torch.equal(pool, want)
    ops.keep_path([pool], i32([[0, 9]]), i32([0]), i32([[0, 5]]), i32([2]))
    assert ops.device_error() == 1 and torch.equal(pool, want)
    ops.keep_path([pool], table, i32([0]), i32([[0, 5]]), i32([0]))
    assert ops.device_error() == 0 and torch.equal(pool, want)


# -------------------------------------------------------------------------------------- refusals
def test_refusals():
    from dispec_b200 import ops
    dev = "cuda:0"
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    good = dict(q=torch.zeros(2, 32, device=dev), k_pool=torch.zeros(2, 2, 4, 8, device=dev),
                v_pool=torch.zeros(2, 2, 4, 8, device=dev), page_table=i32([[0, 1]]), ctx_len=i32([3]), node_start=i32([0, 2]),
                visible=torch.ones(2, 1, dtype=torch.int64, device=dev), depth=i32([0, 1]), max_nodes=2, scale=1.0)
    ops.tree_attention(**good)
    bad = [dict(q=good["q"].half()), dict(q=good["q"].bfloat16()), dict(q=torch.zeros(2, 24, device=dev)),
           dict(k_pool=torch.zeros(2, 2, 4, 16, device=dev)), dict(v_pool=good["v_pool"].cpu()),
           dict(k_pool=torch.zeros(2, 4, 2, 8, device=dev).transpose(1, 2)), dict(page_table=good["page_table"].long()),
           dict(ctx_len=good["ctx_len"].long()), dict(node_start=i32([0])), dict(visible=good["visible"].int()),
           dict(max_nodes=65), dict(max_nodes=0), dict(scale=0.0), dict(scale=float("nan")), dict(window=-1),
           dict(depth=None, window=4), dict(depth=i32([0])), dict(out=torch.zeros(2, 16, device=dev)),
           dict(q=torch.zeros(2, 32 * 2, device=dev)[:, ::2]),
           dict(q=torch.zeros(2, 8, device=dev), k_pool=torch.zeros(2, 1, 4, 4, device=dev), v_pool=torch.zeros(2, 1, 4, 4, device=dev)),
           dict(q=torch.zeros(65, device=dev)[1:].view(2, 32))]
    for change in bad:
        with pytest.raises(ops.KernelError):
            ops.tree_attention(**{**good, **change})
    good = dict(logits=torch.zeros(2, 9, device=dev), tokens=i32([1, 2]), parents=i32([-1, 0]), node_start=i32([0, 2]),
                temperature=torch.ones(1, device=dev), uniforms=torch.zeros(2, device=dev), draws=torch.zeros(1, device=dev), max_nodes=2)
    ops.verify_tree(**good)
    bad = [dict(logits=good["logits"].half()), dict(logits=torch.zeros(9, 2, device=dev).t()), dict(tokens=i32([1])),
           dict(parents=good["parents"].long()), dict(node_start=i32([0, 2, 2])), dict(temperature=good["temperature"].double()),
           dict(uniforms=torch.zeros(3, device=dev)), dict(draws=good["draws"].cpu()), dict(draft_probs=torch.zeros(2, 8, device=dev)),
           dict(draft_probs=good["logits"].bfloat16()), dict(max_nodes=0), dict(max_nodes=5000), dict(logits=good["logits"].cpu())]
    for change in bad:
        with pytest.raises(ops.KernelError):
            ops.verify_tree(**{**good, **change})
    pool = torch.zeros(1, 2, 1, 4, 8, device=dev)
    table, ctx, path, count = i32([[0, 1]]), i32([0]), i32([[0, 1]]), i32([2])
    ops.keep_path([pool], table, ctx, path, count)
    for args in ([[], table, ctx, path, count], [[pool] * 9, table, ctx, path, count], [[pool[..., :2]], table, ctx, path, count],
                 [[pool.cpu()], table, ctx, path, count], [[torch.zeros(1, 2, 1, 4, 2, device=dev)], table, ctx, path, count],
                 [[pool], table.long(), ctx, path, count], [[pool], table, ctx, path.long(), count],
                 [[pool], table, ctx, path[0], count], [[pool], table, ctx, path, i32([2, 2])],
                 [[pool, torch.zeros(1, 2, 1, 8, 8, device=dev)], table, ctx, path, count]):
        with pytest.raises(ops.KernelError):
            ops.keep_path(*args)


def test_empty_batches():
    from dispec_b200 import ops
    dev = "cuda:0"
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    none = torch.empty((0,), dtype=torch.int32, device=dev)
    pool = torch.zeros(2, 2, 4, 8, device=dev)
    out = ops.tree_attention(torch.zeros(0, 32, device=dev), pool, pool, i32([[0]]), i32([4]), i32([0, 0]),
                             torch.zeros(0, 1, dtype=torch.int64, device=dev), max_nodes=1, scale=1.0)
    assert out.shape == (0, 32)
    f = torch.empty((0,), device=dev)
    got = ops.verify_tree(torch.zeros(0, 9, device=dev), none, none, i32([0]), f, f, f, max_nodes=3)
    assert got.count.shape == (0,) and got.path.shape == (0, 3)
    ops.keep_path([pool.view(1, 2, 2, 4, 8)], torch.zeros((0, 1), dtype=torch.int32, device=dev), none,
                  torch.zeros((0, 3), dtype=torch.int32, device=dev), none)
    no_device_error()
