"""Attention of sequences with a shared beginning, the choice of beams and the reordering of slots, against plain forms in 64 bits."""
import math
import random

import pytest
import torch

from beams_util import SharedCase, plain_select, select_keys, select_tolerance

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
DEV = "cuda:0"


def no_device_error():
    from dispec_b200 import ops
    ops.raise_on_device_error("test")


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------------------------- attention
def long_pages(table):
    """Places for so many tokens more that the kernel for many rows a key is taken where there are such."""
    return torch.nn.functional.pad(table, (0, 1600), value=-1)


@pytest.mark.parametrize("groups", [[(300, [301 + j % 5 for j in range(70)])], [(130, [131] * 40), (700, [701] * 40), (64, [90] * 40)],
                                    [(900, [905] * 60), (200, [201, 210]), (70, [80] * 33), (5, [300])],
                                    [(90, [100] * 17 + [0, 40] * 9)] * 2, [(1, [2] * 70)], [(5000, [5001] * 33)], [(63, [64] * 64)],
                                    [(64, [63] * 65), (0, [5] * 65), (129, [0] * 65)]])
@pytest.mark.parametrize("dim,window,page_size,scatter", [(128, 0, 16, True), (64, 0, 16, True), (128, 60, 16, True), (64, 130, 16, False),
                                                          (128, 0, 8, True), (128, 0, 64, False), (64, 90, 32, True)])
def test_attention_kernel_for_many_rows(groups, dim, window, page_size, scatter):
    case = SharedCase(groups, 8, 2, dim, BF16, window=window, page_size=page_size, scatter=scatter)
    case.table = long_pages(case.table)
    case.check()
    no_device_error()


@pytest.mark.parametrize("heads,kv_heads", [(7, 1), (16, 1), (28, 4), (64, 8), (65, 1), (3, 3)])
def test_attention_head_layouts_of_many_rows(heads, kv_heads):
    case = SharedCase([(200, [203] * 90), (500, [501, 560] * 50)], heads, kv_heads, 128, BF16)
    case.table = long_pages(case.table)
    case.check()
    no_device_error()


@pytest.mark.parametrize("groups", [[(0, [1])], [(0, [0, 1, 0])], [(64, [65, 64, 70])], [(63, [64, 65]), (65, [66, 130, 65])],
                                    [(100, [101]), (100, [101, 140])], [(40, [30, 50, 0, 40])], [(700, [701] * 40)], [(3, [5, 4])] * 90])
@pytest.mark.parametrize("heads,kv_heads,window,page_size,scatter", [(12, 2, 0, 16, True), (3, 1, 0, 8, True), (28, 4, 60, 32, True),
                                                                     (8, 8, 0, 64, False), (33, 1, 7, 16, False), (40, 8, 130, 8, False)])
def test_attention_heads_of_32(groups, heads, kv_heads, window, page_size, scatter):
    SharedCase(groups, heads, kv_heads, 32, BF16, window=window, page_size=page_size, scatter=scatter).check()
    no_device_error()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dim", [32, 64])
def test_attention_hidden_keys_of_few_rows_may_be_anything(bad, dim):
    """What a row does not see does not reach it; a value that is not finite reaches the rows that see it."""
    case = SharedCase([(130, [131, 200, 100, 135]), (20, [40, 21])], 8, 2, dim, BF16)
    want, bound = case.plain()
    hidden = 105  # behind the third sequence's last key, in the part that the others see
    page, o = int(case.table[0, hidden // 16]), hidden % 16
    sees = torch.tensor([any(j == hidden for _, j in case.keys(0, r)) for r in range(4)] + [False] * 2)
    case.v[page, :, o] = bad
    got = case.run().double().cpu()
    assert ((got - want).abs() <= bound)[~sees].all() and not torch.isfinite(got[sees]).any()
    case.k[page, :, o] = bad
    got = case.run().double().cpu()
    assert ((got - want).abs() <= bound)[~sees].all()
    no_device_error()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("window", [0, 90])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_hidden_keys_of_many_rows_may_be_anything(bad, window, dim):
    """What a row does not see does not reach it; a value that is not finite reaches the rows that see it."""
    case = SharedCase([(230, [231, 300, 200, 105] * 20)], 8, 2, dim, BF16, window=window)
    case.table = long_pages(case.table)
    want, bound = case.plain()
    hidden = 202  # behind the last key of half of the sequences, in the part that the others see
    page, o = int(case.table[0, hidden // 16]), hidden % 16
    sees = torch.tensor([any(j == hidden for _, j in case.keys(0, r)) for r in range(80)])
    assert sees.any() and not sees.all()
    case.v[page, :, o] = bad
    got = case.run().double().cpu()
    assert ((got - want).abs() <= bound)[~sees].all() and not torch.isfinite(got[sees]).any()
    case.k[page, :, o] = bad
    got = case.run().double().cpu()
    assert ((got - want).abs() <= bound)[~sees].all()
    no_device_error()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("groups", [[(0, [1])], [(1, [1, 1])], [(0, [0, 1, 0])], [(64, [65, 64, 70])], [(63, [64, 65]), (65, [66, 130, 65])],
                                    [(100, [101]), (100, [101, 140])], [(40, [30, 50, 0, 40])], [(100, [0, 0]), (7, [9, 8])],
                                    [(700, [701] * 40)], [(5, [900, 6, 333])], [(5000, [5001, 5003])], [(3, [5, 4])] * 90])
def test_attention_lengths(dtype, groups):
    SharedCase(groups, 12, 2, 128, dtype, seed=3).check()
    no_device_error()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads,kv_heads,dim", [(12, 2, 128), (28, 4, 128), (8, 8, 64), (3, 1, 32), (5, 1, 8), (16, 4, 256),
                                                (40, 8, 128), (16, 4, 64), (70, 1, 64), (140, 1, 64)])
def test_attention_head_layouts(dtype, heads, kv_heads, dim):
    SharedCase([(100, [109, 101, 130, 100, 163]), (0, [5, 9]), (63, [80] * 7), (200, [201])], heads, kv_heads, dim, dtype).check()
    no_device_error()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kv_heads,window", [(8, 0), (3, 50), (5, 0), (7, 100)])
def test_attention_many_shares_a_cta(dim, kv_heads, window):
    """Work that is cut at every place: shares of one key tile and of many follow one another in a CTA."""
    groups = [(100 + 61 * i % 400, [101 + 61 * i % 400 + 17 * j % 90 for j in range(1 + 7 * i % 11)]) for i in range(40)]
    SharedCase(groups, 4 * kv_heads, kv_heads, dim, BF16, window=window).check()
    no_device_error()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("groups", [[(300, [301 + j % 5 for j in range(70)])], [(130, [131] * 40), (700, [701] * 40), (64, [90] * 40)],
                                    [(900, [905] * 60), (200, [201, 210]), (70, [80] * 33), (5, [300])],
                                    [(90, [100] * 17 + [0, 40] * 9)] * 2])
@pytest.mark.parametrize("dim,window", [(128, 0), (64, 0), (128, 60), (64, 130)])
def test_attention_many_rows_a_key(dtype, groups, dim, window):
    """Shared parts of more than 64 rows a head, alike in their row tiles and not, beside smaller ones."""
    SharedCase(groups, 8, 2, dim, dtype, window=window).check()
    no_device_error()


@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (8, 1), (16, 1), (17, 1), (32, 1), (33, 1), (64, 1)])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_rows_of_a_tile(heads, kv_heads, dim):
    """A tile's rows in one, two and four tiles of sixteen, whole and not."""
    SharedCase([(200, [230, 201]), (90, [91, 140, 95]), (0, [333])], heads, kv_heads, dim, BF16).check()
    no_device_error()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("page_size", [1, 8, 16, 24, 32, 64, 128])
@pytest.mark.parametrize("scatter", [False, True])
def test_attention_pages(dtype, page_size, scatter):
    SharedCase([(333, [345, 340, 334]), (64, [67, 64, 190])], 8, 2, 128, dtype, page_size=page_size, scatter=scatter).check()
    no_device_error()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window", [1, 2, 7, 64, 100, 1000])
def test_attention_window(dtype, dim, window):
    SharedCase([(300, [320, 301, 310]), (0, [9, 4]), (129, [141, 300, 130]), (50, [51])], 8, 2, dim, dtype, window=window).check()
    no_device_error()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_rows_that_see_nothing_and_rows_of_no_group(dtype):
    case = SharedCase([(70, [0, 75, 0]), (0, [0, 0]), (9, [0])], 8, 2, 128, dtype, behind=3)
    out = torch.full((9, 8 * 128), 7.0, dtype=dtype, device=DEV)
    case.check(out=out)
    assert not out[[0, 2, 3, 4, 5]].any() and (out[6:] == 7).all()
    no_device_error()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("window", [0, 90])
def test_attention_hidden_keys_and_values_may_be_anything(dtype, bad, window):
    """What a row does not see does not reach it, whatever its numbers are; a value that it sees does."""
    case = SharedCase([(130, [131, 200, 100, 135]), (20, [40, 21])], 8, 2, 128, dtype, window=window)
    want, bound = case.plain()
    hidden = 105  # behind the third sequence's last key, in the part that the others see
    page, o = int(case.table[0, hidden // 16]), hidden % 16
    for pool in (case.k, case.v):
        pool[page, :, o] = bad
    sees = torch.tensor([any(j == hidden for _, j in case.keys(0, r)) for r in range(4)] + [False] * 2)
    assert sees.tolist()[2] is False and sees.any()
    got = case.run().double().cpu()
    assert ((got - want).abs() <= bound)[~sees].all()
    no_device_error()
    case = SharedCase([(130, [131, 200, 100, 135]), (20, [40, 21])], 8, 2, 128, dtype, window=window)
    case.v[page, :, o] = bad
    got = case.run().double().cpu()
    assert ((got - want).abs() <= bound)[~sees].all() and not torch.isfinite(got[sees]).any()
    no_device_error()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("scale", [1e-4, 4.0])
def test_attention_flat_and_sharp_weights(dtype, scale):
    SharedCase([(400, [409, 500]), (31, [35, 32])], 4, 2, 128, dtype, scale=scale).check()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_rows_of_wider_matrices(dtype):
    case = SharedCase([(90, [95, 100]), (10, [13, 11])], 4, 2, 64, dtype, extra_columns=64)
    wide = torch.full((4, 4 * 64 + 32), 7.0, dtype=dtype, device=DEV)
    case.check(out=wide[:, 16:16 + 256])
    assert (wide[:, :16] == 7).all() and (wide[:, 272:] == 7).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_same_bits_again_and_on_another_stream(dtype):
    case = SharedCase([(900, [920, 901, 950]), (35, [42] * 6)], 12, 2, 128, dtype)
    first = case.run()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        second = case.run()
    side.synchronize()
    assert torch.equal(first, second) and torch.equal(first, case.run())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_in_a_graph(dtype):
    from dispec_b200 import ops
    case = SharedCase([(150, [159, 151, 190]), (35, [42, 36])], 12, 2, 128, dtype)
    tensors = case.tensors()
    call = lambda: ops.shared_prefix_attention(*tensors, scale=case.scale)
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
    tensors[4].copy_(i32([97, 151, 100, 36, 36]))  # lengths and groups are the device's
    tensors[6].copy_(i32([80, 35]))
    graph.replay()
    want = call()
    torch.cuda.synchronize()
    # (the second sequence now reads places 144 to 149 of its own page, where nothing was stored: NaN)
    assert torch.isnan(want[1]).all() and torch.isfinite(want[[0, 2, 3, 4]]).all()
    assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))
    no_device_error()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_page_outside_the_pool_is_reported(dtype):
    from dispec_b200 import ops
    case = SharedCase([(100, [104, 102])], 4, 2, 64, dtype)
    case.v = torch.nan_to_num(case.v)
    case.table[0, 2] = case.k.shape[0] + 5
    case.run()
    assert ops.device_error() == 1
    case.table[0, 2] = -1
    got = case.run()
    assert ops.device_error() == 1 and torch.isfinite(got).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("starts", [[0, 2, 1, 4], [-1, 2, 3, 4], [0, 2, 3, 9], [3, 3, 3, 2]])
def test_attention_groups_outside_the_rows_are_reported_and_left_out(dtype, starts):
    from dispec_b200 import ops
    case = SharedCase([(40, [50, 45]), (0, [9]), (3, [8])], 4, 2, 64, dtype)
    case.k, case.v = torch.nan_to_num(case.k), torch.nan_to_num(case.v)
    case.table = torch.where(case.table < 0, 0, case.table)
    q, k, v, table, lens, _, prefix = case.tensors()
    out = torch.full_like(q, 7.0)
    ops.shared_prefix_attention(q, k, v, table, lens, i32(starts), prefix, scale=1.0, out=out)
    assert ops.device_error() == 16 and torch.isfinite(out).all()
    inside = {r for a, b in zip(starts, starts[1:]) if 0 <= a <= b <= 4 for r in range(a, b)}
    assert (out[[r for r in range(4) if r not in inside]] == 7).all()


def test_attention_lengths_beyond_the_pages_are_cut():
    from dispec_b200 import ops
    case = SharedCase([(60, [64, 64, 64])], 4, 2, 64, BF16)
    q, k, v, table, lens, starts, prefix = case.tensors()
    want = ops.shared_prefix_attention(q, k, v, table, lens, starts, prefix, scale=1.0)
    got = ops.shared_prefix_attention(q, k, v, table, lens.fill_(2 ** 31 - 1), starts, prefix, scale=1.0)
    assert torch.equal(got, want)
    got = ops.shared_prefix_attention(q, k, v, table, lens, starts, prefix.fill_(2 ** 31 - 1), scale=1.0)
    assert torch.isfinite(got).all()
    got = ops.shared_prefix_attention(q, k, v, table, lens.fill_(-5), starts, prefix.fill_(-3), scale=1.0)
    assert not got.any()
    assert ops.device_error() == 1  # (the table is three places wider than the pages that are there: their keys are hidden)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("bad", [-2, -2 ** 31, 2 ** 31 - 1])
def test_attention_pages_of_any_number_are_reported(dtype, bad):
    """In the shared part of many rows, in that of few, and in a sequence's own: the other rows keep their results."""
    from dispec_b200 import ops
    case = SharedCase([(700, [720] * 70), (90, [100, 101]), (0, [40])], 8, 2, 128, dtype)
    case.table = long_pages(case.table)
    want = case.run()
    for row, page, spoilt in ((0, 3, range(70)), (70, 2, (70, 71)), (72, 1, (72,)), (71, 6, (71,))):
        table = case.table.clone()
        case.table[row, page] = bad
        got = case.run()
        case.table = table
        rest = [r for r in range(73) if r not in spoilt]
        assert ops.device_error() == 1 and torch.isfinite(got).all() and torch.equal(got[rest], want[rest])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("groups,heads,kv_heads,dim", [([(16000, [16010, 16001])], 2, 1, 128), ([(11, [12, 9000, 14, 11])], 4, 1, 64),
                                                       ([(9000, [9001])], 1, 1, 32), ([(7000, [7040] * 70)], 2, 1, 64)])
def test_attention_items_of_many_parts(dtype, groups, heads, kv_heads, dim):
    """A row's partial results come from many CTAs, and several threads join them."""
    SharedCase(groups, heads, kv_heads, dim, dtype).check()
    no_device_error()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_calls_behind_and_beside_one_another(dtype):
    """Calls of few and of many rows in turn, without a pause, in a graph, and on two streams at once."""
    from dispec_b200 import ops
    cases = [SharedCase([(900, [905 + j % 7 for j in range(70)])], 8, 2, 128, dtype, seed=1), SharedCase([(300, [310, 305])], 8, 2, 128, dtype, seed=2),
             SharedCase([(640, [700] * 40), (900, [901] * 30)], 8, 2, 128, dtype, seed=3)]
    calls = []
    for case in cases:
        q, k, v, table, lens, starts, prefix = case.tensors()
        table = long_pages(table)
        calls.append(lambda t=(q, k, v, table, lens, starts, prefix), c=case: ops.shared_prefix_attention(*t, scale=c.scale))
    want = []
    for call in calls:
        want.append(call())
        torch.cuda.synchronize()
    turns = [0, 1, 2, 1, 0, 2] * 3
    got = [calls[i]() for i in turns]
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for n, i in enumerate(turns):
        with torch.cuda.stream(sides[n % 2]):
            got.append(calls[i]())
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    for graph in graphs:
        with torch.cuda.graph(graph):
            got += [calls[i]() for i in turns]
    for _ in range(2):
        for graph, side in zip(graphs, sides):
            with torch.cuda.stream(side):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for x, i in zip(got, turns * 4))
    no_device_error()


@pytest.mark.parametrize("dim", [64, 128])
def test_attention_values_that_are_not_finite_in_many_shares_a_cta(dim):
    """Shares of few key tiles follow one another in a CTA, each with such a value that some of its rows see."""
    case = SharedCase([(100 + 64 * (g % 3), [101 + 64 * (g % 3), 300, 90, 95] * 20) for g in range(24)], 8, 2, dim, BF16)
    case.table = long_pages(case.table)
    want, bound = case.plain()
    for g in range(24):
        page = int(case.table[case.starts[g], 95 // 16])
        case.v[page, :, 95 % 16] = float("inf")
    sees = torch.tensor([n > 95 for n in case.lens])
    for _ in range(3):
        got = case.run().double().cpu()
        assert ((got - want).abs() <= bound)[~sees].all() and not torch.isfinite(got[sees]).any()
    no_device_error()


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (BF16, 32), (F32, 128)])
@pytest.mark.parametrize("groups,long", [([(100, [131, 101, 140]), (0, [90])], False), ([(300, [311] * 70)], True)])
def test_attention_pools_beyond_32_bits(dtype, dim, groups, long):
    """More than 2^31 numbers in a pool, and the pages that are read are its last ones."""
    case = SharedCase(groups, 8, 2, dim, dtype)
    if long:
        case.table = long_pages(case.table)
    q, k, v, table, lens, starts, prefix = case.tensors()
    first = (2 ** 31 + 2 ** 24) // k[0].numel() - k.shape[0]
    pools = []
    for pool in (k, v):
        big = torch.empty((first + k.shape[0], *k.shape[1:]), dtype=dtype, device=DEV)
        big[first:] = pool
        pools.append(big)
    from dispec_b200 import ops
    got = ops.shared_prefix_attention(q, *pools, torch.where(table < 0, table, table + first), lens, starts, prefix, scale=case.scale)
    want, bound = case.plain()
    assert ((got.double().cpu() - want).abs() <= bound).all()
    no_device_error()


def test_attention_refusals():
    from dispec_b200 import ops
    from dispec_b200.ops import KernelError
    case = SharedCase([(20, [24, 22])], 4, 2, 64, BF16)
    q, k, v, table, lens, starts, prefix = case.tensors()
    call = lambda *a, **kw: ops.shared_prefix_attention(*a, **{"scale": 1.0, **kw})
    for args in [(q.float(), k, v, table, lens, starts, prefix), (q, k, v[:, :1], table, lens, starts, prefix),
                 (q, k, v, table.long(), lens, starts, prefix), (q, k, v, table, lens[:1], starts, prefix),
                 (q, k, v, table, lens, starts[:2].repeat(2), prefix), (q[:, :192], k, v, table, lens, starts, prefix),
                 (q, k.half(), v.half(), table, lens, starts, prefix), (q, k, v, table, lens.cpu(), starts, prefix),
                 (q.cpu(), k, v, table, lens, starts, prefix), (q, k, v, table[:1], lens, starts, prefix),
                 (q, k, v, table, lens, torch.zeros(1026, dtype=torch.int32, device=DEV), torch.zeros(1025, dtype=torch.int32, device=DEV))]:
        with pytest.raises(KernelError):
            call(*args)
    for kw in [dict(scale=0.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(window=-1), dict(out=q.float()), dict(out=q[:1])]:
        with pytest.raises(KernelError):
            call(q, k, v, table, lens, starts, prefix, **kw)
    empty = call(q[:0], k, v, table[:0], lens[:0], starts[:1], prefix[:0])
    assert empty.shape == (0, 256)
    no_device_error()


# ------------------------------------------------------------------------------------- selection
def choose(logits, scores, starts, count):
    from dispec_b200 import ops
    got = ops.beam_select(logits.to(DEV) if logits.device.type == "cpu" else logits, scores.to(DEV), i32(starts), count=count)
    return got.parent.cpu().long(), got.token.cpu().long(), got.score.cpu()


def check_choice(logits, scores, starts, count, exact=False):
    """Every choice is a candidate, once, in order, and as good as the plain form's at its rank."""
    parent, token, score = choose(logits, scores, starts, count)
    logits = logits.cpu()
    want_parent, want_token, want = plain_select(logits.float(), scores, starts, count)
    keys = select_keys(logits.float(), scores)
    there = want > -math.inf
    largest = float(want[there].abs().max()) if there.any() else 0.0
    tolerance = 2 * select_tolerance(logits.shape[1], largest)
    assert torch.equal(parent >= 0, there) and torch.equal(token >= 0, there)
    assert (score[~there] == -math.inf).all() and (parent[~there] == -1).all() and (token[~there] == -1).all()
    for g, (a, b) in enumerate(zip(starts, starts[1:])):
        p, t = parent[g][there[g]], token[g][there[g]]
        assert len({(int(x), int(y)) for x, y in zip(p, t)}) == len(p)
        assert ((p >= a) & (p < b)).all()
        assert ((keys[p, t] - want[g][there[g]]).abs() <= tolerance).all()
        assert ((score[g][there[g]].double() - keys[p, t]).abs() <= tolerance).all()
        assert (score[g][:-1] >= score[g][1:]).all()
    if exact:
        assert torch.equal(parent, want_parent) and torch.equal(token, want_token)
    no_device_error()


def random_choice(rows, vocab, seed=0, spread=2.5, dtype=F32):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, vocab, generator=gen) * spread).to(dtype), -20.0 - 3 * torch.rand(rows, generator=gen)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [1, 2, 7, 200, 4099, 8192, 8193, 16400, 40001, 151936])
@pytest.mark.parametrize("count", [1, 8, 37, 256])
def test_select_vocabularies(dtype, vocab, count):
    logits, scores = random_choice(9, vocab, seed=vocab + count, dtype=dtype)
    check_choice(logits, scores, [0, 4, 4, 5, 9], count)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [3, 31, 127, 128, 129, 255, 256, 257, 511, 640, 1023, 1024, 1093, 1792, 2047, 2049, 8192 + 130])
@pytest.mark.parametrize("count", [1, 11, 33, 64, 200])
def test_select_rows_that_few_warps_have(dtype, vocab, count):
    logits, scores = random_choice(9, vocab, seed=vocab + count, dtype=dtype)
    check_choice(logits, scores, [0, 3, 4, 9], count)


@pytest.mark.parametrize("starts", [[0, 300], list(range(301)), [0, 1, 1, 150, 300], [5, 40]])
def test_select_groups(starts):
    logits, scores = random_choice(300, 5000, seed=1)
    check_choice(logits, scores, starts, 16)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,vocab,count", [(1, 30000, 256), (4, 9000, 100), (64, 20000, 256), (3, 10, 64)])
def test_select_equal_logits_go_to_the_lowest_row_and_token(dtype, rows, vocab, count):
    logits = torch.zeros(rows, vocab, dtype=dtype)
    check_choice(logits, torch.zeros(rows), [0, rows], count, exact=True)
    logits[:, vocab // 3:] = 1.0  # and above the others
    check_choice(logits, torch.zeros(rows), [0, rows], count, exact=True)
    few = torch.randint(0, 3, (rows, vocab), generator=torch.Generator().manual_seed(1)).to(dtype)
    check_choice(few, torch.zeros(rows), [0, rows], count)
    check_choice(few[:1].expand(rows, vocab).contiguous(), torch.zeros(rows), [0, rows], count, exact=True)


def test_select_sorted_and_lopsided_rows():
    """All that is large in one place: more candidates than the usual bound lets through."""
    ramp = torch.arange(30001, dtype=torch.float32)[None] * 1e-3
    for logits in (ramp, ramp.flip(1)):
        check_choice(logits.contiguous(), torch.zeros(1), [0, 1], 256, exact=True)
    logits, scores = random_choice(2, 30000, seed=4)
    logits.view(2, -1, 4)[:, :, 0] += 50.0  # every thread's first
    logits[0, 8192:8192 + 4 * 700] += 100.0
    check_choice(logits, scores, [0, 2], 256)
    owned = torch.full((1, 8192), -5.0)
    owned[0, torch.arange(8) * 1024] = torch.arange(8).float()  # one thread has all that is large
    check_choice(owned, torch.zeros(1), [0, 1], 64, exact=True)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_select_numbers_that_are_not_finite(dtype):
    logits, scores = random_choice(8, 9001, seed=2, dtype=dtype)
    logits[0] = -math.inf           # nothing to choose
    logits[1, 5:] = -math.inf       # five tokens allowed
    logits[2, ::2] = float("nan")
    logits[3, 4000] = math.inf      # one infinity has all the mass
    logits[4, [7, 9000]] = math.inf
    logits[5, :8999] = torch.finfo(dtype).min
    scores[6], scores[7] = -math.inf, float("nan")
    check_choice(logits, scores, [0, 1, 2, 3, 4, 5, 6, 7, 8], 12)
    check_choice(logits, scores, [0, 8], 40)
    scores[6] = math.inf
    check_choice(logits, scores, [0, 8], 40)
    check_choice(logits[:2], scores[:2], [0, 2], 9)


def test_select_masked_vocabulary_of_many_beams():
    logits = torch.full((40, 151936), -math.inf)
    gen = torch.Generator().manual_seed(0)
    for r in range(40):
        logits[r, torch.randint(0, 151936, (3,), generator=gen)] = torch.randn(3, generator=gen)
    check_choice(logits, -torch.rand(40, generator=gen), [0, 10, 40], 64)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_select_equal_rows_wherever_they_lie(dtype):
    """Rows of an odd length begin at every alignment; equal ones tie all the same, and the lowest row wins."""
    logits, _ = random_choice(1, 20003, seed=5, dtype=dtype)
    check_choice(logits.expand(12, 20003).contiguous(), torch.full((12,), -3.0), [0, 12], 30, exact=True)
    wide = torch.full((12, 20011), math.nan, dtype=dtype, device=DEV)
    wide[:, 3:20006] = logits.to(DEV)
    check_choice(wide[:, 3:20006], torch.full((12,), -3.0), [0, 5, 12], 30, exact=True)


def test_select_same_bits_again_in_a_graph_and_on_another_stream():
    from dispec_b200 import ops
    logits, scores = random_choice(12, 30011, seed=6)
    logits, scores, starts = logits.to(DEV), scores.to(DEV), i32([0, 4, 12])
    call = lambda: ops.beam_select(logits, scores, starts, count=16)
    first = call()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        second = call()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        third = call()
    graph.replay()
    torch.cuda.synchronize()
    for other in (second, third):
        assert torch.equal(first.parent, other.parent) and torch.equal(first.token, other.token) and torch.equal(first.score, other.score)
    logits.copy_(random_choice(12, 30011, seed=7)[0])
    graph.replay()
    again = call()
    torch.cuda.synchronize()
    assert torch.equal(again.token, third.token) and not torch.equal(again.token, first.token)


def test_select_without_rows_follows_what_comes_before_it():
    """The groups are read when the kernels in front have written them."""
    from dispec_b200 import ops
    logits, scores = random_choice(64, 40001, seed=8)
    logits, scores = logits.to(DEV), scores.to(DEV)
    starts = i32([0, 32, 64])
    for _ in range(20):
        first = ops.beam_select(logits, scores, starts, count=8)
        none = ops.beam_select(logits[:0], scores[:0], first.parent[0, :3] * 0, count=8)
        assert (none.parent == -1).all() and (none.token == -1).all() and (none.score == -math.inf).all()
    no_device_error()


@pytest.mark.parametrize("starts", [[0, 3, 2, 4], [-1, 2, 3, 4], [0, 2, 3, 9]])
def test_select_groups_outside_the_rows_are_reported(starts):
    from dispec_b200 import ops
    logits, scores = random_choice(4, 300)
    got = ops.beam_select(logits.to(DEV), scores.to(DEV), i32(starts), count=4)
    assert ops.device_error() == 16
    for g, (a, b) in enumerate(zip(starts, starts[1:])):
        if not 0 <= a <= b <= 4:
            assert (got.parent[g] == -1).all() and (got.token[g] == -1).all() and (got.score[g] == -math.inf).all()
        else:
            assert ((got.parent[g] >= a) & (got.parent[g] < b)).all()


def test_select_logits_beyond_32_bits():
    rows, vocab = 15000, 152064
    from dispec_b200 import ops
    logits = torch.empty((rows, vocab), dtype=BF16, device=DEV).normal_(std=2.5)
    scores = -torch.rand(rows, device=DEV)
    got = ops.beam_select(logits, scores, torch.arange(0, rows + 1, 5, dtype=torch.int32, device=DEV), count=10)
    for g in (0, 1500, 2999):
        of = slice(5 * g, 5 * g + 5)
        alone = ops.beam_select(logits[of].clone(), scores[of].clone(), i32([0, 5]), count=10)
        assert torch.equal(got.token[g], alone.token[0]) and torch.equal(got.parent[g], alone.parent[0] + 5 * g) and torch.equal(got.score[g], alone.score[0])
    of = slice(rows - 5, rows)
    parent, token, best = plain_select(logits[of].cpu(), scores[of].cpu(), [0, 5], 10)
    assert (got.score[-1].cpu().double() - best[0]).abs().max() <= select_tolerance(vocab, 30.0)
    no_device_error()


def test_select_refusals():
    from dispec_b200 import ops
    from dispec_b200.ops import KernelError
    logits, scores = (x.to(DEV) for x in random_choice(4, 300))
    starts = i32([0, 4])
    for args, count in [((logits.half(), scores, starts), 4), ((logits, scores.double(), starts), 4), ((logits, scores[:3], starts), 4),
                        ((logits, scores, starts.long()), 4), ((logits, scores, starts), 0), ((logits, scores, starts), 257),
                        ((logits.t(), scores, starts), 4), ((logits[0], scores, starts), 4), ((logits.cpu(), scores, starts), 4),
                        ((logits, scores.cpu(), starts), 4), ((logits, scores, starts[:0]), 4)]:
        with pytest.raises(KernelError):
            ops.beam_select(*args, count=count)
    none = ops.beam_select(logits[:0], scores[:0], i32([0, 0]), count=3)
    assert (none.parent == -1).all() and (none.token == -1).all() and none.parent.shape == (1, 3)
    assert ops.beam_select(logits, scores, starts[:1], count=3).parent.shape == (0, 3)
    no_device_error()


# ------------------------------------------------------------------------------------ reordering
def reorder(pools, src, dst):
    from dispec_b200 import ops
    want = [p.clone() for p in pools]
    for w, p in zip(want, pools):
        w[:, dst] = p[:, src]
    ops.reorder_slots(pools, i32(src), i32(dst))
    for w, p in zip(want, pools):
        assert torch.equal(w, p)
    no_device_error()


def pool(layers, slots, *shape, dtype=BF16, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randint(-1000, 1000, (layers, slots) + shape, generator=gen, device=DEV).to(dtype)


@pytest.mark.parametrize("shape", [(8, 16, 128), (2, 8, 32), (3,), (1,), (5, 7), (4, 128, 128), (1, 16, 24)])
@pytest.mark.parametrize("dtype", [BF16, F32, torch.int32, torch.int64])
def test_reorder_rows_of_every_size(shape, dtype):
    pools = [pool(3, 20, *shape, dtype=dtype, seed=s) for s in range(2)]
    reorder(pools, [4, 4, 1, 0, 19], [0, 1, 2, 7, 12])


@pytest.mark.parametrize("n", [1, 2, 3, 64, 511, 512, 513, 1000, 2048, 5000, 8192])
def test_reorder_all_slots_at_once(n):
    """Every slot is read and written: a cycle, a permutation, one slot for all."""
    src = list(range(n))
    for order in (src[1:] + src[:1], random.Random(n).sample(src, n), [n // 2] * n):
        reorder([pool(2, n, 3, 40), pool(1, n, 8, dtype=F32)], order, src)


@pytest.mark.parametrize("n", [11, 12, 144, 147, 148, 149, 295, 296, 297, 384])
def test_reorder_whole_lines_and_parts_of_them(n):
    """Entries whose columns are copied by lines of 128 bytes and by less, with rows that are no multiple of either."""
    for shape in ((8, 208), (5, 8), (2, 16, 128)):
        src = torch.randperm(n + 5, generator=torch.Generator().manual_seed(n))[:n].tolist()
        reorder([pool(2, n + 5, *shape, dtype=BF16)], src, list(range(5, n + 5)))
        no_device_error()


def test_reorder_many_pools_of_different_rows():
    pools = [pool(1 + s % 3, 9, 1 + s % 5, 8 * (1 + s % 7), dtype=(BF16, F32)[s % 2], seed=s) for s in range(64)]
    reorder(pools, [8, 0, 3, 3], [0, 1, 2, 8])


def test_reorder_in_a_graph_and_on_another_stream():
    from dispec_b200 import ops
    p = pool(2, 8, 4, 16)
    src, dst = i32([1, 0, 5]), i32([0, 1, 2])
    before = p.clone()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        ops.reorder_slots([p], src, dst)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.reorder_slots([p], src, dst)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(p[:, :2], before[:, :2]) and torch.equal(p[:, 2], before[:, 5]) and torch.equal(p[:, 3:], before[:, 3:])


@pytest.mark.parametrize("src,dst,kept", [([1, 2, 3], [0, 4, 4], 2), ([1, 2, 3], [5, 3, 6], 1), ([1, 8, 3], [0, 4, 5], 1),
                                          ([-1, 2], [0, 1], 0), ([1, 2], [0, 8], 1), ([1, 2], [-1, 3], 0)])
def test_reorder_slots_that_do_not_ascend_or_are_not_there_are_reported(src, dst, kept):
    from dispec_b200 import ops
    p = pool(2, 8, 4, 16)
    want = p.clone()
    want[:, dst[:kept]] = p[:, src[:kept]]
    ops.reorder_slots([p], i32(src), i32(dst))
    assert ops.device_error() == 16 and torch.equal(p, want)


@pytest.mark.parametrize("shape", [(40, 2 ** 16), (40, 2 ** 16 - 2)])
def test_reorder_pools_beyond_32_bits(shape):
    """More than 2^32 bytes in front of the slots, in both ways of copying."""
    p = torch.zeros((2, 900, *shape), dtype=BF16, device=DEV)
    p[:, 890:] = torch.randn((2, 10, *shape), device=DEV).to(BF16)
    want = p[:, 890:].clone()
    want[:, [0, 3, 9]] = want[:, [9, 0, 5]]
    from dispec_b200 import ops
    ops.reorder_slots([p], i32([899, 890, 895]), i32([890, 893, 899]))
    assert torch.equal(p[:, 890:], want) and not p[:, :890].any()
    no_device_error()


def test_reorder_refusals():
    from dispec_b200 import ops
    from dispec_b200.ops import KernelError
    p, one = pool(2, 8, 4, 16), i32([1])
    for args in [([], one, one), ([p.cpu()], one, one), ([p], one.long(), one), ([p], one, i32([1, 2])), ([p], one.cpu(), one),
                 ([p, pool(2, 9, 4)], one, one), ([p.transpose(2, 3)], one, one), ([p.half()], one, one), ([p[:, :, 0, 0]], one, one),
                 ([p, p], one, one), ([p[None, None]], one, one), ([pool(1, 8, 2) for _ in range(65)], one, one),
                 ([p], torch.zeros(8193, dtype=torch.int32, device=DEV), torch.arange(8193, dtype=torch.int32, device=DEV))]:
        with pytest.raises(KernelError):
            ops.reorder_slots(*args)
    before = p.clone()
    ops.reorder_slots([p], one[:0], one[:0])
    assert torch.equal(p, before)
    no_device_error()
