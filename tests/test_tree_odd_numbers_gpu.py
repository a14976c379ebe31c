"""Attention of drafted trees over queries, keys and values that are not finite: what the definition gives in 64 bits, however
the work is cut among CTAs."""
import random

import pytest
import torch

from tree_util import AttentionCase, random_tree

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
NAN, INF = float("nan"), float("inf")


def no_device_error():
    from dispec_b200 import ops
    ops.raise_on_device_error("test")


def agrees(case):
    """Numbers that are finite in the definition within its bound, the others as they are there."""
    want, bound = case.plain()
    got = case.run().double().cpu()
    finite = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got == INF, want == INF) and torch.equal(got == -INF, want == -INF)
    assert ((got - want).abs() <= bound)[finite].all()
    no_device_error()
    return want


def alone_or_among_others(ctx, n, alone):
    """A tree whose items several CTAs share, or (many trees) one CTA finishes."""
    rng = random.Random(6)
    return [(ctx, random_tree(n, rng))] + ([] if alone else [(ctx - 3 * i % 50, random_tree(n, rng)) for i in range(90)])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("ctx", [5, 200, 4000])
def test_a_query_that_is_no_number_gives_none(dtype, dim, ctx):
    case = AttentionCase([(ctx, random_tree(9, random.Random(2)))], 8, 2, dim, dtype)
    case.q[3, 2 * dim + 5] = NAN
    case.q[5, :] = NAN
    want = agrees(case)
    assert torch.isnan(want[3, 2 * dim:3 * dim]).all() and torch.isfinite(want[3, :2 * dim]).all() and torch.isnan(want[5]).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("alone", [True, False])
@pytest.mark.parametrize("place", [0, 63, 150, 201])
def test_a_key_that_is_no_number_is_in_every_row_that_sees_it(dtype, alone, place):
    case = AttentionCase(alone_or_among_others(200, 6, alone), 8, 2, 128, dtype)
    p, o = int(case.table[0, place // 16]), place % 16
    case.k[p, :, o] = NAN
    want = agrees(case)
    rows = torch.isnan(want[:6]).all(1)
    assert rows.all() if place < 200 else 0 < int(rows.sum()) < 6


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_part_of_keys_that_are_no_numbers(dtype):
    """All scores of the CTA that has them are NaN: its part has no largest score, and still counts."""
    case = AttentionCase([(3000, random_tree(5, random.Random(3)))], 4, 2, 64, dtype)
    for j in range(1024, 1536):
        case.k[int(case.table[0, j // 16]), 0, j % 16] = NAN
    want = agrees(case)
    assert torch.isnan(want[:, :128]).all() and torch.isfinite(want[:, 128:]).all()


# ------------------------------------------------------------------------------------------ values
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim", [64, 128])
def test_values_at_both_ends_of_a_window_stay_with_the_rows_that_see_them(dtype, dim):
    """Window 4,096: the tile at its lower edge and the nodes' are 64 tiles of 64 keys apart, and where there are many
    items one CTA has both."""
    window, ctx, n = 4096, 5000, 9
    rng = random.Random(2)
    case = AttentionCase([(ctx - 64 * (i % 3), random_tree(n, rng)) for i in range(5 if dim == 128 else 10)], 32 * 64 // dim, 32 * 64 // dim,
                         dim, dtype, window=window)
    for s, c in enumerate(case.ctx):
        for j in (c - window + 2, c + 2):
            case.v[int(case.table[s, j // 16]), :, j % 16, 3] = NAN
    want = agrees(case)
    hit = [int(torch.isnan(want[s * n:s * n + n]).any(1).sum()) for s in range(len(case.ctx))]
    assert all(h > 0 for h in hit) and sum(h < n for h in hit) > 1


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("ctx,n,window", [(50, 6, 0), (64, 6, 0), (3000, 70, 0), (200, 9, 3), (1000, 40, 120), (0, 130, 0)])
def test_values_that_are_not_finite_reach_their_own_columns(dtype, dim, ctx, n, window):
    """Infinities of both signs and NaN, in tiles that every row sees whole and in others, a part's first and only tile among them."""
    case = AttentionCase([(ctx, random_tree(n, random.Random(4))), (90, [-1, 0])], 28, 4, dim, dtype, window=window)
    put = lambda s, j, head, column, x: case.v[int(case.table[s, j // 16]), head, j % 16].__setitem__(column, x)
    put(0, ctx + n - 1, 1, 0, INF)
    put(0, ctx + 1, 1, 5, -INF)
    put(0, ctx + 1, 3, dim - 1, NAN)
    put(0, ctx + n // 2, 3, 7, INF)
    put(0, ctx + n // 2, 2, 40, INF)
    put(0, ctx + 1, 2, 40, -INF)
    if ctx:
        put(0, ctx - 1, 0, 2, -INF)
        put(0, max(ctx - 2, ctx - 1 - window // 2) if window else ctx // 3, 0, 33, INF)
    put(1, 10, 2, 17, NAN)
    put(1, 91, 2, 18, -INF)
    want = agrees(case)
    assert torch.isinf(want).any() and torch.isnan(want).any() and torch.isfinite(want).any(1).all()


@pytest.mark.parametrize("dim", [64, 128])
def test_values_that_are_not_finite_on_a_full_server(dim):
    rng = random.Random(9)
    spec = [(100 + 61 * i % 400, random_tree(1 + 7 * i % 40, rng)) for i in range(60)]
    case = AttentionCase(spec, 20, 5, dim, BF16)
    for s, (c, tree) in enumerate(spec):
        for j in (c + len(tree) - 1, c // 2):
            case.v[int(case.table[s, j // 16]), s % 5, j % 16, 3 * s % dim] = (NAN, INF, -INF)[s % 3]
    agrees(case)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim", [64, 128])
def test_a_value_that_is_not_finite_beside_a_page_that_is_not_there(dtype, dim):
    """A page outside the pool hides its own keys only; of the other pages of its tile, values are still the rows' that see them."""
    from dispec_b200 import ops
    case = AttentionCase([(200, random_tree(9, random.Random(4)))], 8, 2, dim, dtype)
    case.v[int(case.table[0, 70 // 16]), 1, 70 % 16, 9] = INF
    case.table[0, 5] = -1  # keys 80 to 95
    got = case.run().double().cpu().view(9, 8, dim)
    assert ops.device_error() == 1
    assert (got[:, 4:, 9] == INF).all()
    got[:, 4:, 9] = 0
    assert torch.isfinite(got).all()
