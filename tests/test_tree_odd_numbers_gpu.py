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
