"""Operators on drafted trees whose device lists point outside the arrays: recorded, left out, and everything else as it was."""
import random

import pytest
import torch

from tree_util import AttentionCase, random_tree

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
LAST = 2 ** 31 - 1


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda:0")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("starts,whole", [([0, 5, 900], [0]), ([0, 5, LAST], [0]), ([-3, 5, 12], [1]), ([-LAST, 5, 12], [1]), ([0, 5, 3], [0]),
                                          ([13, 5, 12], [1]), ([LAST, LAST, -LAST], [])])
def test_attention_trees_outside_the_rows_are_left_out(dtype, starts, whole):
    from dispec_b200 import ops
    case = AttentionCase([(70, random_tree(5, random.Random(1))), (30, random_tree(7, random.Random(2)))], 4, 2, 64, dtype)
    want, bound = case.plain()
    case.starts = starts
    wide = torch.full((16, 256), 7.0, dtype=dtype, device="cuda:0")
    got = case.run(out=wide[2:14]).double().cpu()
    assert ops.device_error() == 8
    rows = [slice(0, 5), slice(5, 12)]
    for s, r in enumerate(rows):
        if s in whole:
            assert ((got[r] - want[r]).abs() <= bound[r]).all()
        else:
            assert (got[r] == 7).all()
    assert (wide[:2] == 7).all() and (wide[14:] == 7).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("ctx", [10 ** 6, LAST, LAST - 40])
def test_attention_more_stored_tokens_than_pages(dtype, ctx):
    from dispec_b200 import ops
    case = AttentionCase([(70, random_tree(5, random.Random(1))), (30, random_tree(7, random.Random(2)))], 4, 2, 64, dtype)
    case.k, case.v = torch.nan_to_num(case.k), torch.nan_to_num(case.v)
    want, bound = case.plain()
    case.ctx = [70, ctx]
    got = case.run().double().cpu()
    assert ops.device_error() == 1
    assert ((got[:5] - want[:5]).abs() <= bound[:5]).all() and torch.isfinite(got[5:]).all()


@pytest.mark.parametrize("vocab", [300, 40000])
@pytest.mark.parametrize("drafted", [False, True])
@pytest.mark.parametrize("starts,whole", [([0, 4, 900], [0]), ([0, 4, LAST], [0]), ([-3, 4, 9], [1]), ([-LAST, 4, 9], [1]), ([0, 4, 3], [0]),
                                          ([11, 4, 9], [1]), ([LAST, -LAST, LAST], [])])
def test_verification_trees_outside_the_rows_have_no_nodes(vocab, drafted, starts, whole):
    from dispec_b200 import ops
    gen = torch.Generator().manual_seed(3)
    parents = [-1, 0, 0, 1, -1, 0, 1, 1, 3]
    logits = torch.randn(9, vocab, generator=gen).cuda()
    draft = torch.softmax(torch.randn(9, vocab, generator=gen), -1).cuda() if drafted else None
    args = (logits, i32(list(range(9))), i32(parents))
    rest = (torch.tensor([0.9, 0.9]).cuda(), torch.rand(9, generator=gen).cuda(), torch.rand(2, generator=gen).cuda(), draft)
    good = ops.verify_tree(*args, i32([0, 4, 9]), *rest, max_nodes=5)
    got = ops.verify_tree(*args, i32(starts), *rest, max_nodes=5)
    assert ops.device_error() == 8
    for s in range(2):
        if s in whole:
            assert got.count[s] == good.count[s] and got.token[s] == good.token[s] and torch.equal(got.path[s], good.path[s])
        else:
            assert got.count[s] == 0 and got.token[s] == -1 and (got.path[s] == -1).all()


# The place of a node is ctx + node: with the node 2^31 - 1 behind 5 tokens that sum, in 32 bits, is negative, and
# divided by the size of a page still below the width of the table.
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("ctx,node", [(5, LAST), (1, LAST), (LAST, 2), (LAST, LAST), (-5, 7), (-LAST, LAST), (0, LAST), (8, 0x40000000)])
def test_keeping_nodes_and_tokens_beyond_what_can_be_counted(dtype, ctx, node):
    from dispec_b200 import ops
    pool = torch.randn(3, 6, 2, 4, 16, generator=torch.Generator().manual_seed(5)).to(dtype).cuda()
    want = pool.clone()
    table = i32([[3, 0, 4], [1, 2, 5]])
    want[:, 2, :, 1] = pool[:, 2, :, 3]  # request 1: node 2 behind 4 + 1 tokens goes where node 0 is
    ops.keep_path([pool], table, i32([ctx, 4]), torch.tensor([[0, node, -1], [0, 3, -1]], dtype=torch.int32).cuda(), i32([2, 2]))
    assert ops.device_error() == 1
    assert torch.equal(pool, want)
