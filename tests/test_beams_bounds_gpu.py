"""Operators on beams whose device lists overlap or point outside the arrays: recorded, left out, and everything else as it was."""
import pytest
import torch

from beams_util import SharedCase

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
DEV = "cuda:0"
LAST = 2 ** 31 - 1


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


# dtype, head size, places for so many tokens that the kernel for many rows a key is taken
KERNELS = [(BF16, 128, False), (BF16, 64, True), (BF16, 32, False), (F32, 64, False)]


@pytest.mark.parametrize("dtype,dim,long", KERNELS)
@pytest.mark.parametrize("groups,starts,prefix", [
    # behind the group that there is, one that has two of its rows, and an empty one
    ([(90, [130 + j % 70 for j in range(301)])], [0, 301, 299, 301, 301], [90, 0, 4000, 0]),
    ([(400, [405 + j % 9 for j in range(90)])], [0, 90, 20, 90, 50, 90], [400, 0, 64, 0, 64]),
    # groups that end beyond the rows or begin in front of them, between others that are there
    ([(70, [90] * 40), (130, [140, 131])], [0, 40, LAST, 40, 42], [70, 9, 9, 130]),
    ([(70, [90] * 40), (130, [140, 131])], [0, 40, -LAST - 1, 40, 42], [70, 9, 9, 130]),
    ([(70, [90] * 5), (0, [60]), (130, [140, 131])], [-3, LAST, 0, 5, 6, 8, 7, 6, 8, 9], [9, 9, 70, 0, 130, 7, 7, 8, 9])])
def test_attention_groups_that_overlap_are_left_out(dtype, dim, long, groups, starts, prefix):
    from dispec_b200 import ops
    case = SharedCase(groups, 8, 2, dim, dtype)
    if long:
        case.table = torch.nn.functional.pad(case.table, (0, 1600), value=-1)
    want, bound = case.plain()
    q, k, v, table, lens, _, _ = case.tensors()
    out = torch.full((q.shape[0], q.shape[1]), 7.0, dtype=dtype, device=DEV)
    for _ in range(3):
        ops.shared_prefix_attention(q, k, v, table, lens, i32(starts), i32(prefix), scale=case.scale, out=out)
        got = out.double().cpu()
        assert ops.device_error() == 16 and ((got - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype,dim,long", KERNELS)
def test_attention_rows_between_groups_that_are_there_stay(dtype, dim, long):
    """Every other group is out; its rows are in none."""
    from dispec_b200 import ops
    lengths = [100 + 7 * r % 60 for r in range(60)]
    case = SharedCase([(0, [n]) for n in lengths], 8, 2, dim, dtype)
    if long:
        case.table = torch.nn.functional.pad(case.table, (0, 1600), value=-1)
    want, bound = case.plain()
    q, k, v, table, lens, _, _ = case.tensors()
    starts = [x for r in range(0, 60, 3) for x in (r, r + 1, LAST)] + [60]  # rows 0, 3, 6, ...
    out = torch.full((60, q.shape[1]), 7.0, dtype=dtype, device=DEV)
    ops.shared_prefix_attention(q, k, v, table, lens, i32(starts), i32([50] * 60), scale=case.scale, out=out)
    got = out.double().cpu()
    there = torch.arange(60) % 3 == 0
    assert ops.device_error() == 16 and ((got - want).abs() <= bound)[there].all() and (got[~there] == 7).all()


@pytest.mark.parametrize("dtype,dim,long", KERNELS)
@pytest.mark.parametrize("scale", [1e-44, 1e-38])
def test_attention_of_the_smallest_scales(dtype, dim, long, scale):
    """All weights are one, and hidden keys have none."""
    from dispec_b200 import ops
    case = SharedCase([(100, [130, 101, 90] * 30), (9, [20])], 8, 2, dim, dtype, scale=scale)
    if long:
        case.table = torch.nn.functional.pad(case.table, (0, 1600), value=-1)
    case.check()
    ops.raise_on_device_error("test")


def test_reorder_lists_in_a_pool_are_refused():
    """Blocks would read them while others write there."""
    from dispec_b200 import ops
    from dispec_b200.ops import KernelError
    pool = torch.arange(2 * 8 * 16, dtype=torch.int32, device=DEV).view(2, 8, 16) % 8
    before = pool.clone()
    inside, apart = pool.view(-1)[4:6], i32([1, 2])
    for src, dst in ((inside, apart), (apart, inside), (pool.view(-1)[-2:], apart), (apart, pool.view(-1)[:2])):
        with pytest.raises(KernelError, match="pool 1"):
            ops.reorder_slots([torch.zeros(1, 8, 4, dtype=torch.int32, device=DEV), pool], src, dst)
    assert torch.equal(pool, before)
    both = i32([0, 1] + list(range(100, 164)) + [2, 5])  # beside a pool is not in it
    want = both[2:66].view(2, 8, 4).clone()
    want[:, [2, 5]] = want[:, [0, 1]]
    ops.reorder_slots([both[2:66].view(2, 8, 4)], both[:2], both[66:])
    assert torch.equal(both[2:66].view(2, 8, 4), want)
    assert ops.device_error() == 0


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("masked", [-1e9, torch.finfo(torch.bfloat16).min])
@pytest.mark.parametrize("kept,count", [(3, 8), (20, 8), (20, 40), (9000, 256)])
def test_select_rows_masked_by_a_finite_number(dtype, masked, kept, count):
    """Most of a piece is equal, and it may take masked tokens to fill the choice: the lowest ones."""
    from beams_util import plain_select, select_tolerance
    from dispec_b200 import ops
    gen = torch.Generator().manual_seed(kept)
    logits = torch.full((6, 30000), masked)
    for row in logits:
        row[torch.randperm(30000, generator=gen)[:kept]] = 2.5 * torch.randn(kept, generator=gen)
    logits, scores = logits.to(dtype), -10 * torch.rand(6, generator=gen)
    starts = [0, 4, 6]
    got = ops.beam_select(logits.to(DEV), scores.to(DEV), i32(starts), count=count)
    parent, token, key = plain_select(logits.float(), scores, starts, count)
    assert ops.device_error() == 0 and (got.parent >= 0).all()
    # scores are rounded to 32 bits, and those of masked tokens are as large as the mask
    tolerance = select_tolerance(30000, 30.0) + key.abs() * 2.0 ** -23
    assert ((got.score.cpu().double() - key).abs() <= tolerance).all()
    sure = torch.ones_like(key, dtype=torch.bool)  # where the next in line is not as good
    sure[:, 1:] &= (key[:, :-1] - key[:, 1:]) > 2 * tolerance[:, 1:]
    sure[:, :-1] &= (key[:, :-1] - key[:, 1:]) > 2 * tolerance[:, :-1]
    sure[:, -1] = False
    assert torch.equal(got.parent.cpu()[sure].long(), parent[sure]) and torch.equal(got.token.cpu()[sure].long(), token[sure])
    # of one row's masked tokens, which are all equal, the lowest are taken, in order
    for g in range(2):
        p, t = got.parent[g].cpu(), got.token[g].cpu()
        for r in set(p.tolist()):
            mine = t[(p == r) & (logits[p.long(), t.long()] == logits.min())]
            lowest = (logits[r] == logits.min()).nonzero()[:len(mine), 0]
            assert torch.equal(mine.long(), lowest)
