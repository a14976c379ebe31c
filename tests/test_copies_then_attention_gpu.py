"""Attention of single tokens right behind a kernel that moves what is stored, with nothing between the two: it sees what was moved,
though it asks for its first keys before the kernel in front of it is complete."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
PAGE, KVH, GROUP, DIM = 16, 4, 7, 128


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


class Step:
    """A step of single tokens, planned: every list is on the device, and one kernel runs."""

    def __init__(self, ctx, table):
        gen = torch.Generator(device=DEV).manual_seed(1)
        self.n, self.table = len(ctx), table
        self.q = torch.randn(self.n, KVH * GROUP * DIM, generator=gen, device=DEV).to(torch.bfloat16)
        self.ctx, self.start, self.seq, self.tok0 = i32(ctx), i32(range(self.n + 1)), i32(range(self.n)), i32([0] * self.n)

    def attend(self, k, v):
        from dispec_b200.ops.attention import paged_attention_tiles
        out = torch.empty_like(self.q)
        paged_attention_tiles(self.q, self.q.stride(0), k, v, self.table, self.start, self.ctx, self.seq, self.tok0, self.n, self.n, out,
                              KVH * GROUP, KVH, DIM, 0, DIM ** -0.5, splits=4)
        return out


def many_times(move, attend, contents):
    """``move(c)`` puts content c where the attention reads; then, with nothing between, ``attend()``."""
    want = []
    for c in range(contents):
        move(c)
        torch.cuda.synchronize()
        want.append(attend())
        torch.cuda.synchronize()
    assert all(not torch.equal(want[0], w) for w in want[1:])
    turns = [c for _ in range(20) for c in range(contents)]
    got = []
    for c in turns:
        move(c)
        got.append(attend())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for c in turns:
            move(c)
            got.append(attend())
    for _ in range(10):
        for x in got[len(turns):]:
            x.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, want[c]) for x, c in zip(got, turns * 2))


@pytest.mark.parametrize("seqs,tokens,layers", [(2, 200, 6), (8, 1000, 3), (16, 1000, 2)])
def test_attention_behind_reordered_pages(seqs, tokens, layers):
    """By bulk copies (up to 512 entries) and through registers."""
    from dispec_b200 import ops
    pages = -(-tokens // PAGE)
    n = seqs * pages
    gen = torch.Generator(device=DEV).manual_seed(2)
    # the pages that are read, and two contents for them
    k, v = (torch.randn(layers, 3 * n, KVH, PAGE, DIM, generator=gen, device=DEV).to(torch.bfloat16) for _ in range(2))
    step = Step([tokens] * seqs, torch.randperm(n, generator=torch.Generator().manual_seed(3)).to(torch.int32).view(seqs, pages).to(DEV))
    dst, src = i32(range(n)), [i32(range(n, 2 * n)), i32(range(2 * n, 3 * n))]
    many_times(lambda c: ops.reorder_slots([k, v], src[c], dst), lambda: step.attend(k[-1], v[-1]), 2)
    ops.raise_on_device_error("test")


@pytest.mark.parametrize("seqs,tokens,layers", [(2, 200, 12), (16, 1000, 6)])
def test_attention_behind_an_accepted_branch(seqs, tokens, layers):
    """The branch's keys and values lie, once moved, in front of the newest token, in pages that the attention asks for early."""
    from dispec_b200 import ops
    nodes = 96  # behind them lie the newest token and as many nodes again
    pages = -(-(tokens + 2 * nodes) // PAGE)
    gen = torch.Generator(device=DEV).manual_seed(4)
    k, v = (torch.randn(layers, seqs * pages, KVH, PAGE, DIM, generator=gen, device=DEV).to(torch.bfloat16) for _ in range(2))
    table = torch.randperm(seqs * pages, generator=torch.Generator().manual_seed(5)).to(torch.int32).view(seqs, pages).to(DEV)
    step = Step([tokens + nodes // 2] * seqs, table)
    stored, count = i32([tokens] * seqs), i32([nodes // 2] * seqs)
    # node j's branch: every second node from j on, so that each call moves other numbers to the same places
    paths = [i32([[c + 2 * j for j in range(nodes // 2)]] * seqs).contiguous() for c in (0, 1)]
    first = [x.clone() for x in (k, v)]

    def move(c):
        k.copy_(first[0])
        v.copy_(first[1])
        ops.keep_path([k, v], table, stored, paths[c], count)

    many_times(move, lambda: step.attend(k[-1], v[-1]), 2)
    ops.raise_on_device_error("test")
