"""Drafted trees: what needs no GPU."""
import pytest
import torch

from dispec_b200.ops import library as L
from dispec_b200.ops import tree


def test_ancestors():
    bits, depth = tree.ancestors([-1, 0, 0, 1, 3])
    assert bits == [[1], [3], [5], [11], [27]] and depth == [0, 1, 1, 2, 3]
    bits, depth = tree.ancestors([i - 1 for i in range(130)])
    assert bits[63] == [-1, 0, 0] and bits[64] == [-1, 1, 0] and bits[129] == [-1, -1, 3] and depth[129] == 129
    assert tree.ancestors([]) == ([], [])


@pytest.mark.parametrize("parents", [[0], [-1, -1], [-1, 1], [-1, 0, 2], [-1, 0, -2]])
def test_ancestors_refuses_what_is_no_tree(parents):
    with pytest.raises(ValueError):
        tree.ancestors(parents)


def test_tensors_on_the_host_are_refused():
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)
    with pytest.raises(L.KernelError, match="CUDA"):
        tree.tree_attention(torch.zeros(1, 8), torch.zeros(1, 1, 4, 8), torch.zeros(1, 1, 4, 8), i32(0)[None], i32(1), i32(0, 1),
                            torch.ones(1, 1, dtype=torch.int64), max_nodes=1, scale=1.0)
    with pytest.raises(L.KernelError, match="CUDA"):
        tree.verify_tree(torch.zeros(1, 8), i32(0), i32(-1), i32(0, 1), torch.ones(1), torch.zeros(1), torch.zeros(1), max_nodes=1)
    with pytest.raises(L.KernelError, match="CUDA"):
        tree.keep_path([torch.zeros(1, 1, 1, 4, 8)], i32(0)[None], i32(0), i32(0)[None], i32(1))
