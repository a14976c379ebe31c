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


def test_quotients_by_a_reciprocal_are_rounded_correctly():
    """What the verification's passes use for logit / temperature: a reciprocal rounded once and two corrections with
    exact remainders (Markstein) give the correctly rounded quotient."""
    import random
    from fractions import Fraction

    import numpy as np

    rng = random.Random(7)
    f32 = np.float32

    def rounded(x: Fraction):  # to 24 bits, ties to even; no number here is near the ends of the range
        if x == 0:
            return Fraction(0)
        e = 0
        a = abs(x)
        while a >= 2 ** 24:
            a /= 2
            e += 1
        while a < 2 ** 23:
            a *= 2
            e -= 1
        n = a.numerator // a.denominator
        rest = a - n
        n += rest > Fraction(1, 2) or (rest == Fraction(1, 2) and n % 2 == 1)
        return (1 if x > 0 else -1) * Fraction(n) * Fraction(2) ** e

    for _ in range(4000):
        t = Fraction(float(f32(rng.choice([0.1, 0.7, 0.8, 1.3, 1.9999999, 3.0, rng.uniform(1e-3, 1e3), 2 ** rng.uniform(-20, 20)]))))
        l = Fraction(float(f32(rng.choice([rng.gauss(0, 5), rng.uniform(-40, 40), 2 ** rng.uniform(-30, 30)]))))
        inv = rounded(1 / t)
        q = rounded(l * inv)
        for _ in range(2):
            rest = rounded(l - q * t)  # one fused multiply-add
            q = rounded(q + rest * inv)
        assert q == rounded(l / t), (float(l), float(t))
