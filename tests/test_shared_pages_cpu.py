"""Pages that requests share, counted on from step to step, while windows give some of them back."""
import random

import pytest

from test_beam_cpu import grow, manager


def plain(m, names, group=0):
    tables = [m.block_table(r, group) for r in names]
    n = 0
    while n < min(map(len, tables)) and len({t[n] for t in tables}) == 1:
        n += 1
    return n


def test_pages_that_one_has_given_back_and_the_other_still_reads():
    m = manager(window=12)
    m.admit("a")
    grow(m, "a", 16)
    m.fork("a", "b")
    known = m.shared_pages(["a", "b"])
    assert known == 4
    grow(m, "a", 29)  # sees 17 and on
    grow(m, "b", 18)  # sees 6 and on: pages 1, 2 and 3 of those it had in common
    assert m.block_table("a")[:4] == [-1] * 4 and all(p >= 0 for p in m.block_table("b")[1:4])
    known = m.shared_pages(["a", "b"], 0, known)
    assert known == 1 == plain(m, ["a", "b"])  # (nobody reads that one)
    grow(m, "b", 29)
    assert m.shared_pages(["a", "b"], 0, known) == 4 == plain(m, ["a", "b"])


@pytest.mark.parametrize("window", [0, 5, 12, 30])
@pytest.mark.parametrize("seed", range(5))
def test_counted_on_as_counted_anew(window, seed):
    rng = random.Random(seed)
    m = manager(pages=200, window=window)
    m.admit(0)
    grow(m, 0, rng.randrange(1, 30))
    names = [0, 1, 2]
    for n in names[1:]:
        m.fork(0, n)
    known = 0
    for _ in range(40):
        r = rng.choice(names)
        grow(m, r, m.num_tokens(r) + rng.randrange(1, 6))
        known = m.shared_pages(names, 0, known)
        assert known == plain(m, names)
    m.check()
