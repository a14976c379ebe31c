"""Drafts looked up: an occurrence counts once, however many of the last tokens it shares."""
import random

import pytest

from dispec_b200.engine.speculative import look_up


def branches_of(nodes, parents):
    """Token paths from the root's children down, one per leaf."""
    leaves = set(range(len(nodes))) - set(parents)
    out = []
    for leaf in sorted(leaves):
        path, k = [], leaf
        while k > 0:
            path.append(nodes[k])
            k = parents[k]
        out.append(path[::-1])
    return out


def test_what_followed_shorter_tails_is_drafted_beside_the_longest_match():
    tokens = [9, 3, 50, 8, 3, 60, 1, 2, 3, 70, 71, 1, 2, 3]
    assert branches_of(*look_up(tokens, 16)) == [[70, 71, 1, 2, 3], [60, 1, 2, 3, 70], [50, 8, 3, 60, 1]]
    # the longest match first, where there is room for fewer
    assert [b[0] for b in branches_of(*look_up(tokens, 16, branches=2))] == [70, 60]
    assert [b[0] for b in branches_of(*look_up(tokens, 16, branches=1))] == [70]


@pytest.mark.parametrize("seed", range(20))
def test_continuations_are_the_latest_of_the_longest_tails(seed):
    """Against a list of all earlier occurrences, ordered by how many of the last tokens they share and by how late they are."""
    rng = random.Random(seed)
    tokens = [rng.randrange(4) for _ in range(rng.randrange(2, 40))]
    longest, branches, max_nodes = rng.randrange(1, 4), rng.randrange(1, 4), rng.randrange(2, 20)
    shared = {}
    for end in range(1, len(tokens)):  # a continuation begins at `end`
        n = 0
        while n < min(longest, end) and tokens[end - 1 - n] == tokens[-1 - n]:
            n += 1
        if n:
            shared[end] = n
    order = sorted(shared, key=lambda end: (-shared[end], -end))[:branches]
    each = max(1, (max_nodes - 1) // branches)
    paths, want = [()], [()]  # nodes as paths of tokens behind the root
    for end in order:
        path = ()
        for t in tokens[end:end + each]:
            path += (t,)
            if path not in want:
                if len(want) == max_nodes:
                    break
                want.append(path)
    nodes, parents = look_up(tokens, max_nodes, longest, branches)
    for i in range(1, len(nodes)):
        paths.append(paths[parents[i]] + (nodes[i],))
    assert nodes[0] == tokens[-1] and parents[0] == -1 and paths == want
