"""Drafts looked up in a request's own tokens."""
from dispec_b200.engine.speculative import look_up


def test_nothing_to_look_up():
    assert look_up([5], 8) == ([5], [-1])
    assert look_up([1, 2, 3, 4], 8) == ([4], [-1])
    assert look_up([1, 2, 1], 1) == ([1], [-1])


def test_a_repeated_tail_drafts_what_followed_it():
    tokens = [1, 2, 3, 4, 5, 9, 1, 2, 3]
    assert look_up(tokens, 5, branches=1) == ([3, 4, 5, 9, 1], [-1, 0, 1, 2, 3])


def test_continuations_share_their_beginning():
    tokens = [7, 1, 2, 3, 7, 1, 2, 4, 7]
    nodes, parents = look_up(tokens, 16, longest=1, branches=2)
    assert nodes == [7, 1, 2, 4, 7, 3] or (nodes[:4] == [7, 1, 2, 4] and 3 in nodes)
    for i, p in enumerate(parents):
        assert -1 <= p < i or i == 0
    paths = set()
    for i in range(len(nodes)):
        path, k = [], i
        while k >= 0:
            path.append(nodes[k])
            k = parents[k]
        paths.add(tuple(path[::-1]))
    assert (7, 1, 2, 4) in paths and (7, 1, 2, 3) in paths and len(paths) == len(nodes)


def test_a_tree_never_has_more_nodes_than_asked():
    tokens = [1, 2] * 30
    for n in range(1, 20):
        nodes, parents = look_up(tokens, n)
        assert 1 <= len(nodes) <= n and len(nodes) == len(parents) and nodes[0] == 2
