"""Forked requests in the cache manager, and what the host keeps of a beam search."""
import random

import pytest

from dispec_b200.cache import CacheGroupSpec, CacheManager, OutOfPagesError, OutOfSlotsError
from dispec_b200.engine.beam import Beam, BeamSet


def manager(pages=40, slots=8, window=0, page_size=4, groups=1):
    return CacheManager([CacheGroupSpec.key_value(2, 16, window=window) for _ in range(groups)], page_size=page_size, num_pages=pages,
                        max_num_seqs=slots)


def grow(m, r, n):
    m.extend(r, n)
    return m.commit(r, n)


@pytest.mark.parametrize("tokens", [0, 1, 3, 4, 7, 8, 13])
def test_a_fork_shares_filled_pages_and_copies_the_last_one(tokens):
    m = manager()
    m.admit("a")
    if tokens:
        grow(m, "a", tokens)
    slot, copies = m.fork("a", "b")
    full, rest = divmod(tokens, 4)
    a, b = m.block_table("a"), m.block_table("b")
    assert slot != m.state_slot("a") and m.num_tokens("b") == tokens
    assert a[:full] == b[:full] and len(copies) == (rest > 0) and m.shared_pages(["a", "b"]) == full
    if rest:
        assert copies == [(0, a[full], b[full])] and a[full] != b[full]
    m.check()
    grow(m, "a", tokens + 5)
    grow(m, "b", tokens + 5)
    assert m.shared_pages(["a", "b"]) == full
    m.check()
    freed = {p for _, p in m.free("a")}
    assert freed.isdisjoint(b[:full])
    m.check()
    m.free("b")
    assert m.num_free_pages() == 40
    m.check()


def test_window_pages_go_back_when_nobody_reads_them():
    m = manager(window=6)
    m.admit("a")
    grow(m, "a", 12)
    m.fork("a", "b")
    m.check()
    shared = [p for p in m.block_table("a") if p >= 0]
    assert grow(m, "a", 16) == []  # the other one still has it
    m.check()
    assert {p for _, p in grow(m, "b", 16)} <= set(shared)
    m.check()
    assert m.shared_pages(["a", "b"]) == 3  # given back in both


def test_forks_that_are_refused_take_nothing():
    m = manager(pages=3, slots=2, groups=2)
    m.admit("a")
    grow(m, "a", 9)
    with pytest.raises(OutOfPagesError):
        m.fork("a", "b")
    m.check()
    with pytest.raises(ValueError):
        m.fork("a", "a")
    m = manager(slots=1)
    m.admit("a")
    with pytest.raises(OutOfSlotsError):
        m.fork("a", "b")
    m = manager()
    m.admit("a", prompt_len=9)
    with pytest.raises(ValueError, match="promises"):
        m.fork("a", "b")
    m.check()


def test_random_forks_and_ends():
    rng = random.Random(0)
    for window in (0, 9):
        m = manager(pages=200, slots=16, window=window, groups=2)
        live, lens = [], {}
        for step in range(600):
            what = rng.random()
            if not live or (what < 0.1 and len(live) < 16):
                m.admit(step)
                live.append(step)
                lens[step] = 0
            elif what < 0.35 and len(live) < 16:
                of = rng.choice(live)
                m.fork(of, step)
                live.append(step)
                lens[step] = lens[of]
            elif what < 0.5:
                m.free(live.pop(rng.randrange(len(live))))
            else:
                r = rng.choice(live)
                lens[r] += rng.randint(1, 6)
                if m.can_extend(r, lens[r]) and lens[r] < 60:
                    grow(m, r, lens[r])
                else:
                    lens[r] = m.num_tokens(r)
            m.check()


def beams(*of):
    return [Beam(i, tokens, total) for i, (tokens, total) in enumerate(of)]


def test_the_best_that_do_not_end_go_on():
    s = BeamSet(2, 10, 1.0, eos=9, beams=beams(([4], -1.0), ([5], -2.0)))
    going = s.advance([(0, 9, -1.5), (0, 3, -1.6), (1, 9, -2.5), (1, 2, -3.0)])
    assert going == [(0, 3, -1.6), (1, 2, -3.0)] and not s.done
    # the end behind the first two candidates is not taken
    assert [(h.tokens, h.score) for h in s.finished] == [([4, 9], -0.75)]


def test_done_when_nothing_can_be_ranked_before_what_is_finished():
    s = BeamSet(1, 10, 0.0, eos=9, beams=beams(([4], -1.0)))
    assert s.advance([(0, 9, -1.1), (0, 3, -1.2)]) == [] and s.done
    s = BeamSet(1, 10, 2.0, eos=9, beams=beams(([4], -1.0)))
    assert s.advance([(0, 3, -1.2), (0, 9, -1.1)]) == [(0, 3, -1.2)] and not s.done


def test_beams_as_long_as_they_may_be_are_finished():
    s = BeamSet(2, 2, 1.0, eos=9, beams=beams(([4], -1.0), ([5], -2.0)))
    assert s.advance([(1, 7, -2.5), (0, 3, -2.6), (0, 9, -3.0)]) == [] and s.done
    assert [(h.tokens, h.score) for h in s.finished] == [([5, 7], -1.25), ([4, 3], -1.3)]


def test_fewer_candidates_than_beams_and_none():
    s = BeamSet(3, 9, 1.0, eos=None, beams=beams(([4], -1.0)))
    assert s.advance([(0, 1, -1.5)]) == [(0, 1, -1.5)] and not s.done
    assert s.advance([]) == [] and s.done and s.finished == []


def test_refused_arguments():
    from dispec_b200.engine.beam import BeamSearchEngine
    for kw in (dict(beam_width=0), dict(beam_width=129, max_num_seqs=200), dict(beam_width=8, max_num_seqs=7)):
        with pytest.raises(ValueError):
            BeamSearchEngine(None, **kw)
