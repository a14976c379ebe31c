"""Length penalties by whose power a continuation's length cannot be counted are refused before anything runs."""
import pytest

from dispec_b200.engine.beam import BeamSearchEngine


@pytest.mark.parametrize("penalty,new", [(200.0, 64), (-200.0, 64), (1e300, 2), (-1e300, 2), (1100.0, 2)])
def test_penalties_beyond_numbers(penalty, new):
    engine = object.__new__(BeamSearchEngine)  # (no model: nothing of it is asked)
    with pytest.raises(ValueError, match="length_penalty"):
        engine.generate([[1, 2]], new, length_penalty=penalty)


@pytest.mark.parametrize("penalty,new", [(1e300, 1), (-1e300, 1), (150.0, 64), (-150.0, 64), (0.0, 1 << 20)])
def test_penalties_that_can_be_counted(penalty, new):
    from dispec_b200.engine.beam import Beam, BeamSet
    for length in {1, new}:
        found = BeamSet(1, new, penalty, None, beams=[Beam("x", [5] * (length - 1), -1.0)])
        found._finish([5] * length, -1.0)
        assert found.finished[0].score == -1.0 / length ** penalty

    engine = object.__new__(BeamSearchEngine)
    engine.max_num_seqs, engine.beam_width = 4, 4
    assert engine.generate([], new, length_penalty=penalty) == []
