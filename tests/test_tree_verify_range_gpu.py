"""Verification of drafted trees at the ends of what temperatures and logits may be."""
import pytest
import torch

from test_tree_gpu import verify_case
from tree_util import VerifyCase

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


def follows(case, spec):
    from dispec_b200 import ops
    count, path, token = case.run()
    for s in range(len(spec)):
        case.follow(s, count[s], path[s], token[s])
    assert ops.device_error() == 0
    return count, path, token


# temperatures around and beyond those for which quotients are formed from a reciprocal, with logits that leave the
# quotients between 0.01 and 1,000 or so
@pytest.mark.parametrize("drafted", [False, True])
@pytest.mark.parametrize("vocab", [37, 5003, 40000])
@pytest.mark.parametrize("temperature", [1e-30, 9.2e-10, 9.4e-10, 1e-4, 0.03, 40.0, 1e8, 1.2e9, 1e20])
def test_extreme_temperatures(drafted, vocab, temperature):
    spec = [1, 2, 7, 16]
    case = verify_case(spec, vocab, temperature, drafted, seed=vocab + 1)
    case.logits = (case.logits.double() * temperature).float()
    follows(case, spec)


@pytest.mark.parametrize("drafted", [False, True])
@pytest.mark.parametrize("size", [1e-30, 1e17, 1e19, 1e37])
def test_extreme_logits_at_ordinary_temperatures(drafted, size):
    """A few logits of one size beside ordinary ones: the mass is theirs (or, where the size is small, everybody's)."""
    spec = [5, 9, 3]
    case = verify_case(spec, 500, 0.8, drafted, seed=12)
    case.logits[:, ::50] = size
    follows(case, spec)


@pytest.mark.parametrize("vocab", [70, 9000, 151936])
def test_an_infinite_temperature_shares_the_mass_alike(vocab):
    """Every finite logit has the same mass; where some are infinite, those have it, as at any other temperature."""
    logits = torch.randn(4, vocab, generator=torch.Generator().manual_seed(1))
    logits[0, 3] = -INF
    logits[1, 5] = logits[1, 60] = INF
    logits[2, :] = -INF
    logits[2, 7] = logits[2, 9] = logits[2, 66] = 3.0
    logits[2, 8] = NAN
    logits[3, 61] = INF
    case = VerifyCase([[-1]] * 4, [0] * 4, logits, [INF] * 4, [0.0] * 4, [0.0, 0.9, 0.9, 0.9])
    assert case.run()[2] == [0, 60, 66, 61]
    # the walk: both infinite logits' tokens are drafts
    case = VerifyCase([[-1, 0, 0]], [0, 5, 60], logits[1:2].repeat(3, 1), [INF], [0.0, 0.6, 0.9], [0.2])
    assert case.run() == ([2], [[0, 2, -1]], [5])


@pytest.mark.parametrize("temperature", [0.0, -1.0, -INF, NAN])
def test_what_is_no_temperature_takes_the_largest_logit(temperature):
    logits = torch.zeros(2, 300)
    logits[:, 7] = 1.0
    case = VerifyCase([[-1, 0]], [0, 7], logits, [temperature], [0.999] * 2, [0.999])
    assert case.run() == ([2], [[0, 1]], [7])


@pytest.mark.parametrize("drafted", [False, True])
@pytest.mark.parametrize("vocab", [95000, 188000, 262144, 393216])
@pytest.mark.parametrize("trees", [1, 24])
def test_shares_of_every_size(drafted, vocab, trees):
    """Vocabularies whose shares fit an SM twice, once, and up to the largest."""
    spec = [3] * trees
    case = verify_case(spec, vocab, 0.9, drafted, seed=vocab + trees)
    follows(case, spec)


@pytest.mark.parametrize("drafted", [False, True])
def test_a_vocabulary_beyond_the_largest_is_refused(drafted):
    from dispec_b200 import ops
    case = verify_case([2], 393217, 0.9, drafted, seed=1)
    with pytest.raises(ops.KernelError, match="393216"):
        case.run()
