"""Which mixers read pages that sequences share once for all of them, and by kernels of which arithmetic."""
import importlib

import pytest
import torch

import replay_util as ru

BF16, F32 = torch.bfloat16, torch.float32
FMA = "32 bits for tensor cores"


def mixers(config):
    from dispec_b200 import build_model, load_model_config
    model = build_model(load_model_config(config))
    return [model.layers[call.layer].mixer for call in model.schedule]


@pytest.mark.parametrize("dim,heads,kv_heads,page,dtype,by", [
    (128, 28, 4, 16, BF16, BF16), (64, 16, 4, 8, BF16, BF16), (32, 3, 1, 64, BF16, BF16), (32, 3, 1, 64, F32, F32), (128, 12, 2, 16, F32, F32),
    # single tokens have a tensor-core kernel there, shared pages have none
    (96, 28, 4, 16, BF16, None), (16, 4, 2, 16, BF16, FMA), (256, 8, 8, 16, BF16, FMA), (256, 9, 3, 16, BF16, None),
    (128, 28, 4, 4, BF16, None), (64, 16, 8, 128, BF16, FMA), (64, 16, 16, 24, BF16, FMA),
    # neither has one
    (24, 8, 2, 16, BF16, F32), (8, 4, 2, 16, BF16, F32), (64, 130, 2, 16, BF16, F32), (96, 28, 4, 16, F32, F32),
    # no kernel takes these heads
    (20, 4, 2, 16, F32, None), (20, 4, 2, 16, BF16, None), (12, 4, 2, 8, F32, None), (264, 4, 2, 16, F32, None)])
def test_heads_of_every_kind(dim, heads, kv_heads, page, dtype, by):
    for mixer in mixers(dict(ru.CONFIG_A, head_dim=dim, num_attention_heads=heads, num_key_value_heads=kv_heads)):
        assert mixer.takes_shared(page, dtype) == (by and (by, heads // kv_heads))


def test_what_has_to_be_saved():
    from dispec_b200.engine.runner import FILLED_ROWS, SHARED_BYTES, _least_saved
    assert _least_saved((BF16, 7), BF16, 128, 5) == _least_saved((BF16, 7), BF16, 32, 500) == SHARED_BYTES[BF16]
    assert _least_saved((F32, 1), BF16, 24, 2) == SHARED_BYTES[F32]
    # on FMA units for tensor cores: tiles have to be filled
    filled = _least_saved((FMA, 1), BF16, 128, FILLED_ROWS)
    assert filled == SHARED_BYTES[FMA] == _least_saved((FMA, 2), BF16, 128, 300)
    assert _least_saved((FMA, 1), BF16, 128, FILLED_ROWS / 2) == 16 * filled
    assert _least_saved((FMA, 2), BF16, 32, 300) == filled / 2
    assert _least_saved((FMA, 1), BF16, 96, 5) > 50e9


@pytest.mark.parametrize("family", ["puludra", "murutar", "desalix", "milivik", "bepepel", "pikalorn"])
def test_other_mixers_read_them_for_each(family):
    from dispec_b200.parts.attention import GQAAttention
    util = importlib.import_module(f"{family}_util")
    for name in sorted(util.CONFIGS):
        for mixer in mixers(util.CONFIGS[name]["config"]):
            if type(mixer) is not GQAAttention:
                assert mixer.takes_shared(16, BF16) is None and mixer.takes_shared(16, F32) is None


def test_mixers_that_know_nothing_of_it_and_ones_without_a_cache():
    from types import SimpleNamespace as N
    from dispec_b200.engine.runner import ModelRunner
    takes, states = N(takes_shared=lambda page, dtype: (dtype, page)), N(takes_shared=lambda page, dtype: 1 / 0)
    layers = [N(mixer=m) for m in (takes, N(), states, takes)]
    run = object.__new__(ModelRunner)
    run.cache, run.page_size, run.dtype = N(groups=[0, 1, 2]), 16, BF16
    run.model = N(schedule=[N(layer=i) for i in (0, 1, 2, 3)], layers=layers, call_cache=[0, 1, None, 2],
                  placement={0: N(group=0), 1: N(group=1), 2: N(group=0)})
    assert run._shared_by == [{(BF16, 16)}, set(), set()]
