"""When a step of beams takes the attention that reads shared pages once."""
import importlib
import math
import tempfile

import pytest
import torch

import replay_util as ru

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
DEV = "cuda:0"


def runner_of(dtype="bfloat16", page_size=16, num_pages=400, max_num_seqs=40, **changes):
    from dispec_b200 import ModelRunner, load_model_config
    from dispec_b200.weights import load_random_model
    model = load_random_model(load_model_config(dict(ru.CONFIG_A, max_position_embeddings=1 << 16, **changes)), 3, 0.05, dtype, DEV)
    return ModelRunner(model, page_size=page_size, num_pages=num_pages, max_num_seqs=max_num_seqs)


def beams_behind(run, tokens, width, name="x"):
    """Requests that have a prompt's pages in common (of which nothing but their number matters here)."""
    run.admit(name)
    run.cache.extend(name, tokens)
    run.cache.commit(name, tokens)
    names = [name] + [(name, i) for i in range(1, width)]
    run.fork([(name, n) for n in names[1:]])
    return names


def shared_calls(run, monkeypatch, groups, tokens):
    """Calls of the attention in one step, one token for each."""
    from dispec_b200 import SeqEntry, ops
    calls = []
    real = ops.shared_prefix_attention
    with monkeypatch.context() as m:
        m.setattr(ops, "shared_prefix_attention", lambda *a, **kw: calls.append(a[1].shape[3]) or real(*a, **kw))
        logits, _ = run.beam_step([[SeqEntry(n, [7], tokens) for n in names] for names in groups], [[0] * len(run.cache.groups) for _ in groups])
    assert torch.isfinite(logits).all()
    return len(calls)


def zeros(run):
    for pools in run.storage.pools:
        for pool in pools.values():
            pool.zero_()


@pytest.mark.parametrize("changes,dtype,page_size,calls", [
    (dict(head_dim=64), "bfloat16", 16, 2), (dict(head_dim=96), "bfloat16", 16, 0), (dict(head_dim=64), "bfloat16", 4, 0),
    (dict(head_dim=24), "bfloat16", 16, 2), (dict(head_dim=96), "float32", 16, 2),
    (dict(head_dim=20), "float32", 16, 0), (dict(head_dim=20), "bfloat16", 16, 0)])
def test_heads_whose_kernel_would_be_the_slower_one(changes, dtype, page_size, calls, monkeypatch):
    from dispec_b200.engine import runner
    monkeypatch.setattr(runner, "SHARED_BYTES", {**runner.SHARED_BYTES, BF16: 1, F32: 1})
    run = runner_of(dtype, page_size, **changes)
    zeros(run)
    assert shared_calls(run, monkeypatch, [beams_behind(run, 100, 4)], 100) == calls


def test_mixers_that_do_not_take_shared_pages_are_not_given_any(monkeypatch):
    from dispec_b200 import SeqEntry
    from dispec_b200.engine import runner
    monkeypatch.setattr(runner, "SHARED_BYTES", {BF16: 1, F32: 1})
    util = importlib.import_module("murutar_util")
    name = sorted(util.CONFIGS)[0]
    with tempfile.TemporaryDirectory() as td:
        util.make_folder(td, name)
        from dispec_b200 import ModelRunner, load_model
        run = ModelRunner(load_model(td, "float32", DEV), page_size=util.CONFIGS[name]["page_size"], num_pages=200, max_num_seqs=4)
    zeros(run)
    seen = []
    real = run.model.forward
    monkeypatch.setattr(run.model, "forward", lambda ctx: seen.append(ctx.shared) or real(ctx))
    names = beams_behind(run, 70, 3)
    run.beam_step([[SeqEntry(n, [5], 70) for n in names]], [[0] * len(run.cache.groups)])
    assert seen == [None]
