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
    (dict(head_dim=96, num_attention_heads=6), "bfloat16", 16, 0),
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


@pytest.mark.parametrize("dtype,tokens,width,chain,calls", [
    # 4,096 bytes a token and layer; 150 MB have to be saved
    ("bfloat16", 16384, 2, True, 0), ("bfloat16", 16384, 2, False, 0), ("bfloat16", 16384, 4, False, 2),
    ("bfloat16", 16384, 3, False, 0),
    # and where the layers otherwise run behind one call, 600 MB read, at 1.4 times their size
    ("bfloat16", 16384, 4, True, 0), ("bfloat16", 16384, 6, True, 0), ("bfloat16", 16384, 7, True, 2),
    # 8,192 bytes a token and layer; half a megabyte
    ("float32", 63, 2, False, 0), ("float32", 64, 2, False, 2), ("float32", 16, 4, False, 0), ("float32", 32, 4, False, 2)])
def test_on_both_sides_of_the_thresholds(dtype, tokens, width, chain, calls, monkeypatch):
    run = runner_of(dtype, num_pages=1100, head_dim=128, num_attention_heads=8, num_key_value_heads=8)
    assert run.model.dense_chain == (dtype == "bfloat16")
    run.model.dense_chain = chain
    zeros(run)
    assert shared_calls(run, monkeypatch, [beams_behind(run, tokens, width)], tokens) == calls


def test_windows_count_what_they_let_through(monkeypatch):
    """Of 16,384 shared tokens a layer with a window of 1,000 reads a sixteenth: not worth it, beside a full layer that is."""
    run = runner_of(num_pages=1100, head_dim=128, num_attention_heads=8, num_key_value_heads=8, use_sliding_window=True, sliding_window=1000,
                    max_window_layers=1, layer_types=["full_attention", "sliding_attention"])
    assert len(run.cache.groups) == 2
    run.model.dense_chain = False
    zeros(run)
    assert shared_calls(run, monkeypatch, [beams_behind(run, 16384, 8)], 16384) == 1


def test_the_same_logits_either_way(monkeypatch):
    """Above the threshold and below it, in 32 bits."""
    from dispec_b200 import SeqEntry
    from dispec_b200.engine import runner
    run = runner_of("float32", head_dim=128, num_attention_heads=8, num_key_value_heads=8)
    gen = torch.Generator(device=DEV).manual_seed(1)
    for pools in run.storage.pools:
        for pool in pools.values():
            pool.normal_(generator=gen)
    groups = [beams_behind(run, n, 5, name=f"g{n}") for n in (300, 1000)]
    others = [[(n, "other") for n in names] for names in groups]
    run.fork([(n, o) for names, more in zip(groups, others) for n, o in zip(names, more)])
    step = lambda of: run.beam_step([[SeqEntry(n, [3 + i], at) for i, n in enumerate(names)] for names, at in zip(of, (300, 1000))],
                                    [[0]] * 2)[0]
    got = step(groups)
    monkeypatch.setattr(runner, "SHARED_BYTES", {F32: math.inf})
    want = step(others)
    # logits of tiny models are off by up to 1e-4 in 32 bits, as the tests of steps have it
    assert not torch.equal(got, want) and (got - want).abs().max() <= 1e-4 * max(1.0, float(want.abs().max()))


def test_sixteen_rows_of_heads_without_a_kernel_on_tensor_cores(monkeypatch):
    """8 heads of 96: 3,072 bytes a token and layer, of which 520 MB have to be saved, by groups that fill tiles of rows."""
    run = runner_of(num_pages=1100, head_dim=96, num_attention_heads=8, num_key_value_heads=8, max_num_seqs=60)
    zeros(run)
    names = beams_behind(run, 16384, 16)
    assert shared_calls(run, monkeypatch, [names], 16384) == 2   # 755 MB
    few = beams_behind(run, 96, 11, "few")
    assert shared_calls(run, monkeypatch, [names[:11]], 16385) == 0  # 503 MB
    assert shared_calls(run, monkeypatch, [[n] for n in few], 96) == 0


@pytest.mark.parametrize("first", [0, 1])
def test_sequences_of_different_lengths_behind_a_window(first, monkeypatch):
    """The longer one has given back pages that the shorter one reads, and that were known to be shared."""
    from dispec_b200 import SeqEntry, ops
    from dispec_b200.engine import runner
    monkeypatch.setattr(runner, "SHARED_BYTES", {F32: 1})
    run = runner_of("float32", head_dim=32, use_sliding_window=True, sliding_window=40, max_window_layers=1,
                    layer_types=["full_attention", "sliding_attention"])
    gen = torch.Generator(device=DEV).manual_seed(2)
    for pools in run.storage.pools:
        for pool in pools.values():
            pool.normal_(generator=gen)
    names = beams_behind(run, 64, 2)
    known = [[0, 0]]
    run.beam_step([[SeqEntry(n, [5], 64) for n in names]], known)
    assert known == [[4, 4]]
    at = [130, 70]  # the window begins at 91 and 31
    for n, length in zip(names, at):
        run.cache.extend(n, length)
        run.cache.commit(n, length)
    others = [(n, "other") for n in names]
    run.fork(list(zip(names, others)))
    entries = lambda of: [SeqEntry(of[i], [7 + i], at[i]) for i in (first, 1 - first)]
    got = run.beam_step([entries(names)], known)[0]
    monkeypatch.setattr(runner, "SHARED_BYTES", {F32: math.inf})
    want = run.beam_step([entries(others)], [[0, 0]])[0]
    assert ops.device_error() == 0 and (got - want).abs().max() <= 1e-4 * max(1.0, float(want.abs().max()))
