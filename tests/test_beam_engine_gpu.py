"""Beam search against a search over the plain implementations' logits, one whole forward pass per beam and step."""
import importlib
import subprocess
import sys
import tempfile

import pytest
import torch

import plain_qwen2
import replay_util as ru

pytestmark = pytest.mark.gpu
FAMILIES = ["puludra", "murutar", "desalix", "milivik", "bepepel", "pikalorn"]


def search(logits_of, prompt, width, max_new, penalty, eos):
    """[(tokens, score)], the best first."""
    beams, finished = [([], 0.0)], []
    for length in range(1, max_new + 1):
        candidates = []
        for i, (tokens, total) in enumerate(beams):
            log_p = torch.log_softmax(logits_of(prompt + tokens).double(), -1)
            best = torch.topk(log_p, min(2 * width, log_p.numel()))
            candidates += [(total + float(v), -i, -int(t)) for v, t in zip(best.values, best.indices)]
        candidates = sorted(candidates, reverse=True)[:2 * width]
        going = []
        for rank, (total, i, t) in enumerate(candidates):
            tokens = beams[-i][0] + [-t]
            if -t == eos:
                if rank < width:
                    finished.append((tokens, total / length ** penalty))
            elif len(going) < width:
                going.append((tokens, total))
        finished = sorted(finished, key=lambda h: -h[1])[:width]
        if length == max_new:
            finished += [(tokens, total / length ** penalty) for tokens, total in going]
        elif len(finished) == width and going[0][1] / length ** penalty <= finished[-1][1]:
            break
        beams = going
    return sorted(finished, key=lambda h: -h[1])[:width]


def log_probability(logits_of, prompt, tokens):
    return sum(float(torch.log_softmax(logits_of(prompt + tokens[:i]).double(), -1)[t]) for i, t in enumerate(tokens))


def check(engine, logits_of, prompts, width, max_new, penalty, eos, tolerance):
    got = engine.generate(prompts, max_new, penalty, eos, num_return=width)
    cache = engine.runner.cache
    cache.check()
    assert cache.live_requests() == []
    for prompt, found in zip(prompts, got):
        want = search(logits_of, prompt, width, max_new, penalty, eos)
        assert len(found) == len(want)
        for h, (tokens, score) in zip(found, want):
            # equally good continuations may change places, others not
            assert abs(h.score - score) <= tolerance and len(h.tokens) <= max_new
            own = log_probability(logits_of, prompt, h.tokens) / len(h.tokens) ** penalty
            assert abs(own - h.score) <= tolerance
        assert len({tuple(h.tokens) for h in found}) == len(found)
        assert all(a.score >= b.score for a, b in zip(found, found[1:]))


def engine_for(folder, dtype, page_size, width, **kw):
    from dispec_b200 import BeamSearchEngine, KVConfig, load_model
    engine = BeamSearchEngine(load_model(folder, dtype, "cuda:0"), KVConfig(block_size=page_size), num_blocks=400, beam_width=width,
                              **{"max_num_seqs": 3 * width, **kw})
    engine.runner.poison = True  # pages that nobody holds are NaN
    return engine


@pytest.fixture
def always_shared(monkeypatch):
    """The attention of shared pages wherever there are some, however few."""
    from dispec_b200.engine import runner
    monkeypatch.setattr(runner, "SHARED_BYTES", {torch.bfloat16: 1, torch.float32: 1})


@pytest.mark.parametrize("name", ["a", "b", "c", "d", "e"])
@pytest.mark.parametrize("width,penalty,eos", [(1, 1.0, None), (4, 1.0, None), (3, 0.6, 7), (5, 0.0, None)])
def test_the_found_continuations_are_those_of_the_plain_search(name, width, penalty, eos, always_shared):
    with tempfile.TemporaryDirectory() as td:
        config, weights = ru.make_model_folder(td, name, dtype="float32")
        engine = engine_for(td, "float32", ru.TINY[name]["page_size"], width)
        prompts = [ru.random_ids(n, config["vocab_size"], n) for n in (1, 31, 48)]
        logits_of = lambda ids: plain_qwen2.forward_logits(weights, config, ids)[-1]
        # a sum of ten log-probabilities, each from logits that are off by up to 1e-4 (as the tests of steps have it)
        check(engine, logits_of, prompts, width, 10, penalty, eos, 2e-3)
        assert engine.num_steps == 9 or eos is not None


def test_an_end_token_that_is_likely():
    """Searches that end early, and beams that end while others go on."""
    with tempfile.TemporaryDirectory() as td:
        config, weights = ru.make_model_folder(td, "a", dtype="float32")
        engine = engine_for(td, "float32", ru.TINY["a"]["page_size"], 4)
        logits_of = lambda ids: plain_qwen2.forward_logits(weights, config, ids)[-1]
        prompts = [ru.random_ids(n, config["vocab_size"], n) for n in (20, 5)]
        likely = int(logits_of(prompts[0] + [int(logits_of(prompts[0]).argmax())]).argmax())
        check(engine, logits_of, prompts, 4, 8, 1.0, likely, 2e-3)


@pytest.mark.parametrize("family", FAMILIES)
def test_other_families_keep_their_states_and_pages(family, always_shared):
    """Recurrent states, windows, latents and chunks follow their beams: the same search with one whole pass per beam."""
    from dispec_b200 import SeqEntry
    util = importlib.import_module(f"{family}_util")
    name = "mix" if "mix" in util.CONFIGS else sorted(util.CONFIGS)[0]
    with tempfile.TemporaryDirectory() as td:
        util.make_folder(td, name)
        engine = engine_for(td, "float32", util.CONFIGS[name]["page_size"], 3, max_num_seqs=10)
        run, vocab = engine.runner, engine.runner.vocab_size

        def logits_of(ids):
            run.admit("plain")
            out = run.step([SeqEntry("plain", ids, 0, [len(ids) - 1])])[0].cpu()
            run.release("plain")
            return out

        prompts = [ru.random_ids(n, vocab, n) for n in (3, 40)]
        check(engine, logits_of, prompts, 3, 9, 1.0, None, 2e-3)


def test_bfloat16_scores_are_the_models_own(always_shared):
    with tempfile.TemporaryDirectory() as td:
        config, weights = ru.make_model_folder(td, "c", dtype="bfloat16")
        engine = engine_for(td, "bfloat16", ru.TINY["c"]["page_size"], 4)
        prompts = [ru.random_ids(n, config["vocab_size"], n) for n in (70, 9)]
        got = engine.generate(prompts, 12, num_return=4)
        logits_of = lambda ids: plain_qwen2.forward_logits(weights, config, ids)[-1]
        for prompt, found in zip(prompts, got):
            assert len(found) == 4 and all(len(h.tokens) == 12 for h in found)
            for h in found:
                # logits are off by up to 5e-2 in bfloat16, as the tests of steps have it; a mean of twelve log-probabilities, each
                # off by twice as much
                assert abs(log_probability(logits_of, prompt, h.tokens) / 12 - h.score) <= 0.1


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_shared_pages_are_read_once_a_prompt(dtype, monkeypatch):
    """The attention of shared pages is called in every layer of every step whose beams share enough."""
    from dispec_b200 import ops
    from dispec_b200.engine import runner
    calls = []
    real = ops.shared_prefix_attention
    monkeypatch.setattr(ops, "shared_prefix_attention", lambda *a, **kw: calls.append(a[6].tolist()) or real(*a, **kw))
    with tempfile.TemporaryDirectory() as td:
        config, _ = ru.make_model_folder(td, "a", dtype=dtype)
        engine = engine_for(td, dtype, 16, 4)
        prompts = [ru.random_ids(100, config["vocab_size"], 1), ru.random_ids(40, config["vocab_size"], 2)]
        engine.generate(prompts, 5)
        assert not calls  # (not worth it)
        monkeypatch.setattr(runner, "SHARED_BYTES", {torch.bfloat16: 1, torch.float32: 1})
        engine.generate(prompts, 5)
        layers = config["num_hidden_layers"]
        assert len(calls) == 4 * layers and all(c == [96, 32] for c in calls)
        calls.clear()
        engine.generate([ru.random_ids(7, config["vocab_size"], 1)], 5)  # no page is full
        assert not calls


def test_more_prompts_than_fit_at_once_and_again():
    with tempfile.TemporaryDirectory() as td:
        config, _ = ru.make_model_folder(td, "a", dtype="float32")
        engine = engine_for(td, "float32", ru.TINY["a"]["page_size"], 4, max_num_seqs=9)
        prompts = [ru.random_ids(n, config["vocab_size"], n) for n in (9, 17, 33, 2, 40)]
        one = [engine.generate([p], 7, num_return=2)[0] for p in prompts]
        together = engine.generate(prompts, 7, num_return=2)
        for a, b in zip(one, together):
            assert [h.tokens for h in a] == [h.tokens for h in b]
        assert engine.generate(prompts, 0) == [[]] * 5 and engine.generate([], 5) == []


def test_beams_of_width_one_are_the_greedy_tokens():
    from dispec_b200 import LLMEngine, SamplingParams
    with tempfile.TemporaryDirectory() as td:
        config, _ = ru.make_model_folder(td, "a", dtype="float32")
        engine = engine_for(td, "float32", ru.TINY["a"]["page_size"], 1)
        prompt = ru.random_ids(21, config["vocab_size"], 3)
        greedy = LLMEngine(engine.runner.model).generate(prompt, 12, SamplingParams())
        assert engine.generate([prompt], 12)[0][0].tokens == greedy


def test_a_pool_too_small_raises_and_leaves_nothing_behind():
    from dispec_b200 import BeamSearchEngine, KVConfig, load_model
    from dispec_b200.cache import OutOfPagesError
    with tempfile.TemporaryDirectory() as td:
        config, _ = ru.make_model_folder(td, "a", dtype="float32")
        engine = BeamSearchEngine(load_model(td, "float32", "cuda:0"), KVConfig(block_size=16), num_blocks=6, beam_width=4)
        with pytest.raises(OutOfPagesError):
            engine.generate([ru.random_ids(40, config["vocab_size"], 1)], 60)
        engine.runner.cache.check()
        assert engine.runner.cache.live_requests() == []
        assert len(engine.generate([[1, 2, 3]], 4)[0]) == 1


def test_forks_of_which_one_cannot_be_take_nothing():
    from dispec_b200 import SeqEntry
    with tempfile.TemporaryDirectory() as td:
        ru.make_model_folder(td, "a", dtype="float32")
        run = engine_for(td, "float32", 16, 2).runner
        run.admit("x")
        run.step([SeqEntry("x", list(range(40)), 0, [])])
        for pairs, error in (([("x", "y"), ("x", "y")], ValueError), ([("x", "y"), ("z", "w")], KeyError)):
            with pytest.raises(error):
                run.fork(pairs)
            run.cache.check()
            assert run.cache.live_requests() == ["x"]
        run.fork([("x", "y"), ("y", "z")])
        run.cache.check()
        logits, _ = run.beam_step([[SeqEntry(r, [7], 40) for r in "xyz"]], [[0]])
        assert torch.equal(logits[0], logits[1]) and torch.equal(logits[0], logits[2])


def test_refusals():
    from dispec_b200 import SeqEntry
    with tempfile.TemporaryDirectory() as td:
        ru.make_model_folder(td, "a", dtype="float32")
        engine = engine_for(td, "float32", 16, 2)
        with pytest.raises(ValueError):
            engine.generate([[]], 4)
        with pytest.raises(ValueError):
            engine.generate([[1]], 4, length_penalty=float("nan"))
        run = engine.runner
        run.admit("x")
        run.step([SeqEntry("x", [1, 2, 3], 0, [])])
        for groups in ([], [[]], [[SeqEntry("x", [1, 2], 3)]], [[SeqEntry("x", [1], 2)]], [[SeqEntry("x", [1], 3)], [SeqEntry("x", [1], 3)]]):
            with pytest.raises(ValueError):
                run.beam_step(groups, [[0]] * len(groups))
        with pytest.raises(KeyError):
            run.beam_step([[SeqEntry("y", [1], 0)]], [[0]])


def test_the_command_prints_the_best_continuations():
    import json
    with tempfile.TemporaryDirectory() as td:
        config, _ = ru.make_model_folder(td, "a", dtype="float32")
        cmd = [sys.executable, "-m", "dispec_b200", "beam", "--model", td, "--dtype", "float32", "--prompt-ids", "5,17,3", "--prompt-ids", "9",
               "--max-new", "5", "--width", "3", "--num-return", "2"]
        done = subprocess.run(cmd, capture_output=True, text=True, cwd=ru.ROOT, timeout=300)
        assert done.returncode == 0, done.stderr
        lines = [json.loads(x) for x in done.stdout.splitlines()]
        assert [x["id"] for x in lines] == [0, 0, 1, 1] and all(len(x["output_ids"]) == 5 for x in lines)
