"""Steps over drafted trees: logits at every node, the accepted branch in the cache, and tokens that are the model's own."""
import random
import subprocess
import sys
import tempfile

import pytest
import torch

import plain_qwen2 as plain
import replay_util as ru
from tree_util import random_tree

pytestmark = pytest.mark.gpu


def runner_for(folder, name, dtype, **kw):
    from dispec_b200 import ModelRunner, load_model
    return ModelRunner(load_model(folder, dtype, "cuda:0"), page_size=ru.TINY[name]["page_size"], num_pages=256, max_num_seqs=16,
                       poison=True, **kw)


def branch(parents, node):
    out = []
    while node >= 0:
        out.append(node)
        node = parents[node]
    return out[::-1]


@pytest.mark.parametrize("name", ["a", "b", "c", "d", "e"])
def test_logits_at_every_node_and_behind_the_kept_branch(name):
    from dispec_b200 import SeqEntry, TreeEntry
    from dispec_b200.ops.tree import Verified
    rng = random.Random(len(name) + ord(name))
    with tempfile.TemporaryDirectory() as td:
        config, weights = ru.make_model_folder(td, name, dtype="float32")
        run = runner_for(td, name, "float32")
        vocab = config["vocab_size"]
        prompts = [ru.random_ids(n, vocab, n) for n in (1, 70, 33, 16)]
        trees = [random_tree(n, rng) for n in (9, 1, 30, 70)]
        entries, kept = [], []
        for i, (p, t) in enumerate(zip(prompts, trees)):
            run.admit(i)
            run.step([SeqEntry(i, p, 0, [])])
            entries.append(TreeEntry(i, ru.random_ids(len(t), vocab, 100 + i), t, len(p)))
        ctx, logits = run.tree_step(entries)
        row = 0
        for e, p in zip(entries, prompts):
            for node in range(len(e.tokens)):
                if node % 7 == 0 or node == len(e.tokens) - 1:
                    path = branch(e.parents, node)
                    want = plain.forward_logits(weights, config, p + [e.tokens[k] for k in path])[-1]
                    assert (logits[row + node].cpu() - want).abs().max() <= 1e-4
            row += len(e.tokens)
        # keep the branch of some node of each tree, and go on behind it
        paths = [branch(e.parents, rng.randrange(len(e.tokens))) for e in entries]
        width = max(len(t) for t in trees)
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda:0")
        run.move_accepted(ctx, Verified(i32([len(p) for p in paths]), i32([(p + [-1] * width)[:width] for p in paths]), None))
        run.keep(entries, [len(p) for p in paths])
        run.cache.check()
        steps = [SeqEntry(i, [3], len(prompts[i]) + len(paths[i]), [0]) for i in range(4)]
        logits = run.step(steps)
        for i, e in enumerate(entries):
            want = plain.forward_logits(weights, config, prompts[i] + [e.tokens[k] for k in paths[i]] + [3])[-1]
            assert (logits[i].cpu() - want).abs().max() <= 1e-4
        run.check_device()


@pytest.mark.parametrize("name", ["a", "b", "c", "e"])
@pytest.mark.parametrize("max_nodes", [1, 5, 16])
def test_greedy_tokens_are_the_models_own(name, max_nodes):
    from dispec_b200 import KVConfig, SpeculativeEngine, load_model
    with tempfile.TemporaryDirectory() as td:
        config, weights = ru.make_model_folder(td, name, dtype="float32")
        engine = SpeculativeEngine(load_model(td, "float32", "cuda:0"), KVConfig(block_size=ru.TINY[name]["page_size"]), num_blocks=128,
                                   max_nodes=max_nodes)
        base = ru.random_ids(12, config["vocab_size"], 3)
        prompts = [base * 3, base[:5] + base[:5], [7]]
        got = engine.generate(prompts, 24)
        for p, g in zip(prompts, got):
            want, gaps = plain.greedy_generate(weights, config, p, 24)
            n = next((i for i, gap in enumerate(gaps) if gap < 1e-3), len(want))
            assert len(g) == 24 and g[:n] == want[:n]
        assert engine.num_accepted >= engine.num_steps and not engine.runner.cache.live_requests()
        engine.runner.cache.check()


def test_drafts_are_accepted_where_a_request_repeats_itself():
    """A greedy tiny model soon repeats itself; then the looked-up drafts are right and a step gives several tokens."""
    from dispec_b200 import SpeculativeEngine, load_model
    with tempfile.TemporaryDirectory() as td:
        config, _ = ru.make_model_folder(td, "a", dtype="float32")
        engine = SpeculativeEngine(load_model(td, "float32", "cuda:0"), num_blocks=128, max_nodes=16)
        out = engine.generate([[5, 17, 3]], 96)[0]
        assert len(out) == 96 and engine.num_steps < 95


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_sampled_tokens_are_reproducible_and_stop(dtype):
    from dispec_b200 import SamplingParams, SpeculativeEngine, load_model
    with tempfile.TemporaryDirectory() as td:
        config, _ = ru.make_model_folder(td, "e", dtype=dtype)
        engine = SpeculativeEngine(load_model(td, dtype, "cuda:0"), num_blocks=128, max_nodes=8)
        prompts = [ru.random_ids(20, config["vocab_size"], 1) * 2, ru.random_ids(5, config["vocab_size"], 2)]
        params = [SamplingParams(0.9, seed=4), SamplingParams(0.0)]
        first = engine.generate(prompts, 20, params)
        assert first == engine.generate(prompts, 20, params)
        eos = first[0][7]
        stopped = engine.generate(prompts, 20, params, eos_token_id=eos)[0]
        assert stopped == first[0][:first[0].index(eos) + 1]


def test_refusals():
    from dispec_b200 import SamplingParams, SpeculativeEngine, TreeEntry, load_model
    with tempfile.TemporaryDirectory() as td:
        config, _ = ru.make_model_folder(td, "a", dtype="float32")
        engine = SpeculativeEngine(load_model(td, "float32", "cuda:0"), num_blocks=16)
        for bad in (dict(params=SamplingParams(1.0, top_k=3)), dict(params=SamplingParams(1.0, top_p=0.5)), dict(params=[])):
            with pytest.raises(ValueError):
                engine.generate([[1, 2]], 4, **bad)
        with pytest.raises(ValueError):
            engine.generate([[]], 4)
        with pytest.raises(ValueError):
            SpeculativeEngine(engine.runner.model, num_blocks=16, max_nodes=0)
        run = engine.runner
        run.admit("r")
        for e in (TreeEntry("r", [1], [-1], 3), TreeEntry("r", [1, 2], [-1], 0), TreeEntry("r", [1, 2], [-1, 1], 0),
                  TreeEntry("r", [], [], 0), TreeEntry("r", [1, 256], [-1, 0], 0)):
            with pytest.raises(ValueError):
                run.tree_step([e])
        with pytest.raises(KeyError):
            run.tree_step([TreeEntry("s", [1], [-1], 0)])
        with pytest.raises(ValueError):
            run.tree_step([])
        run.model.layers[0].mixer.takes_trees = False
        with pytest.raises(ValueError, match="drafted trees"):
            run.tree_step([TreeEntry("r", [1], [-1], 0)])


def test_command_line():
    with tempfile.TemporaryDirectory() as td:
        ru.make_model_folder(td, "b")
        run = subprocess.run([sys.executable, "-m", "dispec_b200", "speculate", "--model", td, "--prompt-ids", "5,17,3,5,17,3", "--max-new",
                              "9", "--max-nodes", "6", "--num-blocks", "64"], cwd=ru.ROOT, capture_output=True, text=True, timeout=300)
        assert run.returncode == 0, run.stderr
        assert '"output_ids"' in run.stdout and "tokens a step" in run.stderr
