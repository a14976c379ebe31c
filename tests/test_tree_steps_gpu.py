"""Steps over drafted trees with the tensor-core kernels, against the plain decoder; and the distribution of an engine's tokens."""
import json
import os
import random

import pytest
import torch

import plain_qwen2 as plain
import replay_util as ru
from test_engine_gpu import assert_tokens_within_margin
from test_speculative_gpu import branch
from tree_util import random_tree

pytestmark = pytest.mark.gpu

# head size 128, a group of six, one layer with a window
CONFIG_128 = dict(architectures=["Qwen2ForCausalLM"], model_type="qwen2", num_hidden_layers=2, hidden_size=96, num_attention_heads=12,
                  num_key_value_heads=2, head_dim=128, intermediate_size=160, vocab_size=260, rope_theta=10000.0, rms_norm_eps=1e-6,
                  hidden_act="silu", tie_word_embeddings=True, max_position_embeddings=2048, use_sliding_window=True, sliding_window=90,
                  layer_types=["full_attention", "sliding_attention"])


def model_folder(folder, name, dtype):
    """(config, weights, page size); the bounds for bfloat16 are those of the replayed traces."""
    if name != "h128":
        return ru.make_model_folder(folder, name, dtype=dtype) + (ru.TINY[name]["page_size"],)
    from safetensors.torch import load_file

    from dispec_b200.config import load_model_config
    from dispec_b200.weights import write_random_model
    write_random_model(load_model_config(CONFIG_128), folder, seed=3, std=0.05, dtype=dtype)
    with open(os.path.join(folder, "config.json")) as f:
        config = json.load(f)
    return config, {k: v.float() for k, v in load_file(os.path.join(folder, "model.safetensors")).items()}, 16


def near(got, want, dtype):
    error, scale = (got.cpu() - want).abs().max().item(), max(want.abs().max().item(), 1e-3)
    assert error <= (1e-4 if dtype == "float32" else 0.03 * scale + 0.02), (error, scale)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("name", ["e", "h128"])
def test_logits_at_every_node_and_behind_the_kept_branch(name, dtype, tmp_path):
    from dispec_b200 import ModelRunner, SeqEntry, TreeEntry, load_model
    from dispec_b200.ops.tree import Verified
    rng = random.Random(8)
    config, weights, page = model_folder(str(tmp_path), name, dtype)
    run = ModelRunner(load_model(str(tmp_path), dtype, "cuda:0"), page_size=page, num_pages=256, max_num_seqs=16, poison=True)
    vocab = config["vocab_size"]
    prompts = [ru.random_ids(n, vocab, n) for n in (1, 130, 33, 64)]
    trees = [random_tree(n, rng) for n in (9, 12, 70, 1)]
    entries = []
    for i, (p, t) in enumerate(zip(prompts, trees)):
        run.admit(i)
        run.step([SeqEntry(i, p, 0, [])])
        entries.append(TreeEntry(i, ru.random_ids(len(t), vocab, 100 + i), t, len(p)))
    ctx, logits = run.tree_step(entries)
    row = 0
    for e, p in zip(entries, prompts):
        for node in range(len(e.tokens)):
            if node % 5 == 0 or node == len(e.tokens) - 1:
                near(logits[row + node], plain.forward_logits(weights, config, p + [e.tokens[k] for k in branch(e.parents, node)])[-1], dtype)
        row += len(e.tokens)
    paths = [branch(e.parents, rng.randrange(len(e.tokens))) for e in entries]
    width = max(len(t) for t in trees)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda:0")
    run.move_accepted(ctx, Verified(i32([len(p) for p in paths]), i32([(p + [-1] * width)[:width] for p in paths]), None))
    run.keep(entries, [len(p) for p in paths])
    logits = run.step([SeqEntry(i, [3], len(prompts[i]) + len(paths[i]), [0]) for i in range(4)])
    for i, e in enumerate(entries):
        near(logits[i], plain.forward_logits(weights, config, prompts[i] + [e.tokens[k] for k in paths[i]] + [3])[-1], dtype)
    run.check_device()


@pytest.mark.parametrize("name", ["e", "h128"])
def test_greedy_tokens_in_bfloat16(name, tmp_path):
    """Every token, behind those before it: the plain decoder's, or closer to it than bfloat16 resolves."""
    from dispec_b200 import KVConfig, SamplingParams, SpeculativeEngine, load_model
    config, weights, page = model_folder(str(tmp_path), name, "bfloat16")
    engine = SpeculativeEngine(load_model(str(tmp_path), "bfloat16", "cuda:0"), KVConfig(block_size=page), num_blocks=128)
    base = ru.random_ids(12, config["vocab_size"], 3)
    prompts = [base * 3, base[:5] + base[:5], [7]]
    for p, got in zip(prompts, engine.generate(prompts, 24)):
        assert len(got) == 24
        assert_tokens_within_margin(weights, config, p, got, SamplingParams())


def test_sampled_tokens_follow_the_models_distribution(tmp_path):
    """Tokens behind a prompt, in many requests with seeds of their own: how many are the likeliest one, how many are one of
    the drafts and how many lie in the vocabulary's first half, against the probabilities of the plain decoder behind the
    same tokens.  Five standard deviations."""
    from dispec_b200 import SamplingParams, SpeculativeEngine, load_model
    config, weights, _ = model_folder(str(tmp_path), "b", "float32")
    vocab, T, N, prompt = config["vocab_size"], 2.0, 500, [5, 17, 3, 8]
    known = {}

    def p_behind(tokens):
        key = tuple(tokens)
        if key not in known:
            known[key] = torch.softmax(plain.forward_logits(weights, config, list(tokens))[-1].double() / T, 0)
        return known[key]

    def draft(tokens, max_nodes):
        """The likeliest tokens, likeliest last, and behind the first of them its own likeliest."""
        first = p_behind(tokens).topk(3).indices.flip(0).tolist()
        nodes, parents = [tokens[-1]] + first, [-1, 0, 0, 0]
        nodes.append(int(p_behind(list(tokens) + [first[2]]).argmax()))
        parents.append(3)
        n = max(1, min(max_nodes, 5))
        return nodes[:n], parents[:n]

    engine = SpeculativeEngine(load_model(str(tmp_path), "float32", "cuda:0"), num_blocks=N + 8, max_nodes=5, max_num_seqs=N, draft=draft)
    out = engine.generate([prompt] * N, 4, [SamplingParams(T, seed=i) for i in range(N)])
    counts, expected, variance = torch.zeros(3).double(), torch.zeros(3).double(), torch.zeros(3).double()
    for o in out:
        assert len(o) == 4
        for i in range(1, 4):  # (the first token is the sampler's)
            p = p_behind(prompt + o[:i])
            likely = p.topk(3).indices.tolist()
            each = torch.stack([p[likely[0]], p[likely].sum(), p[:vocab // 2].sum()])
            counts += torch.tensor([o[i] == likely[0], o[i] in likely, o[i] < vocab // 2]).double()
            expected += each
            variance += each * (1 - each)
    assert ((counts - expected).abs() <= 5 * variance.sqrt()).all(), (counts, expected, variance.sqrt())


@pytest.mark.parametrize("draft", [lambda tokens, n: ([tokens[-1] + 1], [-1]), lambda tokens, n: ([], []),
                                   lambda tokens, n: ([tokens[0]], [-1]) if len(tokens) > 5 else ([tokens[-1]], [-1])])
def test_drafts_of_another_root_are_refused(draft, tmp_path):
    """What the model would run on is not what the request holds."""
    from dispec_b200 import SpeculativeEngine, load_model
    model_folder(str(tmp_path), "b", "float32")
    engine = SpeculativeEngine(load_model(str(tmp_path), "float32", "cuda:0"), num_blocks=16, draft=draft)
    with pytest.raises(ValueError, match="last token"):
        engine.generate([[5, 17, 3, 300]], 8)
    assert not engine.runner.cache.live_requests()
