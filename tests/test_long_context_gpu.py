"""Caches of 4 bits and windows with first tokens through the engine on the GPU: prompts in portions, decoded tokens, captured
steps and the command line, against a plain Llama in 64 bits."""
import json
import os
import subprocess
import sys

import pytest
import torch

import plain_llama
import tiny_models
from long_context_util import forward_logits

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NAMES = {"tiny_b": 32, "tiny_d": 64, "tiny_e": 128}


@pytest.fixture(scope="module")
def models(tmp_path_factory):
    base = tmp_path_factory.mktemp("long")
    out = {}
    for name in NAMES:
        path = tiny_models.make_model_dir(str(base / name), name)
        out[name] = (path, *plain_llama.load_model_dir(path))
    return out


def _runner(path, dtype, page=16, pages=64, **o):
    from llm_singularity_b200.engine.runner import ModelRunner
    return ModelRunner(path, dtype=dtype, page_size=page, num_pages=pages, max_requests=3, max_tokens_per_step=512, **o)


def _run(runner, tokens, portions):
    from llm_singularity_b200.engine import StepEntry
    runner.open("a")
    rows, at = [], 0
    for n in portions:
        rows.append(runner.step([StepEntry("a", tokens[at:at + n], list(range(n)))]).double().cpu())
        at += n
    runner.check_kernels()
    runner.cache.check_invariants()
    return torch.cat(rows)


@pytest.mark.parametrize("name", list(NAMES))
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_window_and_first_tokens(models, name, dtype):
    path, cfg, w = models[name]
    tokens = tiny_models.random_tokens(cfg["vocab_size"], 290, 3)
    got = _run(_runner(path, dtype, window=70, first_tokens=5), tokens, [150, 37, 90, 1] + [1] * 12)
    act = dtype if dtype == "bfloat16" else None
    want = forward_logits(cfg, w, tokens, window=70, first=5, act_round=act)
    # (what the first tokens change is the yardstick: rows far behind them would move by it if they were forgotten)
    change = (want - forward_logits(cfg, w, tokens, window=70, act_round=act)).norm()
    assert change > 0.02 * want.norm()
    assert (got - want).norm() < (1e-3 if dtype == "float32" else 0.3) * change


@pytest.mark.parametrize("window, first", [(None, 0), (70, 5)])
@pytest.mark.parametrize("name", list(NAMES))
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_four_bits(models, name, dtype, window, first):
    """What 4 bits change is the yardstick: where a sum falls on the other side of a border between two codes, rows move by a
    small part of that (in bfloat16 a key is off by up to 2^-8 of itself, a fortieth of the step between codes on average)."""
    path, cfg, w = models[name]
    tokens = tiny_models.random_tokens(cfg["vocab_size"], 220, 4)
    got = _run(_runner(path, dtype, kv_cache="int4", window=window, first_tokens=first, page=32), tokens, [140, 37, 30, 1] + [1] * 12)
    act = dtype if dtype == "bfloat16" else None
    want = forward_logits(cfg, w, tokens, kv4=True, window=window, first=first, act_round=act, key_round=torch.float32)
    change = (want - forward_logits(cfg, w, tokens, window=window, first=first, act_round=act)).norm()
    assert change > 0.01 * want.norm() and (got - want).norm() < (0.1 if dtype == "float32" else 0.6) * change


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("kv_cache", ["compute", "int4"])
def test_portions_and_batches_do_not_change_a_sequence(models, kv_cache, dtype):
    """Generated tokens of three requests together, in portions, with captured steps and pages shared out anew, and of each alone."""
    from llm_singularity_b200 import Engine
    path, cfg, w = models["tiny_d"]
    prompts = [tiny_models.random_tokens(cfg["vocab_size"], n, 60 + n) for n in (5, 90, 170)]
    kw = dict(dtype=dtype, kv_block_size=16, kv_cache=kv_cache, window=48, first_tokens=4)
    together = Engine(path, num_kv_blocks=24, max_batch_size=3, max_tokens_per_batch=64, max_model_len=400, **kw)
    outs = together.generate(prompts, max_new_tokens=60, ignore_eos=True)
    assert together.runner.graph_replays > 20 and together.runner.cache.free_pages() == 24
    together.runner.check_kernels()
    together.runner.cache.check_invariants()
    for p, out in zip(prompts, outs):
        want = forward_logits(cfg, w, p + out[:-1], kv4=kv_cache == "int4", window=48, first=4, key_round=torch.float32,
                              act_round="bfloat16" if dtype == "bfloat16" else None)[len(p) - 1:]
        top = want.max(-1).values
        spread = want.std()
        # every token is the plain model's best or within rounding of it (4 bits: a fallen border here and there)
        slack = (1e-3 if dtype == "float32" else 0.1) if kv_cache == "compute" else (0.1 if dtype == "float32" else 0.5) * spread
        for i, t in enumerate(out):
            assert float(want[i, t]) >= float(top[i]) - slack, i


def test_a_sequence_without_end_in_a_small_pool(models):
    from llm_singularity_b200 import Engine
    path, cfg, w = models["tiny_e"]
    eng = Engine(path, dtype="bfloat16", kv_block_size=16, num_kv_blocks=9, max_batch_size=1, max_tokens_per_batch=64, max_model_len=1200,
                 kv_cache="int4", window=64, first_tokens=4)
    out = eng.generate([tiny_models.random_tokens(cfg["vocab_size"], 700, 1)], max_new_tokens=300, ignore_eos=True)[0]
    assert len(out) == 300 and eng.runner.cache.free_pages() == 9
    eng.runner.check_kernels()
    eng.runner.cache.check_invariants()


def test_shared_prefixes(models):
    from llm_singularity_b200 import Engine
    path, cfg, w = models["tiny_d"]
    shared = tiny_models.random_tokens(cfg["vocab_size"], 48, 9)
    prompts = [shared + tiny_models.random_tokens(cfg["vocab_size"], 5, i) for i in range(3)]
    kw = dict(dtype="float32", kv_block_size=16, num_kv_blocks=32, max_batch_size=2, max_tokens_per_batch=64, kv_cache="int4")
    cold = Engine(path, prefix_cache=False, **kw)
    want = [cold.generate([p], max_new_tokens=6, ignore_eos=True)[0] for p in prompts]
    warm = Engine(path, **kw)
    assert [warm.generate([p], max_new_tokens=6, ignore_eos=True)[0] for p in prompts] == want
    assert warm.stats()["prefix_hit_tokens"] == 2 * 48


def test_command_line(models):
    path, cfg, _ = models["tiny_d"]
    cmd = [sys.executable, "-m", "llm_singularity_b200.cli", "--model-dir", path, "--prompt-len", "40", "--num-requests", "2",
           "--max-new-tokens", "6", "--ignore-eos", "--kv-cache", "int4", "--window", "32", "--first-tokens", "4"]
    r = subprocess.run(cmd, cwd=ROOT, capture_output=True, text=True, timeout=240)
    assert r.returncode == 0, r.stderr[-800:]
    lines = [json.loads(x) for x in r.stdout.splitlines() if x.startswith("{")]
    assert len(lines) == 2 and all(len(x["tokens"]) == 6 for x in lines)
