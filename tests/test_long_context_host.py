"""Caches of 4 bits and windows with first tokens, from the options to the pages, without a GPU: what is refused, which pages
stay, and whole models over stand-ins of the kernels against a plain Llama."""
import random

import pytest
import torch

import plain_llama
import tiny_models
from llm_singularity_b200.cache.manager import CacheManager
from llm_singularity_b200.cache.pages import PageError
from llm_singularity_b200.cli import build_parser
from llm_singularity_b200.config.llama import LlamaConfig
from llm_singularity_b200.config.specs import AttentionSpec, with_long_context
from llm_singularity_b200.engine import StepEntry
from llm_singularity_b200.engine.engine import Engine
from llm_singularity_b200.engine.runner import ModelRunner
from llm_singularity_b200.parts.attention import PagedAttention
from llm_singularity_b200.parts.base import CompositeCacheSpec, PagedKV4Spec, PagedKVSpec, Runtime
from long_context_util import Ops, forward_logits


def _spec(name="tiny_b"):
    return LlamaConfig.from_dict(tiny_models.CONFIGS[name]).to_model_spec()


# ------------------------------------------------------------------ options
def test_options_change_every_layer_and_nothing_else():
    spec = _spec()
    assert with_long_context(spec) is spec
    got = with_long_context(spec, "int4", 40, 4)
    assert all((b.mixer.cache_bits, b.mixer.window, b.mixer.first_tokens) == (4, 40, 4) for b in got.blocks)
    assert got.tensor_names == spec.tensor_names and got.order == spec.order
    got = with_long_context(spec, "compute", 7)
    assert all((b.mixer.cache_bits, b.mixer.window, b.mixer.first_tokens) == (None, 7, 0) for b in got.blocks)


@pytest.mark.parametrize("options, says", [(("int8",), "kv_cache"), (("int4", 0), "window"), (("compute", -3), "window"),
                                           (("compute", None, 4), "first_tokens"), (("compute", 9, -1), "first_tokens")])
def test_options_refused(options, says):
    with pytest.raises(ValueError, match=says):
        with_long_context(_spec(), *options)


def test_other_designs_have_caches_of_their_own():
    from dataclasses import replace
    from llm_singularity_b200.config.specs import KVAttentionSpec
    spec = _spec()
    spec = replace(spec, blocks=(replace(spec.blocks[0], mixer=KVAttentionSpec()),) + spec.blocks[1:])
    for options in (("int4",), ("compute", 8)):
        with pytest.raises(ValueError, match="kv_attention"):
            with_long_context(spec, *options)
    assert with_long_context(spec) is spec


def test_sizes_refused():
    rt = Runtime("cpu", torch.float32, ops=Ops())
    with pytest.raises(ValueError, match="multiple of 32"):
        PagedKV4Spec(2, 48)
    with pytest.raises(ValueError, match="up to 256"):
        PagedKV4Spec(2, 288)
    with pytest.raises(ValueError, match="multiple of 16"):
        PagedKV4Spec(2, 64).allocate(rt, 8, 4, 2)
    from llm_singularity_b200.config.specs import RotarySpec
    base = dict(hidden_size=64, num_heads=2, num_kv_heads=1, head_dim=32, position=RotarySpec(head_dim=32, rotary_dim=32))
    for more, says in ((dict(cache_bits=8), "4 bits"), (dict(cache_bits=4, logit_softcap=2.0), "modifies"),
                       (dict(cache_bits=4, linear_bias=True), "modifies"), (dict(window=4, first_tokens=-1), "negative")):
        with pytest.raises(ValueError, match=says):
            PagedAttention(AttentionSpec(**base, **more), rt)
    part = PagedAttention(AttentionSpec(**base, cache_bits=4, window=9, first_tokens=3), rt)
    assert part.cache_spec() == PagedKV4Spec(1, 32, 9, 3)
    assert PagedAttention(AttentionSpec(**base, window=9, first_tokens=3), rt).cache_spec() == PagedKVSpec(1, 32, 9, first=3)
    assert PagedAttention(AttentionSpec(**base, first_tokens=3), rt).cache_spec() == PagedKVSpec(1, 32)
    with pytest.raises(ValueError, match="first tokens"):
        CompositeCacheSpec((PagedKVSpec(1, 32, 9, first=3), PagedKVSpec(1, 32, 9)))


def test_bytes_of_a_page():
    assert PagedKV4Spec(8, 128).bytes_per_page(16, 2) == 8 * 16 * 2 * (128 // 2 + 128 // 16)
    store = PagedKV4Spec(8, 128).allocate(Runtime("cpu", torch.float32, ops=Ops()), 32, 3, 1)
    assert store.numel() == 3 * PagedKV4Spec(8, 128).bytes_per_page(32, 2)


def test_command_line():
    a = build_parser().parse_args(["--model-dir", "x", "--kv-cache", "int4", "--window", "100", "--first-tokens", "4"])
    assert (a.kv_cache, a.window, a.first_tokens) == ("int4", 100, 4)
    a = build_parser().parse_args(["--model-dir", "x"])
    assert (a.kv_cache, a.window, a.first_tokens) == ("compute", None, 0)


# ------------------------------------------------------------------ pages
@pytest.mark.parametrize("seed", range(20))
def test_which_pages_stay(seed):
    """Under random orders of growth and closing: the pages of first tokens and of the window, and no others."""
    rng = random.Random(seed)
    ps, window, first = rng.choice([2, 4, 16]), rng.randint(1, 40), rng.randint(1, 30)
    m = CacheManager([PagedKVSpec(1, 16, window, first=first), PagedKVSpec(1, 16, window), PagedKVSpec(1, 16),
                      PagedKV4Spec(1, 32, window, first)], ps, 400, 3, 100)
    assert [(g.window, g.first) for g in m.groups] == [(window, first), (window, None), (None, None)]
    assert m.group_of(0) == m.group_of(3) == 0
    length = {}
    for _ in range(200):
        r = rng.randrange(4)
        if r not in length:
            if m.open(r) is not None:
                length[r] = 0
        elif rng.random() < 0.1:
            m.close(r)
            del length[r]
        else:
            n = min(length[r] + rng.randint(1, 9), 100 * ps)
            if m.reserve(r, n):
                m.commit(r, n)
                length[r] = n
        m.check_invariants()
        for q, n in length.items():
            for g, keep in ((0, first), (1, 0), (2, 10 ** 6)):
                for i, page in enumerate(m.pages_of(q, g)):
                    needed = i * ps < keep or (i + 1) * ps > max(0, n - window + 1)
                    assert (page >= 0) == needed, (q, n, g, i)
    for r in list(length):
        m.close(r)
    m.check_invariants()
    assert all(g.pool.num_free == 400 for g in m.groups)


def test_what_a_group_keeps_is_said_before_a_request_is_open():
    m = CacheManager([PagedKVSpec(1, 16, 5, first=2)], 4, 9, 2, 9)
    m.open("a")
    assert m._lib.lsbm_keep_first(m._ptr, 0, 3) < 0 and "before" in m._lib.lsbm_last_error(m._ptr).decode()
    m.close("a")
    assert m._lib.lsbm_keep_first(m._ptr, 0, -1) < 0 and m._lib.lsbm_keep_first(m._ptr, 5, 1) < 0
    with pytest.raises(PageError):
        raise m._fail()


# ------------------------------------------------------------------ whole models
@pytest.fixture(scope="module")
def model(tmp_path_factory):
    path = tiny_models.make_model_dir(str(tmp_path_factory.mktemp("m")), "tiny_b")
    return path, *plain_llama.load_model_dir(path)


def _runner(path, **o):
    return ModelRunner(path, dtype="float32", device="cpu", page_size=16, num_pages=40, max_requests=3, ops=Ops(), **o)


def _run(runner, tokens, portions):
    runner.open("a")
    rows, at = [], 0
    for n in portions:
        rows.append(runner.step([StepEntry("a", tokens[at:at + n], list(range(n)))]).clone())
        at += n
    runner.cache.check_invariants()
    return torch.cat(rows).double()


def test_window_and_first_tokens_in_a_model(model):
    path, cfg, w = model
    tokens = tiny_models.random_tokens(512, 90, 3)
    got = _run(_runner(path, window=20, first_tokens=3), tokens, [37, 20, 30, 1, 1, 1])
    want = forward_logits(cfg, w, tokens, window=20, first=3)
    assert (got - want).abs().max() < 1e-3 and (want - forward_logits(cfg, w, tokens, window=20)).abs().max() > 0.05


@pytest.mark.parametrize("window, first", [(None, 0), (20, 3)])
def test_four_bits_in_a_model(model, window, first):
    """The yardstick is what 4 bits change: where a 32-bit sum falls on the other side of a border between two codes, rows move
    by a small part of that."""
    path, cfg, w = model
    tokens = tiny_models.random_tokens(512, 60, 4)
    got = _run(_runner(path, kv_cache="int4", window=window, first_tokens=first), tokens, [37, 20, 1, 1, 1])
    want = forward_logits(cfg, w, tokens, kv4=True, window=window, first=first, key_round=torch.float32)
    change = (want - forward_logits(cfg, w, tokens, window=window, first=first)).norm()
    assert change > 0.01 * want.norm() and (got - want).norm() < 0.1 * change


def test_a_sequence_without_end_in_a_small_pool(model):
    """A prompt and an answer much longer than the pool, in the pages of the window, the first tokens and a step."""
    path, cfg, w = model
    eng = Engine(path, dtype="float32", device="cpu", kv_block_size=16, num_kv_blocks=6, max_batch_size=1, max_tokens_per_batch=24,
                 max_model_len=300, ops=Ops(), window=20, first_tokens=3)
    assert eng.prefix is None
    prompt = tiny_models.random_tokens(512, 150, 8)
    out = eng.generate([prompt], max_new_tokens=40, ignore_eos=True)[0]
    want = forward_logits(cfg, w, prompt + out[:-1], window=20, first=3)[len(prompt) - 1:]
    top = want.topk(2, -1).values
    for i, t in enumerate(out):
        assert float(want[i, t]) >= float(top[i, 0]) - 1e-3
    eng.runner.cache.check_invariants()
    assert eng.runner.cache.free_pages() == 6


def test_a_window_that_no_pool_holds_is_refused(model):
    path, _, _ = model
    eng = Engine(path, dtype="float32", device="cpu", kv_block_size=16, num_kv_blocks=5, max_batch_size=1, max_tokens_per_batch=24,
                 max_model_len=300, ops=Ops(), window=40, first_tokens=3)
    with pytest.raises(RuntimeError, match="pages, the pool has 5"):
        eng.generate([tiny_models.random_tokens(512, 150, 8)], max_new_tokens=4, ignore_eos=True)


def test_shared_prefixes_of_a_four_bit_cache(model):
    path, _, _ = model
    shared = tiny_models.random_tokens(512, 48, 9)
    prompts = [shared + tiny_models.random_tokens(512, 5, i) for i in range(2)]
    kw = dict(dtype="float32", device="cpu", kv_block_size=16, num_kv_blocks=20, max_batch_size=2, max_tokens_per_batch=64, kv_cache="int4")
    cold = [Engine(path, ops=Ops(), prefix_cache=False, **kw).generate([p], max_new_tokens=4, ignore_eos=True)[0] for p in prompts]
    warm = Engine(path, ops=Ops(), **kw)
    assert [warm.generate([p], max_new_tokens=4, ignore_eos=True)[0] for p in prompts] == cold
    assert warm.stats()["prefix_hit_tokens"] == 48
