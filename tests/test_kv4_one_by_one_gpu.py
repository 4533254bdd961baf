"""Prompt portions over a 4-bit cache whose unpacked caches do not fit together: one after the other, to the same bits."""
import math

import pytest
import torch

from kv4_util import step
from test_kv4_long_gpu import _cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window, first", [(0, 0), (150, 4)])
@pytest.mark.parametrize("nh, nkv, hd", [(8, 2, 64), (4, 4, 128)])
def test_one_after_the_other(monkeypatch, nh, nkv, hd, window, first):
    from llm_singularity_b200 import kernels as ops
    from llm_singularity_b200.parts.base import KV4CacheView
    ops.prepare(["kv4_store", "attention_kv4", "attention_tc5", "attention_repair"])
    q_lens, kv_lens = [1, 200, 1, 30, 140], [300, 700, 41, 500, 140]
    g = torch.Generator(device="cuda").manual_seed(4)
    pages, table, _ = _cache(kv_lens, nkv, hd, g, 0)
    q = torch.randn(sum(q_lens), nh * hd, device="cuda", generator=g).bfloat16()
    cache = KV4CacheView(pages, table, 16, window or None, 0)
    results = []
    for room in (1 << 30, 50 * nkv * 64 * hd):                  # (50 tiles: enough for 700 tokens, not for two of them)
        monkeypatch.setattr(ops, "_kv4_expanded", (room, room))
        out, ctx = torch.full_like(q, math.nan), step(q_lens, kv_lens)
        ops.paged_attention_kv4(q, nh, nkv, hd, ctx, cache, hd ** -0.5, window, out, first=first)
        ops.check_status()
        results.append((out, [p[0] for plan in ctx._kv4_plans.values() for p in plan]))
    assert results[0][1] == [1, 3] and results[1][1] == [1, 3, 3, 3]
    assert bool(torch.isfinite(results[0][0]).all()) and torch.equal(results[0][0], results[1][0])
