"""Portions whose cache is unpacked first, in memory that held another step's lengths and pages before."""
import math

import pytest
import torch

from kv4_util import rounded, row_bytes, step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window, first", [(0, 0), (70, 0), (70, 4)])
@pytest.mark.parametrize("captured", [False, True])
def test_lengths_of_an_earlier_step_are_not_read(window, first, captured):
    """The lengths that unpacking writes lie where the step before left others, which would be as good as any: the results are the
    first call's, every time, eagerly and replayed."""
    from llm_singularity_b200 import kernels as ops
    from llm_singularity_b200.parts.base import KV4CacheView
    ops.prepare(["kv4_store", "attention_kv4", "attention_tc5", "attention_repair"])
    nh, nkv, hd, n, L = 8, 2, 64, 200, 900
    g = torch.Generator(device="cuda").manual_seed(3)
    pages = torch.zeros(-(-L // 16), nkv, 1, 18 * hd, dtype=torch.uint8, device="cuda")
    for base, value in ((0, False), (8 * hd, True)):
        codes, scales = rounded(torch.randn(pages.shape[0], nkv, 16, hd, device="cuda", generator=g))
        pages[:, :, 0, base:base + 8 * hd] = row_bytes(codes, value).flatten(-2)
        at = 17 * hd if value else 16 * hd
        pages[:, :, 0, at:at + hd] = scales.to(torch.bfloat16).flatten(-2).contiguous().view(torch.uint8)
    table = torch.arange(pages.shape[0], dtype=torch.int32, device="cuda")[None]
    cache = KV4CacheView(pages, table, 16, window or None, 0)
    q = torch.randn(n, nh * hd, device="cuda", generator=g).bfloat16()
    out = torch.empty_like(q)
    ctx = step([n], [L], fixed=captured)

    def run():
        ops.paged_attention_kv4(q, nh, nkv, hd, ctx, cache, 1 / math.sqrt(hd), window, out, first=first)

    seen = L if not window else min(L, window + n + first)
    room = -(-seen // 16) + 2

    def leave_another_length():
        """Table entries and the row are right, the length is one of a shorter context."""
        ints = torch.zeros(room + 2, dtype=torch.int32, device="cuda")
        ints[-1] = n + 16

    run()
    want = out.clone()
    assert bool(torch.isfinite(want).all()) and want.float().abs().max() > 0.01
    if captured:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run()
        run = graph.replay
    for _ in range(30):
        leave_another_length()
        out.fill_(math.nan)
        run()
        assert torch.equal(out, want)
    ops.check_status()
