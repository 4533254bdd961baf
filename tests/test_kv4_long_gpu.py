"""Attention over a 4-bit cache at long contexts, with bounds that tell: queries whose scores no arithmetic of the kernels rounds.

Zeros as queries make every visible token count alike, so that results are means of values, and one left out or taken in shows.
Queries of small whole numbers have exact sums over a group of 32 dims (whole numbers below 2^24 in either form of the products, codes
raised by 1,024 included), so that a score's error is that of adding up scaled groups alone.  Every test looks, on its oracle, at
what a mistake would have done: a token left out, a query with its dims in another order."""
import math

import pytest
import torch

from kv4_util import attention, rounded, row_bytes, step, values_of

BF16, F32 = torch.bfloat16, torch.float32


def _cache(kv_lens, nkv, hd, g, width):
    """Pages in no order, their tables, and per request keys, values (64-bit) and the scales of values' groups."""
    per = [-(-L // 16) for L in kv_lens]
    ids = torch.randperm(sum(per) + 1, generator=torch.Generator().manual_seed(7))[:sum(per)].to(torch.int32)
    device = g.device
    pages = torch.full((sum(per) + 1, nkv, 1, 18 * hd), 255, dtype=torch.uint8, device=device)
    table = torch.full((len(kv_lens), max(width, max(per))), -1, dtype=torch.int32)
    held, at = [], 0
    for r, (L, n) in enumerate(zip(kv_lens, per)):
        own = ids[at:at + n].to(device).long()
        table[r, :n] = ids[at:at + n]
        at += n
        parts, sizes = [], []
        for value in (False, True):
            codes, scales = rounded(torch.randn(L, nkv, hd, device=device, generator=g))
            held_now = values_of(codes, scales)
            rows = torch.full((n * 16, nkv, hd // 2), 255, dtype=torch.uint8, device=device)
            rows[:L] = row_bytes(codes, value)
            s = torch.full((n * 16, nkv, hd // 32), math.nan, dtype=BF16, device=device)
            s[:L] = scales.to(BF16)
            a, b = (8 * hd, 17 * hd) if value else (0, 16 * hd)
            tiles = pages[own, :, 0]
            tiles[..., a:a + 8 * hd] = rows.view(n, 16, nkv, hd // 2).transpose(1, 2).flatten(-2)
            tiles[..., b:b + hd] = s.view(n, 16, nkv, hd // 32).transpose(1, 2).flatten(-2).contiguous().view(torch.uint8)
            pages[own, :, 0] = tiles
            parts.append(held_now)
            sizes.append(scales.repeat_interleave(32, -1))
        held.append((*parts, sizes[1]))
    return pages, table.to(device), held


def _queries(kind, n, nh, hd, g):
    if kind == "zeros":
        return torch.zeros(n, nh, hd, device=g.device)
    return torch.randint(-4, 5, (n, nh, hd), device=g.device, generator=g).float()


def _bounds(dtype, kind, q, K, V, L, scale, window, first, steps, expanded):
    want, size, per_step = attention(q, K, V, L, scale, window, first, steps)
    wide = dtype == F32
    # Sums over tokens: a warp (of four) or a block takes chunks of 32 or 64 tokens one after the other, and each loses at most 36 units of
    # 2^-24 of what is summed so far; with bfloat16 rows over a 4-bit cache also of codes raised by 136 (up to 143 of a step).
    share = 36 * 2.0 ** -24 * (L / (64 if expanded else 128) + 2) + 2.0 ** -20
    extra = 0.0 if wide or expanded else 36 * 143 * 2.0 ** -24
    if kind != "zeros":
        # Scores: groups (or, on the prompt kernel, dims) are added up in 32-bit, an error of less than 40 units of 2^-24 of the sum of
        # their magnitudes, times the scale; an exponential is within 2^-21; a weight is rounded to bfloat16 (half a step: 2^-8).
        group = q.shape[1] // K.shape[1]
        reach = torch.einsum("ihd,jhd->hij", q.double().abs(), K.repeat_interleave(group, 1).abs()).max().item() * abs(scale)
        share += 2 * 40 * 2.0 ** -24 * reach + 2.0 ** -20 + (0.0 if wide else 2.0 ** -8)
    tol = share * size + extra * per_step + (2.0 ** -24 if wide else 2.0 ** -8) * want.abs()
    return want, tol


def _wrong(kind, q, K, V, L, scale, window, first, steps):
    """The oracle with a mistake: the token before the last one left out of all rows (its value counts as nothing), or a query's dims
    moved on by one."""
    if kind != "zeros":
        return attention(q.roll(1, -1), K, V, L, scale, window, first, steps)[0]
    n, nh, hd = q.shape
    keep = torch.ones(L, dtype=torch.float64, device=q.device)
    keep[max(0, L - n - 2)] = 0
    return attention(q, K, V * keep[:, None, None], L, scale, window, first, steps)[0]


CASES = [([1] * 5, [1, 33, 500, 1111, 2999], 0, 0), ([1] * 3, [700, 2000, 1500], 600, 5), ([40, 7], [1500, 900], 0, 0), ([33], [1700], 900, 20),
         ([1, 150], [400, 1200], 0, 0), ([200], [1600], 700, 70)]
HEADS = [(8, 2, 64), (16, 1, 64), (16, 4, 128), (16, 1, 128), (6, 6, 96), (4, 1, 32), (5, 1, 160), (2, 2, 192), (4, 4, 224), (8, 4, 256)]


def _inputs(device, kind, dtype, nh, nkv, hd, q_lens, kv_lens, width):
    g = torch.Generator(device=device).manual_seed(hd + sum(kv_lens))
    pages, table, held = _cache(kv_lens, nkv, hd, g, width)
    q = [_queries(kind, n, nh, hd, g) for n in q_lens]
    return pages, table, held, q, (1.0 if kind == "zeros" else 3.0 / (2.6 * math.sqrt(hd)))


def _powers(kind, dtype, nh, nkv, hd, case, device="cpu"):
    """How many of a case's results a mistake would have moved out of their bounds."""
    q_lens, kv_lens, window, first = case
    _, _, held, q, scale = _inputs(device, kind, dtype, nh, nkv, hd, q_lens, kv_lens, 0)
    for (K, V, steps), x, L in zip(held, q, kv_lens):
        if L < 30:
            continue
        want, tol = _bounds(dtype, kind, x, K, V, L, scale, window, first, steps, len(x) >= 128 and hd in (64, 128) and dtype == BF16)
        yield ((_wrong(kind, x, K, V, L, scale, window, first, steps) - want).abs() > 2 * tol).double().mean().item()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kind", ["zeros", "whole"])
def test_a_mistake_would_show(kind, dtype):
    """(On the CPU: the oracle against itself with a mistake.)  A tenth of the results, each by twice its bound: a run that makes it is caught
    wherever in its bounds it would else be."""
    for nh, nkv, hd in ((4, 1, 32), (2, 2, 64)):
        for case in CASES:
            assert min(_powers(kind, dtype, nh, nkv, hd, case)) > 0.1, (nh, nkv, hd, case)


@pytest.mark.gpu
@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("kind", ["zeros", "whole"])
@pytest.mark.parametrize("nh, nkv, hd", HEADS)
def test_long_contexts(nh, nkv, hd, kind, dtype, captured):
    from llm_singularity_b200 import kernels as ops
    from llm_singularity_b200.parts.base import KV4CacheView
    ops.prepare(["kv4_store", "attention_kv4", "attention_kv4_f32", "attention_tc5", "attention_repair"])
    for q_lens, kv_lens, window, first in CASES:
        # (a captured step is planned by the table's width: 4,096 tokens and more are spread)
        pages, table, held, q, scale = _inputs("cuda", kind, dtype, nh, nkv, hd, q_lens, kv_lens, 400 if captured else 0)
        rows = torch.cat([x.flatten(1) for x in q]).to(dtype)
        out = torch.full_like(rows, math.nan)
        ctx = step(q_lens, kv_lens, fixed=captured)
        ops.paged_attention_kv4(rows, nh, nkv, hd, ctx, KV4CacheView(pages, table, 16, window or None, 0), scale, window, out, first=first)
        ops.check_status()
        at = 0
        for (K, V, steps), x, L in zip(held, q, kv_lens):
            got = out[at:at + len(x)].double().view(x.shape)
            at += len(x)
            want, tol = _bounds(dtype, kind, x, K, V, L, scale, window, first, steps, max(q_lens) >= 128 and len(x) > 1 and hd in (64, 128) and dtype == BF16)
            assert bool(((got - want).abs() <= tol).all()), (q_lens, kv_lens, L, ((got - want).abs() / tol).max().item())
