"""A sliding window that leaves a request's first tokens visible, over an ordinary cache, against 64 bits: every kernel that takes
it, with what lies between the first tokens and the window given back, its pages' entries gone and all that is stale not a number."""
import math

import numpy as np
import pytest
import torch

from kv4_util import step

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from llm_singularity_b200 import kernels
    kernels.prepare(["attention", "attention_tc", "attention_tc5", "attention_repair", "rope_cache"])
    yield kernels
    kernels.check_status()


def _view(kp, vp, table, page, window):
    from llm_singularity_b200.parts.base import KVCacheView
    return KVCacheView(kp, vp, table, page, window, 0)


def _case(ops, dtype, nh, nkv, hd, q_lens, kv_lens, window, first, page=16, fixed=False, softcap=0.0, bias=False, extra=0, bad=()):
    g = torch.Generator(device="cuda").manual_seed(sum(kv_lens) + hd + window)
    R, T, group = len(q_lens), sum(q_lens), nh // nkv
    ctx = step(q_lens, kv_lens, fixed=fixed)
    per = -(-max(kv_lens) // page)
    ids = torch.randperm(R * per + 1, generator=torch.Generator().manual_seed(2))[:R * per].to(torch.int32)
    table = ids.view(R, per).clone()
    kp, vp = (torch.full((R * per + 1, nkv, page, hd), math.nan, dtype=dtype, device="cuda") for _ in range(2))
    K, V = [], []
    for r, (n, L) in enumerate(zip(q_lens, kv_lens)):
        k, v = (torch.randn(L, nkv, hd, device="cuda", generator=g).to(dtype) for _ in range(2))
        for rr, pos in bad:
            if rr == r:
                k[pos], v[pos] = math.inf, math.nan
        K.append(k)
        V.append(v)
        lo = max(0, L - n - window + 1)
        for pi in range(-(-L // page)):
            a, b = pi * page, min(L, (pi + 1) * page)
            if b <= lo and a >= first:                                  # given back
                table[r, pi] = -1
            else:
                kp[int(table[r, pi]), :, :b - a], vp[int(table[r, pi]), :, :b - a] = k[a:b].transpose(0, 1), v[a:b].transpose(0, 1)
    q = torch.randn(T, nh * hd + extra, device="cuda", generator=g).to(dtype)
    out = torch.full((T, nh * hd), math.nan, dtype=dtype, device="cuda")
    scale = 1.0 / math.sqrt(hd)
    slopes = torch.tensor([2.0 ** (-8.0 * (h + 1) / nh) for h in range(nh)], device="cuda") if bias else None
    ops.paged_attention(q, nh, nkv, hd, ctx, _view(kp, vp, table.cuda(), page, window), scale, window, out, first=first, softcap=softcap,
                        slopes=slopes)
    ops.check_status()
    t = 0
    for r, (n, L) in enumerate(zip(q_lens, kv_lens)):
        x = q[t:t + n, :nh * hd].double().view(n, nh, hd)
        blind = ~torch.isfinite(V[r]).all(-1).all(-1)
        k, v = (torch.where(blind[:, None, None], 0.0, a.double()).repeat_interleave(group, 1) for a in (K[r], V[r]))
        s = torch.einsum("ihd,jhd->hij", x, k) * scale
        pos, key = torch.arange(L - n, L, device="cuda")[:, None], torch.arange(L, device="cuda")
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        if bias:
            s = s - slopes.double()[:, None, None] * (pos - key)
        hidden = (key > pos) | ((key <= pos - window) & (key >= first))
        spoilt = (~hidden & blind).any(-1)
        s = s.masked_fill(hidden, -math.inf)
        w = torch.softmax(s, -1)
        want, size = (torch.einsum("hij,jhd->ihd", w, a).reshape(n, nh * hd) for a in (v, v.abs()))
        # Scores of size |s| are 32-bit sums of hd terms: off by less than 2^-17 (1 + |s|), weights by twice that; on the tensor
        # cores (bfloat16, heads of 64 and 128) a weight is rounded (half a step: 2^-8), and a bfloat16 result is.
        share = 2.0 ** -16 * (1 + s[s > -math.inf].abs().max().item())
        bf16 = dtype == torch.bfloat16
        if bf16 and hd in (64, 128):
            share += 2.0 ** -8
        tol = share * size + (2.0 ** -8 if bf16 else 2.0 ** -24) * want.abs()
        got = out[t:t + n].double()
        assert bool(torch.isnan(got[spoilt]).all()), r
        got, want, tol = got[~spoilt], want[~spoilt], tol[~spoilt]
        assert bool(((got - want).abs() <= tol).all()), (r, ((got - want).abs() / tol).max().item())
        t += n


WINDOWS = [(1, 1), (1, 40), (16, 16), (17, 3), (64, 64), (200, 7), (5000, 4), (31, 1000), (100, 130)]
KINDS = [(torch.float32, 8, 2, 64), (torch.float32, 6, 2, 48), (torch.float32, 4, 4, 128), (torch.float32, 14, 2, 256),
         (torch.bfloat16, 6, 1, 80), (torch.bfloat16, 8, 2, 64), (torch.bfloat16, 16, 1, 128), (torch.bfloat16, 4, 4, 128)]


@pytest.mark.parametrize("window, first", WINDOWS)
@pytest.mark.parametrize("dtype, nh, nkv, hd", KINDS)
def test_single_tokens(ops, dtype, nh, nkv, hd, window, first):
    _case(ops, dtype, nh, nkv, hd, [1] * 6, [1, 15, 64, 65, 333, 1500], window, first)
    _case(ops, dtype, nh, nkv, hd, [1] * 2, [700, 90], window, first, page=8, fixed=True, extra=2 * nkv * hd)


@pytest.mark.parametrize("window, first", WINDOWS)
@pytest.mark.parametrize("dtype, nh, nkv, hd", KINDS)
def test_portions(ops, dtype, nh, nkv, hd, window, first):
    _case(ops, dtype, nh, nkv, hd, [1, 7, 33, 2, 1], [40, 7, 210, 300, 9], window, first)
    _case(ops, dtype, nh, nkv, hd, [200, 1], [900, 700], window, first, page=32)


def test_many_requests_and_modified_scores(ops):
    _case(ops, torch.bfloat16, 4, 4, 64, [1] * 120, [5 + 37 * i % 900 for i in range(120)], 100, 4)
    _case(ops, torch.bfloat16, 8, 2, 64, [1, 30], [400, 300], 50, 4, softcap=2.5, bias=True)
    _case(ops, torch.float32, 4, 2, 32, [1, 30], [400, 300], 50, 4, bias=True)


@pytest.mark.parametrize("dtype, nh, nkv, hd", KINDS)
def test_numbers_that_are_none(ops, dtype, nh, nkv, hd):
    """Rows that see a key and value that are no numbers are none; others do not take them in."""
    _case(ops, dtype, nh, nkv, hd, [1, 1, 1], [50, 200, 200], 40, 4, bad=[(0, 30), (1, 100), (2, 2)])
    _case(ops, dtype, nh, nkv, hd, [150, 40], [500, 60], 50, 4, bad=[(0, 420), (1, 59)])
    _case(ops, dtype, nh, nkv, hd, [140], [300], 30, 2, bad=[(0, 1)])


def test_pages_that_the_prompt_kernel_does_not_take(ops):
    _case(ops, torch.bfloat16, 8, 2, 64, [1, 140], [400, 600], 50, 4, page=24)


def test_no_window_is_no_change(ops):
    """Without a window all tokens are visible, whatever is said of the first."""
    q_lens, kv_lens, nh, nkv, hd = [1, 20], [50, 60], 4, 2, 64
    ctx = step(q_lens, kv_lens)
    kp, vp = (torch.randn(8, nkv, 16, hd, device="cuda").bfloat16() for _ in range(2))
    table = torch.arange(8, dtype=torch.int32).view(2, 4).cuda()
    q = torch.randn(21, nh * hd, device="cuda").bfloat16()
    a, b = torch.empty_like(q), torch.empty_like(q)
    ops.paged_attention(q, nh, nkv, hd, ctx, _view(kp, vp, table, 16, None), 0.125, 0, a)
    ops.paged_attention(q, nh, nkv, hd, ctx, _view(kp, vp, table, 16, None), 0.125, 0, b, first=9)
    assert torch.equal(a, b)


def test_refusals(ops):
    ctx = step([1], [20])
    kp = torch.zeros(2, 1, 16, 64, device="cuda")
    table = torch.arange(2, dtype=torch.int32).view(1, 2).cuda()
    q, out = torch.zeros(1, 64, device="cuda"), torch.zeros(1, 64, device="cuda")
    with pytest.raises(ops.KernelError, match="negative"):
        ops.paged_attention(q, 1, 1, 64, ctx, _view(kp, kp, table, 16, 4), 0.1, 4, out, first=-1)
    with pytest.raises(ops.KernelError, match="rotated"):
        ops.paged_attention(q, 1, 1, 64, ctx, _view(kp, kp, table, 16, 4), 0.1, 4, out, first=2, only="single")


def test_first_page_given_back_is_reported(ops):
    for dtype in (torch.float32, torch.bfloat16):
        for q_len in (1, 140):
            ctx = step([q_len], [400])
            kp, vp = (torch.zeros(25, 2, 16, 64, dtype=dtype, device="cuda") for _ in range(2))
            table = torch.arange(25, dtype=torch.int32).view(1, 25)
            table[0, 0] = -1
            q = torch.zeros(q_len, 256, dtype=dtype, device="cuda")
            ops.paged_attention(q, 4, 2, 64, ctx, _view(kp, vp, table.cuda(), 16, 30), 0.1, 30, torch.empty_like(q), first=4)
            with pytest.raises(ops.KernelError, match="page"):
                ops.check_status()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rotation_store_and_attention_step_by_step(ops, dtype):
    """The operation a layer calls, over a prompt in portions and tokens behind it, against the whole sequence at once."""
    nh, nkv, hd, page, window, first, L = 4, 2, 64, 16, 40, 3, 260
    g = torch.Generator(device="cuda").manual_seed(9)
    qkv = torch.randn(L, (nh + 2 * nkv) * hd, device="cuda", generator=g).to(dtype)
    inv_freq = (10000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)).float().cuda()
    kp, vp = (torch.zeros(L // page + 1, nkv, page, hd, dtype=dtype, device="cuda") for _ in range(2))
    table = torch.arange(L // page + 1, dtype=torch.int32).view(1, -1).cuda()
    rows, at = [], 0
    for n in (150, 90, 17, 1, 1, 1):
        ctx = step([n], [at + n])
        part = qkv[at:at + n].clone()
        out = torch.empty(n, nh * hd, dtype=dtype, device="cuda")
        ops.rope_store_attention(part, nh, nkv, hd, ctx, _view(kp, vp, table, page, window), inv_freq, hd, True, hd ** -0.5, window, out,
                                 first=first)
        rows.append(out)
        at += n
    ops.check_status()
    got = torch.cat(rows).double()
    x = qkv.view(L, -1, hd).double()
    a = torch.arange(L, device="cuda").float()[:, None] * inv_freq[None]
    c, s = torch.cos(a.double())[:, None], torch.sin(a.double())[:, None]
    lo, hi = x[:, :nh + nkv, :hd // 2], x[:, :nh + nkv, hd // 2:]
    turned = torch.cat([lo * c - hi * s, lo * s + hi * c], -1).to(dtype).double()
    k, v = turned[:, nh:].repeat_interleave(2, 1), x[:, nh + nkv:].repeat_interleave(2, 1)
    sc = torch.einsum("ihd,jhd->hij", turned[:, :nh], k) * hd ** -0.5
    pos, key = torch.arange(L, device="cuda")[:, None], torch.arange(L, device="cuda")
    w = torch.softmax(sc.masked_fill((key > pos) | ((key <= pos - window) & (key >= first)), -math.inf), -1)
    want, size = (torch.einsum("hij,jhd->ihd", w, y).reshape(L, nh * hd) for y in (v, v.abs()))
    # in bfloat16 a rotated dim may be rounded to the other neighbour (a whole step, 2^-7) where 32-bit and 64-bit arithmetic fall on
    # two sides of a border: at most a few of a row's 64 products, so a score is off by less than 2^-7 of the sum of its products' sizes
    # over eight; weights by twice that.  Weights and results are rounded (2^-8 each).
    if dtype == torch.bfloat16:
        off = 2.0 ** -10 * (torch.einsum("ihd,jhd->hij", turned[:, :nh].abs(), k.abs()) * hd ** -0.5).max().item()
        tol = (2 * off + 2.0 ** -8) * size + 2.0 ** -8 * want.abs()
    else:
        tol = 2.0 ** -15 * (1 + sc.abs().max().item()) * size
    assert bool(((got - want).abs() <= tol).all()), ((got - want).abs() / tol).max().item()
