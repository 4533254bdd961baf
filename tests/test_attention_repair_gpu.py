"""Portions on the prompt kernel beside tokens whose keys or values are no numbers: which results are NaN, what the others are, and that it
does not take forever."""
import math

import pytest
import torch

from kv4_util import rounded, row_bytes, step, values_of

pytestmark = pytest.mark.gpu
NH, NKV = 8, 2


@pytest.fixture(scope="module")
def ops():
    from llm_singularity_b200 import kernels
    kernels.prepare(["attention", "attention_tc", "attention_tc5", "attention_repair", "kv4_store", "attention_kv4"])
    yield kernels
    kernels.check_status()


def _four_bits(k, v):
    """Pages of a 4-bit cache of one request (in order), and what they hold in 64 bits."""
    L, nkv, hd = k.shape
    pages = torch.zeros(-(-L // 16), nkv, 1, 18 * hd, dtype=torch.uint8, device="cuda")
    held = []
    for x, code_at, scale_at, value in ((k, 0, 16 * hd, False), (v, 8 * hd, 17 * hd, True)):
        codes, scales = rounded(x)
        held.append(values_of(codes, scales))
        rows = torch.zeros(pages.shape[0] * 16, nkv, hd // 2, dtype=torch.uint8, device="cuda")
        rows[:L] = row_bytes(codes, value)
        s = torch.zeros(pages.shape[0] * 16, nkv, hd // 32, dtype=torch.bfloat16, device="cuda")
        s[:L] = scales.to(torch.bfloat16)
        pages[:, :, 0, code_at:code_at + 8 * hd] = rows.view(-1, 16, nkv, hd // 2).transpose(1, 2).flatten(-2)
        pages[:, :, 0, scale_at:scale_at + hd] = s.view(-1, 16, nkv, hd // 32).transpose(1, 2).flatten(-2).contiguous().view(torch.uint8)
    return pages, held


def _run(ops, q, k, v, four, window, first, ctx):
    from llm_singularity_b200.parts.base import KV4CacheView, KVCacheView
    L, nkv, hd = k.shape
    table = torch.arange(-(-L // 16), dtype=torch.int32, device="cuda")[None]
    out = torch.empty_like(q)
    if four:
        pages, held = _four_bits(k, v)
        cache = KV4CacheView(pages, table, 16, window or None, 0)
        call = lambda: ops.paged_attention_kv4(q, NH, NKV, hd, ctx, cache, hd ** -0.5, window, out, first=first)
    else:
        kp, vp = (torch.zeros(table.shape[1] * 16, nkv, hd, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        kp[:L], vp[:L] = k.bfloat16(), v.bfloat16()
        held = [x[:L].double() for x in (kp, vp)]
        kp, vp = (x.view(-1, 16, nkv, hd).transpose(1, 2).contiguous() for x in (kp, vp))
        cache = KVCacheView(kp, vp, table, 16, window or None, 0)
        call = lambda: ops.paged_attention(q, NH, NKV, hd, ctx, cache, hd ** -0.5, window, out, first=first)
    return call, out, held


# (position, "k" or "v", dims) that are no numbers; positions 400 - 599 are the portion's own
BAD = {
    "a key that all see": [(0, "k", slice(0, 1))],
    "a key inside the portion": [(500, "k", slice(40, 41))],
    "two keys": [(30, "k", slice(None)), (590, "k", slice(3, 9))],
    "some dims of a value": [(450, "v", slice(33, 40))],
    "a value of a first token, and one of the last": [(1, "v", slice(0, 5)), (599, "v", slice(60, 64))],
    "values of two groups at several tokens": [(2, "v", slice(5, 6)), (410, "v", slice(32, 64)), (520, "v", slice(5, 6)), (521, "v", slice(6, 7))],
    "keys and values": [(480, "k", slice(None)), (480, "v", slice(None)), (560, "v", slice(1, 2))],
}


@pytest.mark.parametrize("bad", list(BAD))
@pytest.mark.parametrize("four, window, first", [(True, 0, 0), (True, 60, 4), (True, 150, 0), (False, 60, 4), (False, 150, 2)])
@pytest.mark.parametrize("hd", [64, 128])
def test_what_is_none_and_what_is_not(ops, hd, four, window, first, bad):
    n, L = 200, 600
    g = torch.Generator(device="cuda").manual_seed(hd + window)
    k, v = (torch.randn(L, NKV, hd, device="cuda", generator=g) for _ in range(2))
    q = torch.randn(n, NH * hd, device="cuda", generator=g).bfloat16()
    for pos, which, dims in BAD[bad]:
        (k if which == "k" else v)[pos, 0, dims] = math.nan              # (of the first kv head)
    call, out, (K, V) = _run(ops, q, k, v, four, window, first, step([n], [L]))
    call()
    ops.check_status()
    K, V = (x.repeat_interleave(NH // NKV, 1) for x in (K, V))
    pos, key = torch.arange(L - n, L, device="cuda")[:, None], torch.arange(L, device="cuda")
    sees = (key <= pos) & ((key > pos - window) | (key < first)) if window else key <= pos
    s = torch.einsum("ihd,jhd->hij", q.double().view(n, NH, hd), torch.nan_to_num(K)) * hd ** -0.5
    w = torch.softmax(s.masked_fill(~sees, -math.inf), -1)
    want, size = (torch.einsum("hij,jhd->ihd", w, torch.nan_to_num(x)) for x in (V, V.abs()))
    none = torch.einsum("ij,jhd->ihd", sees.double(), torch.isnan(V).double()) > 0
    none |= (torch.einsum("ij,jh->ih", sees.double(), torch.isnan(K).any(-1).double()) > 0)[..., None]
    got = out.double().view(n, NH, hd)
    assert torch.equal(torch.isnan(got), none)
    # scores are 32-bit sums of hd products: off by less than 2^-17 (1 + |s|), weights by twice that, and a weight and the result are rounded
    tol = (2.0 ** -16 * (1 + s.abs().max().item()) + 2.0 ** -8) * size + 2.0 ** -8 * want.abs()
    assert bool(((got - want).abs() <= tol)[~none].all()), ((got - want).abs() / tol)[~none].max().item()


@pytest.mark.parametrize("which", ["k", "v"])
def test_rows_that_see_what_is_none_are_not_formed_again(ops, which):
    """A portion whose rows are all NaN for one early token takes a few times as long as one of numbers (215 times where every row walked
    its keys)."""
    n, L, hd = 1500, 3000, 128
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn(L, NKV, hd, device="cuda", generator=g) for _ in range(2))
    q = torch.randn(n, NH * hd, device="cuda", generator=g).bfloat16()
    took = []
    for spoil in (False, True):
        if spoil:
            (k if which == "k" else v)[100] = math.nan
        call, out, _ = _run(ops, q, k, v, True, 0, 0, step([n], [L]))
        call()
        torch.cuda.synchronize()
        times = []
        for _ in range(5):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            call()
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        took.append(min(times))
        assert bool(torch.isnan(out).all()) == spoil
    assert took[1] < 20 * took[0], took
