"""The 4-bit cache: what the store writes, to the bit, what reading it back gives, and attention over it against 64 bits, at
every head size, with stale and foreign places of the pages full of scales that are no numbers."""
import math

import numpy as np
import pytest
import torch

from kv4_util import attention, put, rounded, row_bytes, scale_of, step, values_of

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16]


@pytest.fixture(scope="module")
def ops():
    from llm_singularity_b200 import kernels
    kernels.prepare(["kv4_store", "attention_kv4", "attention_kv4_f32", "attention_tc5", "attention_repair"])
    yield kernels
    kernels.check_status()


def _view(pages, table, page_size, window=None):
    from llm_singularity_b200.parts.base import KV4CacheView
    return KV4CacheView(pages, table, page_size, window, 0)


def _pool(R, longest, nkv, hd, page_size, seed=1):
    """Pages in no order, every byte of them 0xff (scales that are no numbers), two of them nobody's; and their tables."""
    per = -(-longest // page_size)
    pages = torch.full((R * per + 2, nkv, page_size // 16, 18 * hd), 255, dtype=torch.uint8, device="cuda")
    ids = torch.randperm(R * per + 2, generator=torch.Generator().manual_seed(seed))[:R * per]
    return pages, ids.to(torch.int32).view(R, per).cuda()


# ------------------------------------------------------------------ the store
def _turned(x, pos, inv_freq, rotary_dim):
    """Rotated in 64 bits; x [T, heads, hd]."""
    half = rotary_dim // 2
    a = pos.double()[:, None] * inv_freq.double()[None] if half else pos.double()[:, None].new_zeros(len(pos), 0)
    c, s = torch.cos(a)[:, None], torch.sin(a)[:, None]
    x = x.double()
    lo, hi = x[..., :half], x[..., half:rotary_dim]
    return torch.cat([lo * c - hi * s, lo * s + hi * c, x[..., rotary_dim:]], -1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nh, nkv, hd, rotary_dim, page_size", [
    (4, 1, 32, 32, 16), (8, 2, 64, 64, 32), (6, 3, 96, 36, 16), (8, 8, 128, 128, 48), (3, 1, 160, 0, 16), (2, 2, 192, 190, 16),
    (5, 5, 224, 2, 16), (4, 2, 256, 256, 64)])
def test_store(ops, dtype, nh, nkv, hd, rotary_dim, page_size):
    q_lens, kv_lens = [1, 17, 1, 40], [131071, 17, 33, 100]
    R, T = len(q_lens), sum(q_lens)
    ctx = step(q_lens, kv_lens, rows=[3, 0, 5, 1])
    pages, _ = _pool(7, page_size, nkv, hd, page_size)                   # nine pages
    table = torch.full((6, -(-131072 // page_size)), -1, dtype=torch.int32)
    free = iter(range(9))
    held = {}
    for r, row in enumerate([3, 0, 5, 1]):
        for pi in sorted({p // page_size for p in range(kv_lens[r] - q_lens[r], kv_lens[r])}):
            held[row, pi] = table[row, pi] = next(free)
    before = pages.clone()
    g = torch.Generator(device="cuda").manual_seed(hd + rotary_dim)
    qkv = (torch.randn(T, nh + 2 * nkv, hd, device="cuda", generator=g)
           * torch.exp(0.5 * torch.randn(hd, device="cuda", generator=g))).to(dtype)
    inv_freq = (500000.0 ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / max(1, rotary_dim))).float().cuda()
    q = torch.full((T, nh * hd), math.nan, dtype=dtype, device="cuda")
    kept = qkv.clone()
    ops.rope_kv4_store(qkv.flatten(1), nh, nkv, hd, ctx, _view(pages, table.cuda(), page_size), inv_freq if rotary_dim else None,
                       rotary_dim, q)
    ops.check_status()
    assert torch.equal(qkv, kept)
    want = _turned(qkv[:, :nh + nkv], ctx.positions, inv_freq, rotary_dim)
    # sine, cosine, two products and a sum in 32-bit, each off by half a step of 2^-24 of numbers up to |x0| + |x1|; one rounding
    off = (q.view(T, nh, hd).double() - want[:, :nh]).abs()
    near = torch.finfo(dtype).eps / 2 * want[:, :nh].abs() + 8 * 2.0 ** -24 * qkv[:, :nh].double().abs().amax(-1, keepdim=True)
    assert bool((off <= near).all())
    # codes and scales to the bit, at their places, and no other byte touched
    expect = before.cpu()
    kc, ks = rounded(want[:, nh:].float().to(dtype))
    vc, vs = rounded(qkv[:, nh + nkv:])
    t = 0
    for r, row in enumerate([3, 0, 5, 1]):
        for pos in range(kv_lens[r] - q_lens[r], kv_lens[r]):
            put(expect, table[row], page_size, pos, kc[t].cpu(), ks[t].cpu(), vc[t].cpu(), vs[t].cpu())
            t += 1
    assert torch.equal(pages.cpu(), expect)
    # read back: exact in either type
    k, v = (torch.empty(T, nkv, hd, dtype=dtype, device="cuda") for _ in range(2))
    rows = torch.tensor([3, 0, 5, 1], dtype=torch.int32).cuda()[ctx.token_req.long()]
    ops.read_kv4(_view(pages, table.cuda(), page_size), nkv, hd, rows, ctx.positions, k, v)
    ops.check_status()
    assert torch.equal(k.double(), values_of(kc, ks)) and torch.equal(v.double(), values_of(vc, vs))
    # without storing: the queries alone
    again = pages.clone()
    q2 = torch.empty_like(q)
    ops.rope_kv4_store(qkv.flatten(1), nh, nkv, hd, ctx, _view(pages, table.cuda(), page_size), inv_freq if rotary_dim else None,
                       rotary_dim, q2, store=False)
    ops.check_status()
    assert torch.equal(q2, q) and torch.equal(pages, again)


@pytest.mark.parametrize("dtype", DTYPES)
def test_store_rounds_at_the_borders(ops, dtype):
    """Whole groups of borders between two codes, of the numbers next to them, of zeros, of numbers too small and too large, and of
    ones that are none."""
    step_of = torch.finfo(dtype).eps
    rows = []
    for top in (7.0, 1.0, 3.7, 1e-3, 2.0 ** -99, 2.0 ** -101, 2.0 ** -130, 1e30, 0.0):
        top = torch.tensor(top).to(dtype).double()
        s = float(scale_of(top))
        k = torch.arange(-8, 8, dtype=torch.float64) + 0.5
        x = (k * s).clamp(-float(top), float(top))
        rows += [torch.cat([x, x]), torch.cat([x * (1 + step_of), x * (1 - step_of)]).clamp(-float(top), float(top))]
        rows[-1][5], rows[-2][5] = float(top), -float(top)
    for bad in (math.inf, -math.inf, math.nan):
        rows.append(torch.linspace(-3, 3, 32, dtype=torch.float64))
        rows[-1][11] = bad
    x = torch.stack(rows).to(dtype).cuda()
    n = len(rows)
    nkv = 1
    qkv = torch.stack([torch.zeros_like(x), x, x], 1)
    ctx = step([n], [n])
    pages, table = _pool(1, n, nkv, 32, 16)
    ops.rope_kv4_store(qkv.flatten(1), 1, nkv, 32, ctx, _view(pages, table, 16), None, 0, torch.empty(n, 32, dtype=dtype, device="cuda"))
    k, v = (torch.empty(n, nkv, 32, dtype=torch.float32, device="cuda") for _ in range(2))
    ops.read_kv4(_view(pages, table, 16), nkv, 32, torch.zeros(n, dtype=torch.int32, device="cuda"), ctx.positions, k, v)
    ops.check_status()
    want = values_of(*rounded(x)).float()
    for got in (k[:, 0], v[:, 0]):
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))
    assert bool(torch.isnan(want[-3:]).all()) and not bool(torch.isnan(want[:-3]).any())


# ------------------------------------------------------------------ attention
def _case(ops, dtype, nh, nkv, hd, q_lens, kv_lens, window=0, first=0, page_size=16, fixed=False, seed=0, bad=(), spread=0.4,
          extra=0, scale=None):
    """Attention over a cache written by the restated layout; every place of no visible token holds 0xff.  ``bad``: (request,
    position) whose key and value are no numbers; rows that see one have to be NaN, the others untouched by it."""
    g = torch.Generator(device="cuda").manual_seed(1000 * seed + sum(kv_lens) + hd)
    R, T = len(q_lens), sum(q_lens)
    ctx = step(q_lens, kv_lens, fixed=fixed)
    pages, table = _pool(R, max(kv_lens), nkv, hd, page_size, seed)
    scale = 1.0 / math.sqrt(hd) if scale is None else scale
    q = (torch.randn(T, nh * hd + extra, device="cuda", generator=g) * 1.5).to(dtype)
    K, V, steps = [], [], []
    host = pages.cpu()
    for r, L in enumerate(kv_lens):
        k, v = (torch.randn(L, nkv, hd, device="cuda", generator=g) * torch.exp(spread * torch.randn(hd, device="cuda", generator=g))
                for _ in range(2))
        for rr, pos in bad:
            if rr == r:
                k[pos], v[pos] = math.nan, math.inf
        (kc, ks), (vc, vs) = rounded(k), rounded(v)
        K.append(values_of(kc, ks))
        V.append(values_of(vc, vs))
        steps.append(vs.repeat_interleave(32, -1))
        lo = max(0, L - q_lens[r] - window + 1) if window else 0
        kr, vr = row_bytes(kc, False).cpu(), row_bytes(vc, True).cpu()
        G = hd // 32
        sk, sv = (s.to(torch.bfloat16).contiguous().view(torch.uint8).view(L, nkv, 2 * G).cpu() for s in (ks, vs))
        for pos in range(L):
            if lo <= pos or pos < first:                                # others have been given back
                tile, i = host[int(table[r, pos // page_size]), :, pos % page_size // 16], pos % 16
                tile[:, i * hd // 2:(i + 1) * hd // 2] = kr[pos]
                tile[:, 8 * hd + i * hd // 2:8 * hd + (i + 1) * hd // 2] = vr[pos]
                tile[:, 16 * hd + i * 2 * G:16 * hd + (i + 1) * 2 * G] = sk[pos]
                tile[:, 17 * hd + i * 2 * G:17 * hd + (i + 1) * 2 * G] = sv[pos]
        for pi in range(table.shape[1]):                                # whole pages between the first tokens and the window
            if all(first <= p < lo for p in range(pi * page_size, (pi + 1) * page_size)) and (pi + 1) * page_size <= lo:
                table[r, pi] = -1
    pages.copy_(host)
    out = torch.full((T, nh * hd), math.nan, dtype=dtype, device="cuda")
    ops.paged_attention_kv4(q, nh, nkv, hd, ctx, _view(pages, table, page_size, window or None), scale, window, out, first=first)
    ops.check_status()
    t = 0
    for r, (n, L) in enumerate(zip(q_lens, kv_lens)):
        qr = q[t:t + n, :nh * hd].view(n, nh, hd)
        got = out[t:t + n].view(n, nh, hd).double()
        blind = torch.isnan(K[r]).any(-1).any(-1) | torch.isnan(V[r]).any(-1).any(-1)
        k0 = torch.where(blind[:, None, None], torch.zeros_like(K[r]), K[r])
        v0 = torch.where(blind[:, None, None], torch.full_like(V[r], math.nan), V[r])
        want, size, per_step = attention(qr, k0, v0, L, scale, window, first, steps[r])
        pos, key = torch.arange(L - n, L, device="cuda")[:, None], torch.arange(L, device="cuda")
        sees = (key <= pos) & ((key > pos - window) | (key < first)) if window else key <= pos
        spoilt = (sees & blind).any(-1)
        assert bool(torch.isnan(got[spoilt]).all()), r
        # Scores: within a group of 32 dims an accumulator holds at most 1,039 |q|_1 (a code's 1,024 + 15, and 1,032 taken off) with
        # bfloat16 rows, and 36 additions each lose at most 2^-24 of that; with 32-bit rows 7 |q|_1 and three times the additions.
        # An exponential of 2^-22, the sum over L weights and the merges are within 2^-18 of a weight.  With bfloat16 rows a
        # weight times its scale is rounded (half a step: 2^-8), codes of up to 143 of it are summed over 32 tokens and 136 times
        # their weights taken off again (36 additions), and the result is rounded.
        reach = (qr.double().abs().unflatten(-1, (-1, 32)).sum(-1).amax(0).amax(0) * torch.nan_to_num(k0).abs().unflatten(-1, (-1, 32)).amax(-1).amax(0).amax(0) / 7).sum().item()
        wide = dtype == torch.float32
        lost = 36 * 2.0 ** -24 * abs(scale) * reach * (3 * 7 if wide else 1039)
        share = 2 * lost + 2.0 ** -18 + (0.0 if wide else 2.0 ** -8)
        tol = share * size + (2.0 ** -24 if wide else 2.0 ** -8) * want.abs() + (0.0 if wide else 36 * 143 * 2.0 ** -24 * per_step)
        clear = ~spoilt
        assert bool(((got - want).abs() <= tol)[clear].all()), (r, ((got - want).abs() / tol.clamp_min(1e-30))[clear].max().item())
        t += n


LAYOUTS = [(4, 1, 32), (8, 2, 64), (3, 3, 96), (32, 8, 128), (16, 1, 128), (14, 2, 64), (5, 1, 160), (4, 2, 192), (2, 2, 224), (8, 4, 256),
           (40, 1, 64)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nh, nkv, hd", LAYOUTS)
def test_single_tokens(ops, dtype, nh, nkv, hd):
    _case(ops, dtype, nh, nkv, hd, [1] * 6, [1, 2, 16, 17, 129, 1000])
    _case(ops, dtype, nh, nkv, hd, [1] * 4, [40, 41, 500, 700], window=33, first=5, page_size=32)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nh, nkv, hd", LAYOUTS)
def test_portions(ops, dtype, nh, nkv, hd):
    _case(ops, dtype, nh, nkv, hd, [1, 2, 15, 40], [64, 2, 15, 81])
    _case(ops, dtype, nh, nkv, hd, [3, 1, 33], [300, 90, 120], window=20, first=4)


@pytest.mark.parametrize("nh, nkv, hd", [(8, 2, 64), (4, 1, 128), (3, 3, 64)])
def test_prompts_on_the_prompt_kernel(ops, nh, nkv, hd):
    """Portions long enough to be expanded, beside single tokens and short portions, on every edge of its tiles."""
    bf16 = torch.bfloat16
    _case(ops, bf16, nh, nkv, hd, [128, 1, 200], [128, 70, 333])
    _case(ops, bf16, nh, nkv, hd, [1, 257, 3], [9, 300, 64], page_size=32)
    _case(ops, bf16, nh, nkv, hd, [130], [700], window=64, first=4)
    _case(ops, bf16, nh, nkv, hd, [150, 300], [150, 900], window=100, first=70)
    _case(ops, bf16, nh, nkv, hd, [129], [1000], window=1, first=1, page_size=64)
    _case(ops, bf16, nh, nkv, hd, [140], [600], window=33, first=0)
    _case(ops, bf16, nh, nkv, hd, [140], [600], window=300, first=1000)
    _case(ops, bf16, nh, nkv, hd, [140], [600], window=40, first=4, fixed=True)
    _case(ops, bf16, nh, nkv, hd, [150, 140], [200, 400], bad=[(0, 60), (1, 399)])
    _case(ops, bf16, nh, nkv, hd, [150], [500], window=50, first=4, bad=[(0, 3), (0, 420)])
    _case(ops, bf16, nh, nkv, hd, [150], [200], scale=-0.3)


@pytest.mark.parametrize("window, first", [(1, 0), (1, 1), (1, 40), (16, 16), (17, 3), (64, 0), (64, 64), (200, 7), (5000, 4), (31, 1000)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_windows(ops, dtype, window, first):
    _case(ops, dtype, 8, 2, 64, [1, 1, 1, 1, 1], [1, 15, 64, 65, 333], window, first)
    _case(ops, dtype, 4, 4, 32, [7, 33, 2], [7, 210, 66], window, first, page_size=64)


@pytest.mark.parametrize("dtype", DTYPES)
def test_numbers_that_are_none(ops, dtype):
    """Rows that see a key or value that is no number give NaN; rows whose window has passed it, or that come before it, do not."""
    _case(ops, dtype, 8, 2, 64, [1, 1, 1], [50, 200, 200], window=40, first=4, bad=[(0, 30), (1, 100), (2, 2)])
    _case(ops, dtype, 4, 2, 128, [30, 20], [60, 20], bad=[(0, 45), (1, 19)])
    _case(ops, dtype, 4, 2, 32, [30], [90], window=10, first=3, bad=[(0, 55), (0, 70)])


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_longer_than_the_queries_and_any_scale(ops, dtype):
    _case(ops, dtype, 8, 2, 64, [1, 3], [100, 70], extra=2 * 2 * 64)
    _case(ops, dtype, 8, 2, 64, [1, 3], [100, 70], scale=0.0)
    _case(ops, dtype, 8, 2, 64, [1, 3], [100, 70], scale=-0.4)
    _case(ops, dtype, 8, 2, 64, [1, 3], [100, 70], scale=3.0)


def test_split_and_whole_contexts_agree(ops):
    """A captured launch cuts contexts without knowing their length: most of the blocks of a short one have nothing to do."""
    for fixed in (False, True):
        _case(ops, torch.bfloat16, 8, 2, 64, [1, 1], [3, 9000], fixed=fixed)
        _case(ops, torch.bfloat16, 8, 2, 128, [20], [700], fixed=fixed)
        _case(ops, torch.float32, 4, 1, 32, [1] * 3, [1, 40, 5000], fixed=fixed, window=100, first=4)


def test_many_requests(ops):
    _case(ops, torch.bfloat16, 8, 4, 64, [1] * 100, [1 + 37 * i % 300 for i in range(100)])


def test_a_page_that_is_not_held_is_reported(ops):
    nh, nkv, hd = 4, 2, 64
    pages, table = _pool(2, 64, nkv, hd, 16)
    pages.zero_()
    table[1, 1], table[0, 2] = -1, pages.shape[0]
    ctx = step([1, 1], [64, 64])
    q = torch.randn(2, nh * hd, device="cuda").bfloat16()
    out = torch.empty_like(q)
    ops.paged_attention_kv4(q, nh, nkv, hd, ctx, _view(pages, table, 16), 0.1, 0, out)
    with pytest.raises(ops.KernelError, match="page"):
        ops.check_status()
    ctx = step([1, 1], [48, 20])                                        # both new tokens belong on such a page
    before = pages.clone()
    qkv = torch.randn(2, (nh + 2 * nkv) * hd, device="cuda").bfloat16()
    ops.rope_kv4_store(qkv, nh, nkv, hd, ctx, _view(pages, table, 16), None, 0, out)
    with pytest.raises(ops.KernelError, match="page"):
        ops.check_status()
    assert torch.equal(pages, before)
    k, v = (torch.full((3, nkv, hd), 9.0, device="cuda") for _ in range(2))
    ops.read_kv4(_view(pages, table, 16), nkv, hd, torch.tensor([0, 1, 7], dtype=torch.int32, device="cuda"),
                 torch.tensor([40, 5, 0], dtype=torch.int32, device="cuda"), k, v)
    with pytest.raises(ops.KernelError, match="page"):
        ops.check_status()
    assert not k[0].any() and not k[2].any() and not v[0].any()


def test_the_store_reports_a_negative_position(ops):
    nh, nkv, hd = 4, 2, 64
    pages, table = _pool(2, 64, nkv, hd, 16)
    ctx = step([1, 1], [20, 20])
    ctx.positions[0] = -17
    before, qkv = pages.clone(), torch.randn(2, (nh + 2 * nkv) * hd, device="cuda").bfloat16()
    ops.rope_kv4_store(qkv, nh, nkv, hd, ctx, _view(pages, table, 16), None, 0, torch.empty(2, nh * hd, dtype=qkv.dtype, device="cuda"))
    with pytest.raises(ops.KernelError, match="page"):
        ops.check_status()
    own = table[1, 1].long()
    assert torch.equal(torch.cat([pages[:own], pages[own + 1:]]), torch.cat([before[:own], before[own + 1:]]))
    assert not torch.equal(pages[own], before[own])


def test_captured_steps_on_growing_contexts_and_another_stream(ops):
    """A step of store and attention, captured once and replayed as the lengths grow, beside the same calls made eagerly on
    another stream."""
    nh, nkv, hd, R, page = 8, 2, 128, 3, 16
    g = torch.Generator(device="cuda").manual_seed(5)
    inv_freq = (10000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)).float().cuda()
    pages, table = _pool(R, 400, nkv, hd, page)
    other = pages.clone()
    lens = np.array([0, 30, 141], dtype=np.int32)

    def run(ctx, qkv, pool, q, out):
        view = _view(pool, table, page, 100)
        ops.rope_kv4_store(qkv, nh, nkv, hd, ctx, view, inv_freq, hd, q)
        ops.paged_attention_kv4(q, nh, nkv, hd, ctx, view, hd ** -0.5, 100, out, first=2)

    for r in range(R):                                                  # what the requests hold already
        if lens[r]:
            ctx = step([int(lens[r])], [int(lens[r])], rows=[r])
            qkv = torch.randn(int(lens[r]), (nh + 2 * nkv) * hd, device="cuda", generator=g).bfloat16()
            for pool in (pages, other):
                run(ctx, qkv, pool, *(torch.empty(int(lens[r]), nh * hd, dtype=torch.bfloat16, device="cuda") for _ in range(2)))
    static = step([1] * R, (lens + 1).tolist(), fixed=True)
    qkv_in = torch.zeros(R, (nh + 2 * nkv) * hd, dtype=torch.bfloat16, device="cuda")
    q, out = (torch.zeros(R, nh * hd, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    scratch = pages.clone()
    run(static, qkv_in, scratch, q, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(static, qkv_in, pages, q, out)
    side = torch.cuda.Stream()
    for turn in range(40):
        lens += 1
        now = step([1] * R, lens.tolist())
        fresh = torch.randn(R, (nh + 2 * nkv) * hd, device="cuda", generator=g).bfloat16()
        for name in ("positions", "kv_len"):
            getattr(static, name).copy_(getattr(now, name))
        qkv_in.copy_(fresh)
        graph.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            q2, out2 = (torch.empty(R, nh * hd, dtype=torch.bfloat16, device="cuda") for _ in range(2))
            run(now, fresh, other, q2, out2)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(q, q2) and torch.equal(pages, other)
        # (the two cut the keys differently: sums in another order, probabilities against another reference)
        assert bool(((out.float() - out2.float()).abs() <= 2.0 ** -6 * out2.float().abs() + 2.0 ** -7).all()), turn
    ops.check_status()
