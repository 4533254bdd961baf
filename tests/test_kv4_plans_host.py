"""Which launches attention over a 4-bit cache makes of a step, and with what, without a GPU."""
import types

import numpy as np
import pytest
import torch

from llm_singularity_b200 import kernels as ops
from llm_singularity_b200.parts.base import KV4CacheView

ROOM = 296


@pytest.fixture
def calls(monkeypatch):
    """Every launch as (entry point, arguments); the checks of devices are off."""
    made = []
    monkeypatch.setattr(ops, "_req", lambda t, name, dtype=None, dim=None, contiguous=True: t)
    monkeypatch.setattr(ops, "_call", lambda lib, fn, *a: made.append((fn, [getattr(x, "value", x) for x in a])))
    monkeypatch.setattr(ops, "_same_device", lambda what, *t: None)
    monkeypatch.setattr(ops, "_stream", lambda t: "stream")
    monkeypatch.setattr(ops, "_kv4_room", lambda lib, hd, eights, form, device: ROOM // max(1, form))
    monkeypatch.setattr(ops, "_lib", lambda name: types.SimpleNamespace(lsb_attention_kv4_slot=lambda *a: 8))
    return made


def _step(q_lens, kv_lens, fixed=False):
    q, kv = np.array(q_lens, dtype=np.int32), np.array(kv_lens, dtype=np.int32)
    start = torch.from_numpy(np.concatenate([[0], np.cumsum(q)]).astype(np.int32))
    return types.SimpleNamespace(n_tokens=int(q.sum()), n_requests=len(q), h_q_len=q, h_kv_len=kv, max_q_len=int(q.max()),
                                 max_kv_len=int(kv.max()), q_start=start, kv_len=torch.from_numpy(kv),
                                 table_rows=torch.arange(len(q), dtype=torch.int32), fixed_launch=fixed)


def _attend(ctx, nh=8, nkv=2, hd=64, window=0, first=0, dtype=torch.bfloat16, width=None):
    width = -(-int(ctx.h_kv_len.max()) // 16) if width is None else width
    cache = KV4CacheView(torch.zeros(3, nkv, 1, 18 * hd, dtype=torch.uint8), torch.zeros(len(ctx.h_q_len), width, dtype=torch.int32), 16,
                         window or None, 0)
    q = torch.zeros(ctx.n_tokens, nh * hd, dtype=dtype)
    ops.paged_attention_kv4(q, nh, nkv, hd, ctx, cache, 0.1, window, torch.empty_like(q), first=first)


@pytest.mark.parametrize("window, first", [(0, 0), (50, 0), (50, 4)])
def test_lengths_written_by_a_launch_are_waited_for(calls, window, first):
    """The prompt kernel reads a request's length and row before it waits for the launch before it, as it may with a step's own
    metadata.  Behind the launch that unpacks the cache they are that launch's results: it has to be told, and only then."""
    ctx = _step([200, 1], [400, 30])
    _attend(ctx, window=window, first=first)
    (unpack, of_unpack), (prompt, of_prompt) = [c for c in calls if c[0] in ("lsb_expand_kv4", "lsb_prefill_attention_tc5_first")]
    its_len, its_rows = of_unpack[10], of_unpack[9]
    assert (unpack, prompt) == ("lsb_expand_kv4", "lsb_prefill_attention_tc5_first")
    assert of_prompt[6] == its_len and of_prompt[7] == its_rows and its_len not in (ctx.kv_len.data_ptr(), ctx.table_rows.data_ptr())
    assert of_prompt[-3:] == [first, 1, "stream"]


def test_a_step_s_own_lengths_are_not(calls, monkeypatch):
    from llm_singularity_b200.parts.base import KVCacheView
    monkeypatch.setattr(ops, "_lib", lambda name: types.SimpleNamespace(lsb_prefill_attention_tc5_supported=lambda *a: 1))
    ctx = _step([200], [400])
    cache = KVCacheView(torch.zeros(3, 2, 16, 64).bfloat16(), torch.zeros(3, 2, 16, 64).bfloat16(), torch.zeros(1, 25, dtype=torch.int32), 16, 50, 0)
    q = torch.zeros(200, 512).bfloat16()
    ops.paged_attention(q, 8, 2, 64, ctx, cache, 0.1, 50, torch.empty(200 * 512 + 8).bfloat16()[:200 * 512].view(200, 512), first=4)
    fn, a = calls[0]
    assert fn == "lsb_prefill_attention_tc5_first" and a[6] == ctx.kv_len.data_ptr() and a[-3:] == [4, 0, "stream"]


def _plan(ctx, hd=128, nh=32, nkv=8, window=0, first=0, capacity=131072, lib="attention_kv4"):
    return {p[0]: p for p in ops._kv4_plan(ctx, lib, nh, nkv, hd, window, first, capacity, "cuda:0")}


def test_a_launch_is_sized_by_its_own_requests(calls):
    """A conversation of 131,072 tokens beside two prompts of 200: the prompts' unpacked cache has 13 tiles each and two to spare, and
    few tokens beside a long portion are not split as if they were long."""
    alone = _plan(_step([200, 200], [200, 200]))
    beside = _plan(_step([1, 200, 200], [131072, 200, 200]))
    assert alone[3][6] == beside[3][6] == 15 and set(beside) == {1, 3}
    lib = "attention_kv4_f32"                                    # (no unpacking there: split over a cluster, or spread)
    assert _plan(_step([40], [64]), lib=lib)[2][5:] == _plan(_step([1, 40], [131072, 64]), lib=lib)[2][5:]
    assert _plan(_step([1], [64]), lib=lib)[1][5:] == _plan(_step([1, 40], [64, 131072]), lib=lib)[1][5:]


def test_a_captured_launch_is_sized_by_the_table(calls):
    assert _plan(_step([200], [200], fixed=True), capacity=1600)[3][6] == 102


@pytest.mark.parametrize("lib", ["attention_kv4", "attention_kv4_f32"])
@pytest.mark.parametrize("q_lens, kv_lens", [([1], [64]), ([1] * 8, [4096] * 8), ([40], [64]), ([1] * 64, list(range(1000, 7400, 100)))])
def test_a_window_wider_than_any_context_changes_no_plan(calls, lib, q_lens, kv_lens):
    far = dict(window=(1 << 30) - 1, first=1 << 30)
    assert _plan(_step(q_lens, kv_lens), lib=lib, **far) == _plan(_step(q_lens, kv_lens), lib=lib)


def test_a_spread_launch_has_the_blocks_that_fit_of_its_own_kernel(calls, monkeypatch):
    """The kernel that spreads chunks has more registers than the one with clusters, and fewer of its blocks fit."""
    monkeypatch.setattr(ops, "_kv4_room", lambda lib, hd, eights, spread, device: 296 if spread else 444)
    for ctx in (_step([1], [131072]), _step([1] * 8, [9000] * 8, fixed=True)):
        assert _plan(ctx, hd=64, nh=32, nkv=2)[1][6] == 296                 # 16 rows a block


@pytest.mark.parametrize("requests, window, first", [(1, 1024, 4), (8, 1024, 4), (64, 1024, 4), (32, 4000, 0), (8, 100000, 4), (1, 100000, 0)])
def test_a_captured_launch_with_a_window_is_planned_for_it(calls, requests, window, first):
    """However wide the block tables are, a request is seen in its window only: the plan is that of a step of requests past it."""
    captured = _plan(_step([1] * requests, [5] * requests, fixed=True), hd=64, window=window, first=first)[1]
    eager = _plan(_step([1] * requests, [131072] * requests), hd=64, window=window, first=first)[1]
    assert captured[5:] == eager[5:] and (captured[6] == 0) == (window < 5000)
    assert _plan(_step([1] * requests, [5] * requests, fixed=True), hd=64)[1][6] > 0


def test_clusters_are_counted_by_those_that_fit(calls, monkeypatch):
    """Blocks of 296 places may be 40 clusters of 7 by number, but where only 34 fit they take two rounds: fewer splits, or spread."""
    monkeypatch.setattr(ops, "_kv4_room", lambda lib, hd, eights, form, device: {0: 296, 1: 296, 2: 148, 3: 96, 4: 72, 5: 56, 6: 46, 7: 34, 8: 34}[form])
    at = lambda requests, nkv: _plan(_step([1] * requests, [1500] * requests), nh=nkv, nkv=nkv)[1][5:7]
    assert at(5, 8) == (6, 0)                                    # 40 row tiles
    assert at(4, 8) == (8, 0) and at(34, 1) == (8, 0) and at(35, 1) == (6, 0)


def test_many_short_requests_are_not_spread(calls, monkeypatch):
    """What a block begins anew counts: 64 requests of up to 1,000 tokens run faster a block each, of up to 8,100 spread."""
    monkeypatch.setattr(ops, "_kv4_room", lambda lib, hd, eights, form, device: 444 // max(1, form))
    lens = lambda lo, hi: [lo + (hi - lo) * ((7 * i + 3) % 64) // 63 for i in range(64)]
    assert _plan(_step([1] * 64, lens(300, 1000)))[1][6] == 0
    assert _plan(_step([1] * 64, lens(1000, 8100)))[1][6] == 444
    assert _plan(_step([1] * 64, [9000] * 64), window=1024, first=4)[1][6] == 0


def test_portions_that_pass_the_limit_together_go_one_after_the_other(calls):
    """Three prompts of 131,072 tokens, single tokens between them: each is unpacked by itself, with the launch arrays of its own place."""
    ctx = _step([1, 300, 1, 200, 500], [40, 131072, 9, 131072, 100000])
    plan = ops._kv4_plan(ctx, "attention_kv4", 32, 8, 128, 0, 0, 131072, "cuda:0")
    assert [p for p in plan if p[0] == 3] == [(3, 4 * i, 1, 4 * n, 2, 1, 8194, 0) for i, n in ((1, 300), (3, 200), (4, 500))]
    assert [p[0] for p in plan] == [1, 3, 3, 3]
    assert [p[:3] for p in ops._kv4_plan(_step([300, 200], [100000, 100000]), "attention_kv4", 32, 8, 128, 0, 0, 131072, "cuda:0")] == [(3, 0, 2)]
    assert [p[0] for p in ops._kv4_plan(_step([300, 200], [300000, 300]), "attention_kv4", 32, 8, 128, 0, 0, 300000, "cuda:0")] == [2]


def test_a_device_that_takes_no_such_kernel_is_left_to_say_so(calls, monkeypatch):
    monkeypatch.setattr(ops, "_kv4_room", lambda *a: 0)
    for ctx in (_step([1] * 3, [100] * 3), _step([40], [5000]), _step([1], [5], fixed=True)):
        assert len(ops._kv4_plan(ctx, "attention_kv4_f32", 8, 2, 64, 0, 0, 8192, "cuda:0")) == 1
