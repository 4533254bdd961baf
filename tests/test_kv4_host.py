"""What the operators of a 4-bit cache refuse, without a GPU: their checks run on plain tensors and nothing is launched."""
import types

import pytest
import torch

from llm_singularity_b200 import kernels as ops
from llm_singularity_b200.parts.base import KV4CacheView

NH, NKV, HD, PAGE = 4, 2, 64, 16


class Launched(Exception):
    pass


@pytest.fixture
def checks(monkeypatch):
    """The checks as they are but for the device; a launch raises ``Launched``."""
    def req(t, name, dtype=None, dim=None, contiguous=True):
        if dtype is not None and t.dtype != dtype:
            raise ops.KernelError(f"{name} must be {dtype}, got {t.dtype}")
        if dim is not None and t.dim() != dim:
            raise ops.KernelError(f"{name} must have {dim} dims")
        if contiguous and not t.is_contiguous():
            raise ops.KernelError(f"{name} must be contiguous")
        return t

    def call(*a):
        raise Launched

    monkeypatch.setattr(ops, "_req", req)
    monkeypatch.setattr(ops, "_call", call)
    monkeypatch.setattr(ops, "_same_device", lambda what, *t: None)
    monkeypatch.setattr(ops, "_stream", lambda t: None)
    monkeypatch.setattr(ops, "_kv4_room", lambda *a: 296)
    monkeypatch.setattr(ops, "_lib", lambda name: types.SimpleNamespace(lsb_attention_kv4_slot=lambda *a: 8))


def _ctx(q_lens=(1, 3), kv_lens=(5, 3)):
    import numpy as np
    q, kv = np.array(q_lens), np.array(kv_lens)
    z = torch.zeros(8, dtype=torch.int32)
    return types.SimpleNamespace(n_tokens=int(q.sum()), n_requests=len(q), h_q_len=q, h_kv_len=kv, max_q_len=int(q.max()),
                                 max_kv_len=int(kv.max()), q_start=z, kv_len=z, table_rows=z, positions=z, token_req=z)


def _cache(nkv=NKV, hd=HD, page=PAGE, dtype=torch.uint8, pages=3):
    return KV4CacheView(torch.zeros(pages, nkv, max(1, page // 16), 18 * hd, dtype=dtype), torch.zeros(2, 4, dtype=torch.int32), page, None, 0)


def _attend(**o):
    a = dict(q=torch.zeros(4, NH * HD), nh=NH, nkv=NKV, hd=HD, ctx=_ctx(), cache=_cache(), window=0, first=0, out=torch.zeros(4, NH * HD))
    a.update(o)
    ops.paged_attention_kv4(a["q"], a["nh"], a["nkv"], a["hd"], a["ctx"], a["cache"], 0.1, a["window"], a["out"], first=a["first"])


def test_attention_takes_what_it_says(checks):
    with pytest.raises(Launched):
        _attend()
    with pytest.raises(Launched):
        _attend(q=torch.zeros(4, NH * HD + 128), window=3, first=2)
    with pytest.raises(Launched):
        _attend(q=torch.zeros(4, NH * HD).bfloat16(), out=torch.zeros(4, NH * HD).bfloat16())


@pytest.mark.parametrize("change, says", [
    (dict(q=torch.zeros(4, NH * HD - 1)), "disagree"), (dict(out=torch.zeros(4, NH * HD + 1)), "disagree"),
    (dict(q=torch.zeros(5, NH * HD), out=torch.zeros(5, NH * HD)), "disagree"), (dict(out=torch.zeros(4, NH * HD).bfloat16()), "out"),
    (dict(q=torch.zeros(4, NH * HD).half(), out=torch.zeros(4, NH * HD).half()), "float32 or bfloat16"),
    (dict(q=torch.zeros(8, NH * HD)[::2]), "contiguous"), (dict(nkv=3), "share"), (dict(nkv=0), "share"), (dict(nh=0), "share"),
    (dict(window=-1), "negative"), (dict(first=-1), "negative"), (dict(cache=_cache(nkv=1)), "pages are"),
    (dict(cache=_cache(hd=32)), "pages are"), (dict(cache=_cache(dtype=torch.int8)), "pages"), (dict(cache=_cache(page=8)), "multiple of 16"),
    (dict(hd=48, q=torch.zeros(4, NH * 48), out=torch.zeros(4, NH * 48), cache=_cache(hd=48)), "multiple of 32"),
    (dict(hd=288, q=torch.zeros(4, NH * 288), out=torch.zeros(4, NH * 288), cache=_cache(hd=288)), "up to 256"),
])
def test_attention_refuses(checks, change, says):
    with pytest.raises(ops.KernelError, match=says):
        _attend(**change)


def _store(**o):
    a = dict(qkv=torch.zeros(4, (NH + 2 * NKV) * HD), nh=NH, nkv=NKV, hd=HD, ctx=_ctx(), cache=_cache(), inv=torch.zeros(HD // 2), rot=HD,
             q=torch.zeros(4, NH * HD))
    a.update(o)
    ops.rope_kv4_store(a["qkv"], a["nh"], a["nkv"], a["hd"], a["ctx"], a["cache"], a["inv"], a["rot"], a["q"])


def test_store_takes_what_it_says(checks):
    with pytest.raises(Launched):
        _store()
    with pytest.raises(Launched):
        _store(rot=0, inv=None)
    with pytest.raises(Launched):
        _store(rot=10, inv=torch.zeros(5))


@pytest.mark.parametrize("change, says", [
    (dict(qkv=torch.zeros(4, NH * HD)), "expected"), (dict(q=torch.zeros(4, HD)), "q_out"), (dict(q=torch.zeros(4, NH * HD).bfloat16()), "q_out"),
    (dict(rot=HD + 2), "rotary_dim"), (dict(rot=3), "even"), (dict(inv=torch.zeros(5)), "entries"), (dict(ctx=_ctx((1, 1))), "tokens"),
    (dict(cache=_cache(page=24)), "multiple of 16"), (dict(cache=_cache(nkv=4)), "pages are"),
])
def test_store_refuses(checks, change, says):
    with pytest.raises(ops.KernelError, match=says):
        _store(**change)


@pytest.mark.parametrize("change, says", [
    (dict(k=torch.zeros(3, NKV, HD + 1)), "for each"), (dict(v=torch.zeros(3, NKV, HD).bfloat16()), "v_out"),
    (dict(rows=torch.zeros(2, dtype=torch.int32)), "for each"), (dict(rows=torch.zeros(3)), "token_rows"), ({}, None),
])
def test_reading_back(checks, change, says):
    a = dict(rows=torch.zeros(3, dtype=torch.int32), pos=torch.zeros(3, dtype=torch.int32), k=torch.zeros(3, NKV, HD), v=torch.zeros(3, NKV, HD))
    a.update(change)
    with pytest.raises(Launched if says is None else ops.KernelError, match=says):
        ops.read_kv4(_cache(), NKV, HD, a["rows"], a["pos"], a["k"], a["v"])


def test_no_path_without_a_gpu():
    with pytest.raises(ops.KernelError, match="CUDA"):
        _attend()
    with pytest.raises(ops.KernelError, match="CUDA"):
        _store()
