"""What the C entry point of attention over a 4-bit cache refuses by itself: nothing is launched and nothing is written."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("change", [dict(mode=0), dict(mode=3), dict(splits=0), dict(splits=9), dict(eights=0), dict(eights=3), dict(hd=48), dict(hd=288),
                                    dict(page_size=24), dict(nkv=0), dict(spread=1, parts=None), dict(n_requests=70000)])
def test_refusals(change):
    from llm_singularity_b200 import kernels as ops
    ops.prepare(["attention_kv4"])
    a = dict(mode=1, splits=1, eights=1, hd=64, page_size=16, nkv=1, spread=0, parts=None, n_requests=1)
    a.update(change)
    ints = torch.zeros(64, dtype=torch.int32, device="cuda")
    ints[1], ints[8] = 1, 5                                     # one token, at position 4
    q, out = torch.zeros(1, 64, dtype=torch.bfloat16, device="cuda"), torch.full((1, 64), 9.0, dtype=torch.bfloat16, device="cuda")
    pages = torch.zeros(1, 1, 1, 18 * 64, dtype=torch.uint8, device="cuda")
    p = lambda t, off=0: ctypes.c_void_p(0 if t is None else t.data_ptr() + 4 * off)
    call = lambda **o: ops._lib("attention_kv4").lsb_attention_kv4(
        p(q), 64, p(pages), p(ints), p(ints, 8), p(ints, 16), p(ints, 24), 1, p(out), o["n_requests"], ctypes.c_longlong(1), 1, o["nkv"], o["hd"],
        o["page_size"], 1, ctypes.c_float(0.1), 0, 0, o["mode"], o["eights"], o["splits"], o["spread"], p(o["parts"]),
        ops._stream(out))
    assert call(**a) != 0
    torch.cuda.synchronize()
    assert bool((out == 9.0).all())
    a.update(mode=1, splits=1, eights=1, hd=64, page_size=16, nkv=1, spread=0, n_requests=1)
    assert call(**a) == 0
    torch.cuda.synchronize()
    ops.check_status()
    assert not bool(out.any())
