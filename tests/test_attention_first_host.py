"""What attention over a window with first tokens refuses before any launch, without a GPU."""
import types

import numpy as np
import pytest
import torch

from llm_singularity_b200 import kernels as ops
from llm_singularity_b200.parts.base import KVCacheView


@pytest.fixture
def checks(monkeypatch):
    monkeypatch.setattr(ops, "_req", lambda t, name, dtype=None, dim=None, contiguous=True: t)
    launched = []
    monkeypatch.setattr(ops, "_call", lambda lib, fn, *a: launched.append(fn))
    monkeypatch.setattr(ops, "_stream", lambda t: None)
    return launched


def _run(window, first, **o):
    z = torch.zeros(4, dtype=torch.int32)
    ctx = types.SimpleNamespace(n_tokens=4, n_requests=2, h_q_len=np.array([1, 3]), h_kv_len=np.array([9, 5]), max_q_len=3, max_kv_len=9,
                                q_start=z, kv_len=z, table_rows=z)
    cache = KVCacheView(torch.zeros(3, 2, 16, 32), torch.zeros(3, 2, 16, 32), torch.zeros(2, 2, dtype=torch.int32), 16, window or None, 0)
    ops.paged_attention(torch.zeros(4, 128), 4, 2, 32, ctx, cache, 0.1, window, torch.zeros(4, 128), first=first, **o)


def test_which_kernel_is_asked(checks):
    _run(3, 2)
    _run(0, 2)
    _run(3, 0)
    assert checks == ["lsb_paged_attention_generic_first", "lsb_paged_attention_generic", "lsb_paged_attention_generic"]


@pytest.mark.parametrize("o, says", [(dict(first=-1), "negative"), (dict(first=1, only="single"), "rotated"), (dict(first=1, stream=0), "rotated"),
                                     (dict(first=1, decode_rope=(None, False, 0)), "rotated")])
def test_refusals(checks, o, says):
    with pytest.raises(ops.KernelError, match=says):
        _run(3, **o)
    assert not checks
