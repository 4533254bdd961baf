"""Which steps with a prompt portion are captured where the cache is held in 4 bits, without a GPU."""
import types

import pytest
import torch

import tiny_models
from llm_singularity_b200 import kernels
from llm_singularity_b200.engine import StepEntry
from llm_singularity_b200.engine.runner import ModelRunner
from long_context_util import Ops


class Asked(Ops):
    kv4_portion_captures = staticmethod(kernels.kv4_portion_captures)


@pytest.fixture(scope="module")
def path(tmp_path_factory):
    return tiny_models.make_model_dir(str(tmp_path_factory.mktemp("m")), "tiny_d")


def _captured(path, tokens, **o):
    """Whether a portion of a length that comes again is."""
    import numpy as np
    runner = ModelRunner(path, dtype="bfloat16", device="cpu", page_size=16, num_pages=8, max_requests=2, ops=Asked(), **o)
    part = np.zeros(tokens, dtype=np.int32)
    keys = [runner._graph_key([StepEntry("a", part, [])], [part], None) for _ in range(2)]
    assert runner._graph_key([StepEntry("a", part[:1], [0])], [part[:1]], None) is not None     # single tokens always are
    return keys[-1] is not None


def test_a_portion_is_captured_only_where_that_costs_no_speed(path):
    """A captured portion makes room for the longest context that the block tables can hold.  Where that is more than its unpacked
    cache may take, capturing would send it to the kernel that unpacks a tile again for every few rows."""
    wide, narrow = 16 * 80000, 16 * 1000
    assert _captured(path, 200, max_model_len=narrow, kv_cache="int4")
    assert not _captured(path, 200, max_model_len=wide, kv_cache="int4")
    assert _captured(path, 200, max_model_len=wide, kv_cache="int4", window=1000, first_tokens=4)      # (a window bounds it)
    assert _captured(path, 100, max_model_len=wide, kv_cache="int4")                                   # (never unpacked)
    assert _captured(path, 200, max_model_len=wide)


@pytest.mark.parametrize("nkv, hd, most", [(8, 128, 65504), (8, 64, 131040), (2, 64, 524256)])
def test_the_width_from_which_it_is_not(nkv, hd, most):
    asked = lambda table, **o: kernels.kv4_portion_captures(o.get("dtype", torch.bfloat16), nkv, hd, o.get("tokens", 2048), table)
    assert asked(most) and not asked(most + 16)
    assert asked(10 ** 7, dtype=torch.float32) and asked(10 ** 7, tokens=127)
    ctx = types.SimpleNamespace(n_requests=1, max_q_len=2048, max_kv_len=2048, fixed_launch=True)
    import numpy as np
    ctx.h_q_len, ctx.h_kv_len = np.array([2048]), np.array([2048])
    room = kernels._kv4_room
    try:
        kernels._kv4_room = lambda *a: 296
        lib, kernels._lib = kernels._lib, lambda name: types.SimpleNamespace(lsb_attention_kv4_slot=lambda *a: 8)
        modes = []
        for table in (most, most + 16):
            ctx.__dict__.pop("_kv4_plans", None)
            modes.append(kernels._kv4_plan(ctx, "attention_kv4", nkv, nkv, hd, 0, 0, table, None)[0][0])
    finally:
        kernels._kv4_room, kernels._lib = room, lib
    assert modes == [3, 2]                                      # (the plan itself says the same)
