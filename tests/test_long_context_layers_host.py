"""Windows asked for where layers have windows of their own, without a GPU."""
from dataclasses import replace

import pytest

import tiny_models
from llm_singularity_b200.config.llama import LlamaConfig
from llm_singularity_b200.config.specs import with_long_context


def _spec(*layers):
    """The small model's layers with (window, first tokens) of their own."""
    spec = LlamaConfig.from_dict(tiny_models.CONFIGS["tiny_b"]).to_model_spec()
    blocks = tuple(replace(b, mixer=replace(b.mixer, window=w, first_tokens=f)) for b, (w, f) in zip(spec.blocks, layers))
    return replace(spec, blocks=blocks + spec.blocks[len(blocks):])


def _rules(spec):
    return [(b.mixer.window, b.mixer.first_tokens) for b in spec.blocks]


def _sees(p, window, first):
    return {j for j in range(p + 1) if window is None or j > p - window or j < (first or 0)}


@pytest.mark.parametrize("own", [(512, None), (512, 4), (4096, None), (9000, None), (9000, 2), (9000, 64), (None, None)])
@pytest.mark.parametrize("window, first", [(4096, 8), (512, 0), (100, 8), (20000, 3)])
def test_no_layer_sees_more_than_it_did(own, window, first):
    (w, f), *rest = _rules(with_long_context(_spec(own), "int4", window, first))
    assert all(r == (window, first) for r in rest)
    for p in (0, 3, 99, 511, 600, 4200, 9500):
        assert _sees(p, w, f) <= _sees(p, *own) & _sees(p, window, first), p
    assert w == min(window, own[0] or window) and f is not None       # (said: a sequence may be longer than the pool)


def test_without_a_window_layers_keep_theirs():
    own = [(512, None), (None, None)]
    assert _rules(with_long_context(_spec(*own), "int4"))[:2] == own


@pytest.mark.parametrize("window, first, says", [(2 ** 32 + 5, 0, "window"), (2 ** 31, 0, "window"), (2 ** 30 + 1, 0, "window"),
                                                 (8, 2 ** 30 + 1, "first_tokens"), (8, 2 ** 64 + 1, "first_tokens")])
def test_lengths_of_more_than_30_bits_are_refused(window, first, says):
    """(Cut to 32 bits, a window of 2^32 + 5 would be one of 5.)"""
    with pytest.raises(ValueError, match=says):
        with_long_context(_spec(), "compute", window, first)
    assert _rules(with_long_context(_spec(), "compute", 2 ** 30, 2 ** 30))[0] == (2 ** 30, 2 ** 30)
