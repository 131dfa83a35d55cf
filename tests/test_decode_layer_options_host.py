"""CPU tests of a decode layer's options that go together with others or do not."""
from __future__ import annotations

import pytest
import torch

from vkernels_amd.decode_layer import DecodeLayer

FP8 = torch.float8_e4m3fn


def _layer(**kw):
    w = torch.zeros
    return DecodeLayer(None, w(32, 64), w(32, 32), w(32, 4), kv_heads=1, head_dim=16, top_k=2, sequences=2, pages=10, page_size=4,
                       max_positions=600, **kw)


@pytest.mark.parametrize("bad", [
    dict(budget=100, window=8), dict(budget=100, scale_blocks=1, cache_dtype=FP8), dict(scale_blocks=1), dict(scale_blocks=3, cache_dtype=FP8),
    dict(scale_blocks=0, cache_dtype=FP8), dict(scale_blocks=8, cache_dtype=FP8),
    dict(scale_blocks=2, cache_dtype=FP8, k_scale=torch.ones(1), v_scale=torch.ones(1))])
def test_options_that_do_not_go_together(bad):
    with pytest.raises(ValueError):
        _layer(**bad)


def test_a_refused_prompt_changes_nothing():
    layer = _layer(rotary=dict(inv_freq=torch.ones(8)))
    k, q = torch.zeros((5, 1, 16)), torch.zeros((5, 2, 16))
    for lengths, queries in (([2, 3], None), ([2, 2], q), ([6, -1], q), ([2, 3], q[:4]), ([2, 3], q.half()), ([2, 3], q)):
        with pytest.raises(ValueError):         # (the last one for want of a GPU)
            layer.prefill(k, k, lengths, q=queries)
    with pytest.raises(ValueError):
        layer.attend(q[:2, :1], k[:2], k[:2])
    assert layer.lens == [0, 0] and layer.positions.tolist() == [0, 0] and len(layer.free) == 10


def test_block_scales_are_the_layers_own():
    layer = _layer(scale_blocks=2, cache_dtype=FP8)
    assert layer.scales["k_scale"].shape == layer.scales["v_scale"].shape == (10, 1, 2)
