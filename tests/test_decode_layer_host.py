"""CPU tests of what a decode layer keeps on the host: pages, table and lengths."""
from __future__ import annotations

import pytest
import torch

from vkernels_amd.decode_layer import DecodeLayer


def _layer(sequences=3, pages=10, max_positions=64, page_size=4):
    w = torch.zeros
    return DecodeLayer(None, w(32, 64), w(32, 32), w(32, 4), kv_heads=1, head_dim=16, top_k=2, sequences=sequences,
                       pages=pages, page_size=page_size, max_positions=max_positions)


def _state(layer):
    return sorted(layer.free), [list(x) for x in layer.owned], list(layer.lens), layer.table.tolist(), layer.lens_dev.tolist()


def _consistent(layer, pages):
    assert sorted(layer.free + sum(layer.owned, [])) == list(range(pages))
    assert layer.lens_dev.tolist() == layer.lens
    for b, owned in enumerate(layer.owned):
        assert layer.table[b].tolist() == owned + [-1] * (layer.table.shape[1] - len(owned))
        assert len(owned) * layer.page_size >= layer.lens[b]


@pytest.mark.parametrize("by", [[4, 100, 0], [41, 0, 0], [12, 12, 17], [0, 0, 65]])
def test_a_refused_growth_takes_nothing(by):
    """No page left in the middle of the sequences, for the last one, or no column left in the table: pages,
    table and lengths are as before, and what fits is served afterwards."""
    layer = _layer(pages=10 if by[2] < 65 else 40)
    pages = len(layer.free)
    layer._grow([3, 0, 1])
    before = _state(layer)
    with pytest.raises(RuntimeError, match="no page left for sequence [012]"):
        layer._grow(by)
    assert _state(layer) == before
    _consistent(layer, pages)
    layer._grow([9, 8, 7])
    assert layer.lens == [12, 8, 8]
    _consistent(layer, pages)


def test_growth_takes_the_pages_that_are_needed():
    layer = _layer()
    for by in ([1, 0, 4], [3, 0, 1], [1, 1, 0], [16, 3, 0], [3, 0, 3]):
        layer._grow(by)
        _consistent(layer, 10)
        assert [len(x) for x in layer.owned] == [-(-n // 4) for n in layer.lens]
    assert layer.lens == [24, 4, 8] and len(layer.free) == 1


def test_lengths_of_a_refused_call_are_taken_back():
    """Rows or queries that the cache's operators refuse (here: all of them, without a GPU)."""
    layer = _layer()
    layer._grow([3, 0, 1])
    rows = torch.zeros((5, 1, 16))
    with pytest.raises(ValueError):
        layer.prefill(rows, rows, [2, 3, 0])
    assert layer.lens == [3, 0, 1]
    with pytest.raises(ValueError):
        layer.attend(torch.zeros((3, 2, 16)), rows[:3], rows[:3])
    assert layer.lens == [3, 0, 1]
    _consistent(layer, 10)
    layer._grow([1, 3, 0])
    assert layer.lens == [4, 3, 1]
    _consistent(layer, 10)
