"""A decode layer goes on after a call that it refused as if that call had not been made: the steps behind it
are checked against the definition on what the cache should hold."""
from __future__ import annotations

import pytest
import torch

from test_gpu_decode_layer import _layer

pytestmark = pytest.mark.gpu


def _steps(layer, normal, cfg, n):
    hidden = normal(3, cfg.H)
    for _ in range(n):
        hidden = layer.step(hidden)
        hidden = (hidden.float() / hidden.float().std(-1, keepdim=True)).to(torch.bfloat16)
    assert sorted(layer.free + sum(layer.owned, [])) == list(range(24))


@pytest.mark.parametrize("budget", [None, 40])
def test_steps_after_the_pages_ran_out(hip_lib, budget):
    layer, normal, cfg = _layer(budget, False)
    layer.prefill(normal(40, 2, 64), normal(40, 2, 64), [17, 3, 20])
    with pytest.raises(RuntimeError, match="no page left"):
        layer.prefill(normal(360, 2, 64), normal(360, 2, 64), [120, 120, 120])
    layer.prefill(normal(25, 2, 64), normal(25, 2, 64), [8, 0, 17])
    _steps(layer, normal, cfg, 30)
    assert layer.steps == 30 and (budget is not None or max(layer.lens) == 67)


@pytest.mark.parametrize("budget", [None, 40])
def test_steps_after_refused_rows_and_queries(hip_lib, budget):
    layer, normal, cfg = _layer(budget, False)
    layer.prefill(normal(40, 2, 64), normal(40, 2, 64), [17, 3, 20])
    with pytest.raises(ValueError):
        layer.prefill(normal(30, 2, 64).half(), normal(30, 2, 64).half(), [10, 10, 10])
    with pytest.raises(ValueError):
        layer.attend(normal(3, 5, 64), normal(3, 2, 64), normal(3, 2, 64))
    assert layer.lens == [17, 3, 20] == layer.lens_dev.tolist()
    _steps(layer, normal, cfg, 30)
    assert layer.steps == 30
