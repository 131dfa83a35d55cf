"""GPU tests of the key-value cache's operators at the ends of what their arguments may be, against the
definitions."""
from __future__ import annotations

import pytest
import torch

from test_gpu_kv_cache import BF16, Setup, dev
from vkernels_amd import kv_cache as kv

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window", [2 ** 31 - 17, 2 ** 31 - 16, 2 ** 31 - 1])
@pytest.mark.parametrize("lens", [[40, 0, 130], [1300, 5, 2500]])
def test_a_window_beyond_every_length(hip_lib, window, lens):
    """The largest integers as a window are no window: the same split, results and sums."""
    s = Setup(lens, 2, 4, 64, 16, seed=21)
    out, lse, _ = s.check(window=window, counted=True, sinks=True)
    want, want_lse, _ = s.check(counted=True, sinks=True)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
