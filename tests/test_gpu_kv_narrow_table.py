"""GPU tests of block tables of one column."""
from __future__ import annotations

import pytest
import torch

from test_gpu_kv_window import BF16, FP8, dev
from vkernels_amd import kv_cache as kv

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("block", [0, 8])
def test_a_transposed_row(hip_lib, block):
    """Rows of one element are contiguous whatever their stride says: every call takes a transposed [1, B]."""
    g = torch.Generator().manual_seed(3)
    order, lens = torch.tensor([[4, 0, 3, 1, 2]], dtype=torch.int32, device=dev()), [3, 16, 1, 9, 5]
    turned, plain = order.t(), order.view(5, 1).clone()
    assert turned.stride() == (1, 5) and turned.is_contiguous()
    lens = torch.tensor(lens, dtype=torch.int32, device=dev())
    starts = torch.arange(6, dtype=torch.int32, device=dev())
    q, k, v = (torch.randn((5, h, 64), generator=g).to(BF16).to(dev()) for h in (8, 2, 2))
    results = []
    for table in (plain, turned):
        caches = [torch.zeros((5, 2, 16, 64), dtype=FP8 if block else BF16, device=dev()) for _ in range(2)]
        scales = {n: torch.zeros((5, 2, 2), device=dev()) for n in ("k_scale", "v_scale")} if block else {}
        kv.kv_cache_append(k, v, *caches, table, lens, **scales)
        got = [*caches, *kv.kv_cache_read(*caches, table, lens, **scales),
               kv.paged_attention(q, *caches, table, lens, **scales),
               kv.paged_attention(q, *caches, table, lens, query_start=starts, **scales)]
        if not block:
            sums = torch.rand((5, 2, 16), generator=torch.Generator().manual_seed(1)).to(dev())
            got += [*kv.kv_cache_evict(*caches, table, lens, sums, 4), sums]
        results.append([t.view(torch.uint8) for t in got])
    for a, b in zip(*results):
        assert torch.equal(a, b)
    with pytest.raises(ValueError, match="contiguous rows"):
        kv.kv_cache_read(*caches, order.expand(5, 5)[:, ::2], lens, **scales)
