"""Caches and rows whose offsets pass 32 bits: the same bits as from the same values close together."""
from __future__ import annotations

import pytest
import torch

from vkernels_amd import kv_cache as kv
from vkernels_amd.rotary import qk_norm_rope

pytestmark = pytest.mark.gpu

BF16, FP8 = torch.bfloat16, torch.float8_e4m3fn
PAGES, HEADS, PS, D = 5, 2, 16, 128


def dev():
    return torch.device("cuda", 0)


def _far(shape, dtype, strides):
    """A view of these strides (elements) on memory of its own."""
    size = 1 + sum((n - 1) * s for n, s in zip(shape, strides))
    return torch.empty(size, dtype=dtype, device=dev()).as_strided(shape, strides)


# elements apart: pages, heads or positions
STRIDES = {"pages": (2 ** 30 + 16, PS * D, D), "heads": (PS * D, 2 ** 32 + 16, D), "positions": (2 ** 30, D, 2 ** 26)}


@pytest.mark.parametrize("far", STRIDES)
@pytest.mark.parametrize("dtype,blocks", [(BF16, 0), (FP8, 1), (FP8, 4), (FP8, 16)])
@pytest.mark.parametrize("new", [(3, 4), (40, 9)])
def test_caches(hip_lib, far, dtype, blocks, new):
    gen = torch.Generator(device=dev()).manual_seed(3)
    lens = [PS * 4, 9]
    table = torch.tensor([[4, 1, 3, 0], [2, -1, -1, -1]], dtype=torch.int32, device=dev())
    lens_dev = torch.tensor(lens, dtype=torch.int32, device=dev())
    everything, starts = (torch.tensor([0, *n], device=dev()).cumsum(0).to(torch.int32) for n in (lens, new))
    rows = [torch.randn((sum(lens), HEADS, D), device=dev(), generator=gen).to(BF16) for _ in range(2)]
    q = torch.randn((sum(new), HEADS * 2, D), device=dev(), generator=gen).to(BF16)
    got = []
    for strides in (STRIDES[far], (HEADS * PS * D, PS * D, D)):
        k, v = (_far((PAGES, HEADS, PS, D), dtype, (*strides, 1)) for _ in range(2))
        scales = {} if not blocks else {n: torch.zeros((PAGES, HEADS, blocks), device=dev()) for n in ("k_scale", "v_scale")}
        kv.kv_cache_append(*rows, k, v, table, lens_dev, query_start=everything, **scales)
        read = kv.kv_cache_read(k, v, table, lens_dev, query_start=everything, tokens=sum(lens), **scales)
        out, lse = kv.paged_attention(q, k, v, table, lens_dev, query_start=starts, return_lse=True, **scales)
        one = kv.paged_attention(q[:2], k, v, table, lens_dev, **scales)
        got.append([*read, out, lse, one, *scales.values()])
        del k, v
    assert all(torch.equal(near, away) and bool(torch.isfinite(near.float()).all()) for near, away in zip(got[1], got[0]))
    for x, row in zip(got[0], rows):
        # (codes are off by 2^-4 of themselves and a block's scale by 2^-10 of its largest value, 6 at most)
        assert bool(((x.float() - row.float()).abs() <= (row.float().abs() * 2.0 ** -4 + 2.0 ** -7 if blocks else 0.0)).all())


def test_rows(hip_lib):
    gen = torch.Generator(device=dev()).manual_seed(3)
    q, k = (torch.randn((5, heads, D), device=dev(), generator=gen).to(BF16) for heads in (4, 2))
    freqs = 1e4 ** -(torch.arange(0, D, 2, device=dev()) / D)
    positions = torch.arange(5, dtype=torch.int32, device=dev()) * 1000
    want = qk_norm_rope(q, k, positions, freqs)
    for strides in ((2 ** 30 + 16, D, 1), (D, 2 ** 31 + 16, 1)):
        far = [_far(x.shape, BF16, strides).copy_(x) for x in (q, k)]
        got = qk_norm_rope(*far, positions, freqs, out=tuple(far))
        assert got[0] is far[0] and all(torch.equal(a, b) for a, b in zip(want, got))
        del far, got
    # rows that are appended, and read into
    cache = [torch.zeros((2, 2, 16, D), dtype=FP8, device=dev()) for _ in range(4)]
    scales = [{n: torch.zeros((2, 2, 4), device=dev()) for n in ("k_scale", "v_scale")} for _ in range(2)]
    table, lens = torch.tensor([[1, 0]], dtype=torch.int32, device=dev()), torch.tensor([5], dtype=torch.int32, device=dev())
    starts = torch.tensor([0, 5], dtype=torch.int32, device=dev())
    far = _far(k.shape, BF16, (2 ** 30 + 16, D, 1)).copy_(k)
    kv.kv_cache_append(k, k, *cache[:2], table, lens, query_start=starts, **scales[0])
    kv.kv_cache_append(far, far, *cache[2:], table, lens, query_start=starts, **scales[1])
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(cache[:2], cache[2:]))
    near = kv.kv_cache_read(*cache[:2], table, lens, query_start=starts, tokens=5, **scales[0])
    away = [_far(k.shape, BF16, (2 ** 30 + 16, D, 1)) for _ in range(2)]
    kv.kv_cache_read(*cache[:2], table, lens, query_start=starts, tokens=5, out=tuple(away), **scales[0])
    assert all(torch.equal(a, b) for a, b in zip(near, away))
    # queries
    q_far = _far(q.shape, BF16, (2 ** 30 + 16, D, 1)).copy_(q)
    outs = [kv.paged_attention(x, *cache[:2], table, lens, query_start=starts, **scales[0]) for x in (q, q_far)]
    assert torch.equal(*outs)
