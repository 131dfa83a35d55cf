"""GPU tests of prompts' attention in tiles of 32 rows: weights enter the second product as two 16-bit terms."""
from __future__ import annotations

import math

import pytest
import torch

from test_gpu_kv_window import BF16, F16, FP8, dev
from vkernels_amd import kv_cache as kv

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache,D", [(None, 64), (None, 128), (FP8, 64), (FP8, 192)])
@pytest.mark.parametrize("q", [BF16, F16])
@pytest.mark.parametrize("high", [0.5, 0.75, 1.0, 1.25, 1.5, 1.75])
def test_weights_that_cancel(hip_lib, cache, D, q, high):
    """Half of the positions have one score and the value 1, half a lower score and the value -1: the result is
    tanh of half their difference, a small part of the weights that it is a difference of."""
    step = 2.0 ** -3 if cache else 2.0 ** -6           # (both scores are codes, or bf16 values)
    low, n, Hkv, G = high - step, 640, 2, 2
    odd = torch.arange(n) % 2 == 1
    k, v = torch.zeros((n, D)), torch.zeros((n, D))
    k[:, 0] = torch.where(odd, low, high)
    v[:] = torch.where(odd, -1.0, 1.0)[:, None]
    k, v = (x.view(-1, 1, 16, D).expand(-1, Hkv, 16, D).contiguous().to(cache or q).to(dev()) for x in (k, v))
    assert bool((k[0, 0, :2, 0].float().cpu() == torch.tensor([high, low])).all())
    queries = torch.zeros((8, Hkv * G, D), dtype=q, device=dev())
    queries[..., 0] = 1.0
    table = torch.arange(n // 16, dtype=torch.int32, device=dev())[None].repeat(2, 1)
    lens = torch.tensor([n, n - 40], dtype=torch.int32, device=dev())
    starts = torch.tensor([0, 3, 8], dtype=torch.int32, device=dev())
    scales = {n: torch.ones(Hkv, device=dev()) for n in ("k_scale", "v_scale")} if cache else {}
    out = kv.paged_attention(queries, k, v, table, lens, query_start=starts, scale=1.0, **scales)
    torch.cuda.synchronize()
    for row in range(8):
        seen = n - 2 + row if row < 3 else n - 40 - 7 + row
        a, b = math.exp(high) * (seen - seen // 2), math.exp(low) * (seen // 2)
        want = (a - b) / (a + b)
        # Scores are exact.  The exponent's product with log2(e) and the difference with the reference: 2^-24 of up to 2^3
        # each; the exponential 2^-22; two terms 2^-17 of the weight (bf16: 8 bits and 8 bits); 160 sums of a
        # wavefront in 32 bits, of the weights and of the products, all rounded the same way, 2^-24 each, and their joining:
        # 2^-15 altogether; the result half a step.
        tol = 2.0 ** -15 + torch.finfo(q).eps / 2 * (abs(want) + 2.0 ** -15)
        assert float((out[row].double() - want).abs().max()) <= tol, (row, want)
