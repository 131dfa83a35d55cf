"""GPU tests of block-scaled caches, prompts' attention and rotation at the ends of what their arguments may be."""
from __future__ import annotations

import pytest
import torch

from test_gpu_kv_blocks import BF16, F16, Cache, dev

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("ps,block,D", [(16, 1, 64), (16, 8, 64), (16, 16, 80), (64, 64, 128)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_a_negative_zero_keeps_its_sign(hip_lib, ps, block, D, dtype):
    """-0 / s is -0 whatever the scale: of rows' kernel, a wavefront's and a workgroup's blocks, and of blocks of zeros."""
    c = Cache([90, 40], 2, D, ps, block, seed=D + block)

    def rows(n, size=1.0):
        out = []
        for _ in range(2):
            x = size * torch.randn((n, 2, D), generator=c.g)
            kind = torch.randint(0, 4, x.shape, generator=c.g)
            x = torch.where(kind == 0, -0.0, torch.where(kind == 1, 0.0, x))
            x[n // 2] = -0.0
            out.append(x.to(dtype).to(dev()))
        return out

    c.append([80, 30], [80, 30], rows=rows(110))
    c.append([81, 31], rows=rows(2, 3.0))
    c.append([82, 32], rows=[torch.full((2, 2, D), -0.0, dtype=dtype, device=dev()) for _ in range(2)])
    page, slot = int(c.table[0, 81 // ps]), 81 % ps
    assert bool((c.k.view(torch.uint8)[page, :, slot] == 0x80).all())
