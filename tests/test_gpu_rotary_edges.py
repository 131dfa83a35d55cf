"""GPU tests of norm and rotation: positions of a single token."""
from __future__ import annotations

import pytest
import torch

from test_gpu_kv_window import BF16, dev
from vkernels_amd.rotary import qk_norm_rope

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("axes", [2, 3, 4])
def test_one_token_of_several_axes(hip_lib, axes):
    """Rows of one element are contiguous whatever their stride says: a transposed [1, axes]."""
    q, k = (torch.randn((1, h, 64), device=dev(), dtype=BF16) for h in (4, 2))
    f = 1e4 ** -(torch.arange(32, device=dev()) / 32.0)
    sections = [32 // axes + (1 if i < 32 % axes else 0) for i in range(axes)]
    p = torch.arange(5, 5 + axes, dtype=torch.int32, device=dev())
    want = qk_norm_rope(q, k, p.view(axes, 1).clone(), f, sections=sections)
    turned = p.view(1, axes).t()
    assert turned.stride() == (1, axes) and turned.is_contiguous()
    got = qk_norm_rope(q, k, turned, f, sections=sections)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    wide = torch.zeros((axes, 7), dtype=torch.int32, device=dev())
    wide[:, 3] = p
    got = qk_norm_rope(q, k, wide[:, 3:4], f, sections=sections)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_a_strided_position(hip_lib):
    q, k = (torch.randn((1, h, 64), device=dev(), dtype=BF16) for h in (4, 2))
    f = 1e4 ** -(torch.arange(32, device=dev()) / 32.0)
    p = torch.tensor([1, 9, 4, 2], dtype=torch.int32, device=dev())
    got, want = qk_norm_rope(q, k, p[1::4], f), qk_norm_rope(q, k, p[1:2].clone(), f)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    with pytest.raises(ValueError, match="contiguous rows"):
        qk_norm_rope(q.expand(2, 4, 64), k.expand(2, 2, 64), p[::2], f)
