"""GPU tests of results that the caller gives (out=) where gradients are wanted: refused, or an error in the backward pass
that comes to them; and of what autograd sees of the tensors that are written."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from test_gpu_kv_window import BF16, Setup, dev
from vkernels_amd import kv_cache as kv
from vkernels_amd.rotary import qk_norm_rope

pytestmark = pytest.mark.gpu


def rotate(q, k, **kw):
    t = torch.arange(q.shape[0], dtype=torch.int32, device=dev())
    return qk_norm_rope(q, k, t, 1e4 ** -(torch.arange(32, device=dev()) / 32.0), **kw)


def rows(*shape, **kw):
    return torch.randn(shape, device=dev(), dtype=BF16, **kw)


def test_rotation_in_place(hip_lib):
    x = rows(5, 4, 64, requires_grad=True)
    q, k = x * 2, rows(5, 2, 64)
    before = q.detach().clone()
    with pytest.raises(RuntimeError, match="qk_norm_rope has no backward"):
        rotate(q, k, out=(q, k))
    assert torch.equal(q, before)          # (nothing has run)
    with pytest.raises(RuntimeError, match="qk_norm_rope has no backward"):
        rotate(q.detach(), k, out=(q, k))
    weight = torch.ones(64, device=dev(), requires_grad=True)
    with pytest.raises(RuntimeError, match="qk_norm_rope has no backward"):
        rotate(k, k.clone(), q_weight=weight, out=(torch.empty_like(k), torch.empty_like(k)))
    with torch.no_grad():
        got = rotate(q, k, out=(q, k))
    assert got[0] is q and not torch.equal(q, before)


def test_a_tensor_that_a_node_has_saved(hip_lib):
    """Written in place it is not what the node saved: the backward pass says so, and does not go on with other values."""
    x = rows(5, 4, 64, requires_grad=True)
    q, k = rows(5, 4, 64), rows(5, 2, 64)
    loss = (x * q).float().sum()
    rotate(q, k, out=(q, k))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    s = Setup([40, 30], 2, 2, 64, 16, 0)
    starts = torch.tensor([0, 1, 2], dtype=torch.int32, device=dev())
    for more in (dict(), dict(query_start=starts)):
        out = torch.zeros_like(s.q)
        loss = (rows(*s.q.shape, requires_grad=True) * out).float().sum()
        kv.paged_attention(s.q, s.k, s.v, s.table, s.lens, out=out, **more)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    for i in range(2):
        out = [torch.zeros((2, 2, 64), dtype=BF16, device=dev()) for _ in range(2)]
        loss = (rows(2, 2, 64, requires_grad=True) * out[i]).float().sum()
        kv.kv_cache_read(s.k, s.v, s.table, s.lens, out=out)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    with torch.inference_mode():           # (such tensors have no version)
        q, k = rows(5, 4, 64), rows(5, 2, 64)
        rotate(q, k, out=(q, k))


def test_reading(hip_lib):
    s = Setup([40, 30], 2, 2, 64, 16, 0)
    wide = s.k.clone().requires_grad_()
    room = [torch.full((2, 2, 64), 3.0, dtype=BF16, device=dev()) for _ in range(2)]
    with pytest.raises(RuntimeError, match="kv_cache_read has no backward"):
        kv.kv_cache_read(wide, s.v, s.table, s.lens, out=room)
    with pytest.raises(RuntimeError, match="kv_cache_read has no backward"):
        kv.kv_cache_read(s.k, s.v, s.table, s.lens, out=[room[0], room[1].clone().requires_grad_()])
    assert bool((room[0] == 3).all() and (room[1] == 3).all())


def test_attention(hip_lib):
    s = Setup([40, 30], 2, 2, 64, 16, 0)
    wide, q, sinks = (t.clone().requires_grad_() for t in (s.k, s.q, s.sinks))
    starts = torch.tensor([0, 1, 2], dtype=torch.int32, device=dev())
    for more in (dict(), dict(query_start=starts), dict(return_lse=True)):
        leaf = rows(*s.q.shape, requires_grad=True)
        for args, kw in (((q, s.k, s.v), {}), ((s.q, wide, s.v), {}), ((s.q, s.k, wide), {}), ((s.q, s.k, s.v), dict(sinks=sinks)),
                         ((s.q, s.k, s.v), dict(out=leaf * 2)), ((q, s.k, s.v), dict(out=rows(5, 4, 64)[2:4]))):
            kw.setdefault("out", torch.full_like(s.q, 3.0))
            with torch.no_grad():
                want = kv.paged_attention(*args, s.table, s.lens, **dict(more, return_lse=True, **dict(kw, out=None)))
            got = kv.paged_attention(*args, s.table, s.lens, **more, **kw)
            got, lse = got if more.get("return_lse") else (got, None)
            assert got is kw["out"] and got.requires_grad and torch.equal(got, want[0]) and (lse is None or torch.equal(lse, want[1]))
            # (what is behind `out` is no input of the lse)
            inputs_want = any(t.requires_grad for t in args) or "sinks" in kw
            assert lse is None or lse.requires_grad == inputs_want
            for result in (kw["out"], lse):
                if result is not None and result.requires_grad:
                    with pytest.raises(RuntimeError, match="paged_attention has no backward"):
                        result.float().sum().backward()
        room = torch.full_like(s.q, 3.0).requires_grad_()
        with pytest.raises(RuntimeError, match="leaf"):
            kv.paged_attention(s.q, s.k, s.v, s.table, s.lens, out=room, **more)
        assert bool((room == 3).all())
        with torch.no_grad():
            kv.paged_attention(q, s.k, s.v, s.table, s.lens, out=room, **more)
        assert not bool((room == 3).any())


@pytest.mark.parametrize("block", [-1, 8])
def test_scales_that_want_a_gradient(hip_lib, block):
    s = Setup([40, 30], 2, 2, 64, 16, block)
    for name in ("k_scale", "v_scale"):
        scales = dict(k_scale=s.k_scale, v_scale=s.v_scale)
        scales[name] = scales[name].clone().requires_grad_()
        out = kv.paged_attention(s.q, s.k, s.v, s.table, s.lens, **scales)
        with pytest.raises(RuntimeError, match="paged_attention has no backward"):
            out.float().sum().backward()
        k, v = kv.kv_cache_read(s.k, s.v, s.table, s.lens, **scales)
        with pytest.raises(RuntimeError, match="kv_cache_read has no backward"):
            (k.float().sum() + v.float().sum()).backward()


def test_tangents(hip_lib):
    """Forward-mode derivatives are refused as well, not dropped."""
    s = Setup([40, 30], 2, 2, 64, 16, 0)
    q, k = rows(5, 4, 64), rows(5, 2, 64)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(q, torch.ones_like(q))
        for kw in (dict(), dict(out=(torch.empty_like(q), torch.empty_like(k)))):
            with pytest.raises(RuntimeError, match="qk_norm_rope has no"):
                rotate(dual, k, **kw)
        with pytest.raises(RuntimeError, match="kv_cache_read has no"):
            kv.kv_cache_read(s.k, forward_ad.make_dual(s.v, torch.ones_like(s.v)), s.table, s.lens)
        dual = forward_ad.make_dual(s.q, torch.ones_like(s.q))
        for kw in (dict(), dict(out=torch.empty_like(s.q))):
            with pytest.raises(RuntimeError, match="paged_attention has no"):
                kv.paged_attention(dual, s.k, s.v, s.table, s.lens, **kw)
        rotate(q, k)                       # (tensors without one are as ever)
