"""CPU tests of vk_hip_qk_norm_rope's refusals: nothing is launched."""
from __future__ import annotations

import ctypes

import pytest

from vkernels_amd import rotary
from vkernels_amd import vllm_experts as ve

P = 4096          # an aligned address that nothing dereferences: every call here ends in the checks
ARGS = dict(q=P, k=P, positions=P, inv_freq=P, q_weight=P, k_weight=P, q_out=P, k_out=P, kind=0, weights_f32=0, T=4, Hq=8,
            Hkv=2, D=64, turned=64, pairs=0, axes=1, sections=None, norm=1, eps=1e-6, factor=1.0, q_stride_t=512,
            q_stride_h=64, k_stride_t=128, k_stride_h=64, q_out_stride_t=512, q_out_stride_h=64, k_out_stride_t=128,
            k_out_stride_h=64, axis_stride=4, stream=None)
THREE = (ctypes.c_int32 * 3)(8, 12, 11)
NEGATIVE = (ctypes.c_int32 * 3)(40, -12, 4)
LARGE = (ctypes.c_int32 * 2)(2147483647, 2147483647)


@pytest.fixture(scope="module")
def call():
    if ve.find_libvkernels_hip() is None:
        from vkernels_amd import build
        build.build()
    fn = rotary._fn()
    return lambda **kw: fn(*dict(ARGS, **kw).values())


@pytest.mark.parametrize("bad", [
    dict(T=-1), dict(Hq=0), dict(Hkv=0), dict(D=0), dict(D=24), dict(D=272), dict(turned=0), dict(turned=12), dict(turned=72),
    dict(turned=-8), dict(axes=0), dict(axes=5), dict(axes=2), dict(axes=3, sections=THREE), dict(axes=3, sections=NEGATIVE),
    dict(axes=2, sections=LARGE), dict(q=None), dict(k=None), dict(q_out=None), dict(k_out=None), dict(positions=None),
    dict(inv_freq=None), dict(norm=0), dict(eps=-1e-6), dict(eps=float("nan")), dict(q_weight=P + 8), dict(k_weight=P + 4),
    dict(q=P + 8), dict(k_out=P + 2), dict(q_stride_t=516), dict(k_stride_h=68), dict(q_out_stride_h=60),
    dict(q_stride_t=-512), dict(axis_stride=-4), dict(q_out_stride_t=0), dict(k_out_stride_h=0), dict(k_out_stride_h=32),
    dict(q_out_stride_t=64), dict(q_out_stride_t=504), dict(q_out_stride_t=64, q_out_stride_h=248), dict(k_out_stride_t=-128)])
def test_invalid_arguments(call, bad):
    assert call(**bad) == ve.VK_ERROR_INVALID_ARGUMENT
    assert "vk_hip_qk_norm_rope" in ve.last_error(ve.load_libvkernels_hip())


def test_other_refusals(call):
    assert call(kind=2) == ve.VK_ERROR_UNSUPPORTED
    assert call(T=1 << 30) == ve.VK_ERROR_OUT_OF_RANGE
    assert call(T=1, Hq=2147483647) == ve.VK_ERROR_OUT_OF_RANGE


def test_nothing_to_do(call):
    assert call(T=0, q=None, k=None, q_out=None, k_out=None) == ve.VK_OK
