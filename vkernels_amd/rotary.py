"""Queries and keys in front of the key-value cache: the RMS norm of every head and the rotation by the
token's position, in one pass over them.

The call is enqueued on the current stream of the tensors' device, without host synchronisation, and can be
captured in a graph.  It is an operator of inference: a backward pass that comes to it raises an error, and with
results that the caller gives the call is refused where one of its tensors wants a gradient.

The entry point is additive: the reference leaves queries and keys to its caller.  Everything runs in
``libvkernels_hip.so``; there is no fallback.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd.graph import increment_version

from .kv_cache import _current_device, _dual_level, _failed, _need, _no_backward, _refuse_derivatives, _rows, _stream
from .vllm_experts import load_libvkernels_hip

__all__ = ["qk_norm_rope"]

_KINDS = {torch.bfloat16: 0, torch.float16: 1}
_fn_cache: list = []


def _fn():
    if not _fn_cache:
        fn = getattr(load_libvkernels_hip(), "vk_hip_qk_norm_rope", None)
        if fn is None:
            raise RuntimeError("vk_hip_qk_norm_rope not found in libvkernels_hip.so")
        P, I, L, F = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float
        fn.argtypes, fn.restype = [P] * 8 + [I] * 9 + [P, I, F, F] + [L] * 9 + [P], I
        _fn_cache.append(fn)
    return _fn_cache[0]


_result = _no_backward("qk_norm_rope")


def _weight_at(w, D, of, device, name):
    if not (w.shape == (D,) and w.dtype is of and w.get_device() == device and w.is_contiguous()):
        raise ValueError(f"{name} must be [D] contiguous on q's device, and both weights in float32 or in q's type")
    return w if w.data_ptr() % 16 == 0 else w.clone(memory_format=torch.contiguous_format)


def _check_out(out, like, name):
    s = out.stride()
    _need(out.shape == like.shape and out.dtype is like.dtype and out.get_device() == like.get_device() and s[2] == 1 and
          s[0] % 8 == 0 and s[1] % 8 == 0 and out.data_ptr() % 16 == 0,
          f"the result for {name} must be like {name}, with rows that start on 16 bytes")


# The checks are one expression on the path that is taken (a decode step is short: the host's work per call
# counts); _explain says which part of it did not hold.

def _explain(q, k, positions, inv_freq):
    _need(q.dim() == 3 and k.dim() == 3 and k.shape[0] == q.shape[0] and k.shape[2] == q.shape[2],
          "q and k must be [T, Hq, D] and [T, Hkv, D]")
    _need(q.dtype in _KINDS and k.dtype is q.dtype, "q and k must both be bfloat16 or float16")
    _need(all(t.get_device() == _current_device() for t in (q, k, positions, inv_freq)),
          "the tensors must be on the current device")
    _need(inv_freq.dtype is torch.float32 and inv_freq.dim() == 1 and inv_freq.is_contiguous() and
          inv_freq.shape[0] <= q.shape[2] // 2, "inv_freq must be up to D / 2 contiguous float32 values")
    _need(positions.dtype is torch.int32 and (positions.stride()[-1:] == (1,) or q.shape[0] <= 1),
          "positions must be int32 with contiguous rows")
    _need(False, "q and k must have heads, and sizes below 2^31")


def qk_norm_rope(q, k, positions, inv_freq, *, q_weight=None, k_weight=None, eps=1e-6, sections=None, pairs=False,
                 factor=1.0, out=None):
    """Queries [T, Hq, D] and keys [T, Hkv, D] with every head normed and rotated by its token's position.

    A head x becomes x * weight / sqrt(mean(x^2) + eps) (``q_weight``, ``k_weight`` [D] in q's type or both
    float32, None: 1; ``eps`` None: no norm).  Of the result the first 2 R values, R the number of ``inv_freq``
    (float32), are turned in pairs by the angles position * inv_freq[i], cosine and sine times ``factor``:
    value i with value i + R, or with ``pairs`` 2 i with 2 i + 1.  The others stay.
    ``positions`` [T] int32, or [axes, T] (time, height, width, ...; up to 4) with ``sections``: so many of
    the frequencies, in order, turn by each axis.
    Returns (q, k), new ones, or ``out`` (a pair of tensors, which may be q and k themselves).  q and k may be
    views of one tensor of any strides with D contiguous."""
    device, shape, k_shape, kind = q.get_device(), q.shape, k.shape, _KINDS.get(q.dtype)
    if not (len(shape) == 3 and len(k_shape) == 3 and shape[0] == k_shape[0] and shape[2] == k_shape[2] and
            kind is not None and k.dtype is q.dtype and device == _current_device() and k.get_device() == device and
            positions.get_device() == device and inv_freq.get_device() == device and
            inv_freq.dtype is torch.float32 and inv_freq.dim() == 1 and inv_freq.is_contiguous() and
            inv_freq.shape[0] <= shape[2] // 2 and positions.dtype is torch.int32 and
            (positions.stride()[-1:] == (1,) or shape[0] <= 1) and
            shape[1] > 0 and k_shape[1] > 0 and (shape[0] | shape[1] | k_shape[1]) <= 0x7FFFFFFF):
        _explain(q, k, positions, inv_freq)
    (T, Hq, D), Hkv, R = shape, k_shape[1], inv_freq.shape[0]
    if sections is None:
        if positions.shape != (T,):
            raise ValueError("positions must be [T], or [axes, T] with sections")
        axes, axis_stride, c_sections = 1, 0, None
    else:
        axes = len(sections)
        _need(1 <= axes <= 4 and positions.shape == (axes, T), "positions must be [axes, T] with a section for each of up to 4 axes")
        _need(all(0 <= n <= R for n in sections) and sum(sections) == R, "sections must add up to the number of inv_freq")
        axis_stride, c_sections = positions.stride(0), (ctypes.c_int32 * axes)(*sections)
    weights_f32 = 0
    if q_weight is not None or k_weight is not None:
        _need(eps is not None, "weights belong to the norm, which eps=None leaves out")
        of = (q_weight if q_weight is not None else k_weight).dtype
        weights_f32 = int(of is torch.float32)
        of = torch.float32 if weights_f32 else q.dtype
        q_weight = None if q_weight is None else _weight_at(q_weight, D, of, device, "q_weight")
        k_weight = None if k_weight is None else _weight_at(k_weight, D, of, device, "k_weight")
    inputs = q, k, inv_freq, q_weight, k_weight
    wants_grad = torch.is_grad_enabled() and (
        q.requires_grad or k.requires_grad or inv_freq.requires_grad or q_weight is not None and q_weight.requires_grad or
        k_weight is not None and k_weight.requires_grad)
    if out is None:
        q_out, k_out = q.new_empty((T, Hq, D)), k.new_empty((T, Hkv, D))
    else:
        q_out, k_out = out
        _check_out(q_out, q, "q")
        _check_out(k_out, k, "k")
    if out is not None or _dual_level() >= 0:
        _refuse_derivatives("qk_norm_rope", () if out is None else (q_out, k_out), *inputs)
    q, k = _rows(q), _rows(k)
    qs, ks, qo, ko = q.stride(), k.stride(), q_out.stride(), k_out.stride()
    status = _fn()(
        q.data_ptr(), k.data_ptr(), positions.data_ptr(), inv_freq.data_ptr(),
        None if q_weight is None else q_weight.data_ptr(), None if k_weight is None else k_weight.data_ptr(),
        q_out.data_ptr(), k_out.data_ptr(), kind, weights_f32, T, Hq, Hkv, D, 2 * R, pairs, axes,
        c_sections, eps is not None, 0.0 if eps is None else eps, factor, qs[0], qs[1], ks[0], ks[1], qo[0], qo[1],
        ko[0], ko[1], axis_stride, _stream(device))
    if status:
        _failed(status, "vk_hip_qk_norm_rope")
    if out is not None:
        increment_version((q_out, k_out))
    elif wants_grad:
        q_out, k_out = _result(q_out, k_out, *inputs)
    return q_out, k_out
