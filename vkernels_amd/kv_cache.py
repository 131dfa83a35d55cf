"""A paged key-value cache on torch device tensors: append, reading back, the attention of one or
of several new tokens over it, and eviction by accumulated attention weight.

A cache is two tensors [pages, Hkv, page_size, D] of any strides with D contiguous (a cache that is
[pages, page_size, Hkv, D] in memory goes in as its ``transpose(1, 2)``), bf16, fp16 or
float8_e4m3fn with float32 scales: one for each head, [Hkv], or one for each block of positions of a
page and head, [pages, Hkv, blocks], which append sets from what is written (the selection of an
eviction moves rows between blocks, so it takes caches with a scale for each head alone).
``block_table`` [B, W] int32 names the page of every page_size positions of a sequence,
``seq_lens`` [B] int32 how many positions it has.  Every
call is enqueued on the current stream of the tensors' device, with no host synchronisation; what it
writes besides its arguments comes from torch's allocator, so calls on several streams do not share
scratch and a call can be captured in a graph.

These are operators of inference: no gradient passes through the cache, and a backward pass that comes to
their results raises an error, also where the caller gives them (``paged_attention``; ``kv_cache_read``, whose two may
be parts of one tensor, refuses ``out`` where one of its tensors wants a gradient).  Tensors with forward-mode
tangents are refused.

The entry points are additive: the reference keeps its cache outside this path.  Everything runs in
``libvkernels_hip.so``; there is no fallback.
"""
from __future__ import annotations

import ctypes
import functools

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from .vllm_experts import last_error, load_libvkernels_hip

__all__ = ["kv_cache_append", "kv_cache_evict", "kv_cache_read", "paged_attention"]

_P, _I, _L, _F, _Z = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float, ctypes.c_size_t

# VK_HIP_KV_*: (type of the cache, type of the queries)
_KINDS = {
    (torch.bfloat16, torch.bfloat16): 0,
    (torch.float16, torch.float16): 1,
    (torch.float8_e4m3fn, torch.bfloat16): 2,
    (torch.float8_e4m3fn, torch.float16): 3,
}

_INT32 = torch.int32
_fns: dict = {}


def _fn(name):
    fn = _fns.get(name)
    if fn is None:
        lib = load_libvkernels_hip()
        argtypes, restype = {
            "vk_hip_kv_cache_append": ([_P] * 9 + [_I] * 9 + [_L] * 7 + [_P], _I),
            "vk_hip_kv_cache_append_ex": ([_P] * 9 + [_I] * 10 + [_L] * 7 + [_P], _I),
            "vk_hip_kv_cache_read": ([_P] * 7 + [_I] + [_P] * 2 + [_I] * 10 + [_L] * 7 + [_P], _I),
            "vk_hip_paged_attention_workspace_bytes": ([_I] * 8, _Z),
            "vk_hip_paged_attention_workspace_bytes_ex": ([_I] * 9, _Z),
            "vk_hip_paged_attention_ex": ([_P] * 8 + [_I] + [_P] * 3 + [_I] * 12 + [_F, _F] + [_L] * 7 + [_P, _Z, _P], _I),
            "vk_hip_paged_attention": ([_P] * 11 + [_I] * 11 + [_F, _F] + [_L] * 7 + [_P, _Z, _P], _I),
            "vk_hip_paged_attention_prompt_workspace_bytes": ([_I] * 8, _Z),
            "vk_hip_paged_attention_prompt": ([_P] * 9 + [_I] + [_P] * 2 + [_I] * 14 + [_F, _F] + [_L] * 5 + [_P, _Z, _P], _I),
            "vk_hip_kv_cache_evict_workspace_bytes": ([_I] * 6, _Z),
            "vk_hip_kv_cache_evict": ([_P] * 8 + [_I] * 12 + [_L] * 7 + [_P, _Z, _P], _I),
        }[name]
        try:
            fn = getattr(lib, name)
        except AttributeError:
            raise RuntimeError(f"{name} not found in libvkernels_hip.so") from None
        fn.argtypes, fn.restype = argtypes, restype
        _fns[name] = fn
    return fn


@functools.lru_cache(maxsize=256)
def _bytes(name, *sizes):
    """The workspace of a call of these sizes (the library's answer follows them alone)."""
    return _fn(name)(*sizes)


def _failed(status, name):
    raise RuntimeError(f"{name} failed with status {status}: {last_error(load_libvkernels_hip())}")


def _need(ok, message):
    if not ok:
        raise ValueError(message)


# The checks are one expression each on the path that is taken (a decode step is short: the host's work per
# call counts); the functions _explain_* say which part of it did not hold.

def _cache_ok(k_cache, v_cache, block_table, seq_lens, shape, strides, device, table, table_strides):
    return (v_cache.shape == shape and v_cache.stride() == strides and strides[3] == 1 and
            v_cache.dtype is k_cache.dtype and block_table.dtype is _INT32 and seq_lens.dtype is _INT32 and
            (table_strides[1] == 1 or table[1] <= 1) and seq_lens.shape == table[:1] and seq_lens.is_contiguous() and
            v_cache.get_device() == device and block_table.get_device() == device and
            seq_lens.get_device() == device and device >= 0 and _current_device() == device and
            (shape[0] | shape[1] | shape[2] | table[0] | table[1] | table_strides[0]) <= 0x7FFFFFFF)


def _explain_cache(k_cache, v_cache, block_table, seq_lens):
    _need(k_cache.dim() == 4 and k_cache.shape == v_cache.shape,
          "k_cache and v_cache must be [pages, Hkv, page_size, D] alike")
    _need(k_cache.dtype == v_cache.dtype and k_cache.stride() == v_cache.stride() and k_cache.stride(3) == 1,
          "k_cache and v_cache must have one type and the same strides, rows of D values contiguous")
    _need(block_table.dtype == torch.int32 and block_table.dim() == 2 and
          (block_table.stride(1) == 1 or block_table.shape[1] <= 1),
          "block_table must be int32 [B, W] with contiguous rows")
    _need(seq_lens.dtype == torch.int32 and seq_lens.shape == block_table.shape[:1] and seq_lens.is_contiguous(),
          "seq_lens must be int32 [B], contiguous")
    devices = {t.get_device() for t in (k_cache, v_cache, block_table, seq_lens)}
    _need(len(devices) == 1 and devices != {-1}, "the cache, block_table and seq_lens must be on one device")
    _need(devices == {_current_device()}, "the tensors' device must be the current device")
    _need(not any(n >> 31 for n in (*k_cache.shape, *block_table.shape, block_table.stride(0))),
          "the sizes of the cache and of block_table must be below 2^31")


def _int32(**sizes):
    """The library takes these in 32 bits, and ctypes would cut what does not fit."""
    for name, n in sizes.items():
        if not -0x80000000 <= n <= 0x7FFFFFFF:
            raise ValueError(f"{name} must be within 32 bits, not {n}" +
                             (" (its default is what the table holds)" if name == "max_len" else ""))


# The current device, and a device's current stream as the address that the library takes.
_current_device = torch._C._cuda_getDevice
_stream = torch._C._cuda_getCurrentRawStream


def _head_vector(t, n, name, device):
    if not (t.dtype is torch.float32 and t.numel() == n and t.is_contiguous() and t.get_device() == device):
        raise ValueError(f"{name} must be {n} contiguous float32 values on the cache's device")
    return t.data_ptr()


def _scales(k_scale, v_scale, pages, Hkv, page_size, device):
    """Addresses of the scales of an 8-bit cache and how many a page has for each head: 0 where there is one
    for the head alone, [Hkv], else [pages, Hkv, blocks]."""
    if k_scale is None or v_scale is None or k_scale.dim() != 3:
        return (None if k_scale is None else _head_vector(k_scale, Hkv, "k_scale", device),
                None if v_scale is None else _head_vector(v_scale, Hkv, "v_scale", device), 0)
    blocks = k_scale.shape[2]
    for t, name in ((k_scale, "k_scale"), (v_scale, "v_scale")):
        if not (t.shape == (pages, Hkv, blocks) and blocks and page_size % blocks == 0 and t.dtype is torch.float32 and
                t.is_contiguous() and t.get_device() == device):
            raise ValueError(f"{name} must be contiguous float32 [Hkv], or [pages, Hkv, blocks] with blocks that "
                             "divide a page, on the cache's device, both alike")
    return k_scale.data_ptr(), v_scale.data_ptr(), blocks


def _query_start(t, B, device):
    _need(t.dtype is torch.int32 and t.numel() == B + 1 and t.is_contiguous() and t.get_device() == device,
          "query_start must be int32 [B + 1] on the cache's device")
    return t.data_ptr()


def _cache(k_cache, v_cache, block_table, seq_lens):
    """Checks what every operator takes: (pages, Hkv, page_size, D), the cache's strides, its device, and
    the table's (B, W) and elements from row to row."""
    shape, strides, device = k_cache.shape, k_cache.stride(), k_cache.get_device()
    table, table_strides = block_table.shape, block_table.stride()
    if len(shape) != 4 or len(table) != 2 or not _cache_ok(k_cache, v_cache, block_table, seq_lens, shape, strides,
                                                           device, table, table_strides):
        _explain_cache(k_cache, v_cache, block_table, seq_lens)
    return shape, strides, device, table, table_strides[0] if table[0] > 1 else table[1]


def _sums_ok(t, B, Hkv, positions, device):
    """float32 [B, Hkv, positions or more], rows contiguous and each its own."""
    if t.dim() != 3:
        return False
    (b, h, n), (sb, sh, one) = t.shape, t.stride()
    return (t.dtype is torch.float32 and b == B and h == Hkv and n >= positions and one == 1 and
            (sb > 0 or B <= 1) and (sh > 0 or Hkv == 1) and t.get_device() == device)


def _rows(t):
    """`t` [n, heads, D], or a copy of it where its rows do not start on 16 bytes."""
    s = t.stride()
    if s[2] != 1 or s[0] % 8 or s[1] % 8 or t.data_ptr() % 16:
        # (not contiguous(): that is the tensor itself where an odd stride belongs to a dimension of size 1)
        t = t.new_empty(t.shape).copy_(t)
    return t


def _backward_error(name):
    return RuntimeError(f"{name} has no backward pass: it is an operator of inference "
                        "(call it under torch.no_grad(), or detach what requires a gradient)")


def _no_backward(name):
    """A function that hands an operator's two results on as they are; a backward pass that reaches them is an error
    instead of a gradient lost."""

    class NoBackward(torch.autograd.Function):
        @staticmethod
        def forward(ctx, first, second, *inputs):
            return first.view_as(first), None if second is None else second.view_as(second)

        @staticmethod
        def backward(ctx, *grads):
            raise _backward_error(name)

    return NoBackward.apply


def _no_backward_given(name):
    """The same for one result that the caller has given, and that is written in place."""

    class NoBackwardGiven(torch.autograd.Function):
        @staticmethod
        def forward(ctx, out, *inputs):
            ctx.mark_dirty(out)
            return out

        @staticmethod
        def backward(ctx, *grads):
            raise _backward_error(name)

    return NoBackwardGiven.apply


def _dual_level():
    """0 or more where tensors may have tangents."""
    return getattr(forward_ad, "_current_level", 0)


def _refuse_derivatives(name, out, *inputs):
    """Raises where a derivative would be lost: of what goes to results that the caller has given (`out`, or ()), whose
    node is not this call's, and in forward mode."""
    inputs = [t for t in inputs if t is not None]
    if out and torch.is_grad_enabled() and any(t.requires_grad for t in (*out, *inputs)):
        raise RuntimeError(f"{name} has no backward pass, and out= cannot say so later: call it under torch.no_grad(), or "
                           "detach what requires a gradient")
    if _dual_level() >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in (*out, *inputs)):
        raise RuntimeError(f"{name} has no derivative: it is an operator of inference")


_attention_result, _read_result = _no_backward("paged_attention"), _no_backward("kv_cache_read")
_given_attention_result = _no_backward_given("paged_attention")


def kv_cache_append(k, v, k_cache, v_cache, block_table, seq_lens, *, query_start=None, k_scale=None, v_scale=None):
    """New tokens' keys and values [tokens, Hkv, D] into the pages.

    ``seq_lens`` count the new tokens.  ``query_start`` [B + 1] int32: the new tokens of sequence b are
    query_start[b] .. query_start[b + 1] - 1 and go to its last positions; None: one token for each
    sequence (a sequence of length 0 takes none).  Positions whose page is outside [0, pages) are
    skipped.  An 8-bit cache holds the codes nearest to value / scale of the head (``k_scale``,
    ``v_scale`` [Hkv]), the largest finite code beyond +-448.

    With ``k_scale``, ``v_scale`` [pages, Hkv, blocks] an 8-bit cache has a scale for each head and block of
    page_size / blocks positions, and this call finds it: the block's largest magnitude / 448, of the new
    rows and of the positions already in front of them, whose codes are rounded again where the scale grows
    (a block that begins with a new row takes nothing from what it held).  Infinite values and NaN do not
    count for it."""
    (pages, Hkv, ps, D), strides, device, (B, W), table_stride = _cache(k_cache, v_cache, block_table, seq_lens)
    tokens = k.shape[0]
    _need(k.shape == (tokens, Hkv, D) and v.shape == k.shape and v.dtype is k.dtype and tokens < 1 << 31,
          "k and v must be [tokens, Hkv, D] alike")
    _need(k.get_device() == device and v.get_device() == device, "k and v must be on the cache's device")
    kind = _KINDS.get((k_cache.dtype, k.dtype))
    _need(kind is not None, "the cache's type does not take rows of this type")
    if query_start is not None:
        query_start = _query_start(query_start, B, device)
    else:
        _need(tokens == B, "without query_start there is one token for each sequence")
    k, v = _rows(k), _rows(v)
    ks, vs = k.stride(), v.stride()
    blocks = 0
    if k_scale is not None or v_scale is not None:
        k_scale, v_scale, blocks = _scales(k_scale, v_scale, pages, Hkv, ps, device)
    name, more = ("vk_hip_kv_cache_append_ex", (blocks,)) if blocks else ("vk_hip_kv_cache_append", ())
    status = _fn(name)(
        k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(),
        seq_lens.data_ptr(), query_start, k_scale, v_scale, *more, kind, B, tokens, Hkv, D, pages, ps,
        W, table_stride, ks[0], ks[1], vs[0], vs[1], strides[0], strides[1], strides[2],
        _stream(device))
    if status:
        _failed(status, name)


def kv_cache_read(k_cache, v_cache, block_table, seq_lens, *, query_start=None, tokens=None, k_scale=None, v_scale=None,
                  dtype=None, out=None):
    """Cached positions as rows: (k, v), each [tokens, Hkv, D].

    ``query_start`` [B + 1] int32: rows query_start[b] .. query_start[b + 1] - 1 are the last so many positions of
    sequence b, where ``kv_cache_append`` would have taken them from; ``tokens`` is how many rows there are.
    None: the last position of every sequence.  A 16-bit cache's rows come in its type; of an 8-bit one codes
    times scale ([Hkv] or [pages, Hkv, blocks]) in ``dtype``, bfloat16 (the default) or float16.
    Positions in front of the sequence and those of an entry that is no page are rows of zeros.  Rows that belong to no sequence
    are zeros in new tensors, and left as they are in ``out`` (a pair of tensors with rows that start on 16
    bytes)."""
    (pages, Hkv, ps, D), strides, device, (B, W), table_stride = _cache(k_cache, v_cache, block_table, seq_lens)
    if query_start is not None:
        _need(tokens is not None and 0 <= tokens < 1 << 31, "query_start needs tokens, the number of rows")
        query_start = _query_start(query_start, B, device)
    else:
        _need(tokens is None or tokens == B, "without query_start there is one token for each sequence")
        tokens = B
    if dtype is None:
        dtype = torch.bfloat16 if k_cache.dtype is torch.float8_e4m3fn else k_cache.dtype
    kind = _KINDS.get((k_cache.dtype, dtype))
    _need(kind is not None, "the cache's type does not give rows of this type")
    if out is None:
        k, v = (k_cache.new_empty((tokens, Hkv, D), dtype=dtype) for _ in range(2))
    else:
        k, v = out
        for t in (k, v):
            s = t.stride()
            _need(t.shape == (tokens, Hkv, D) and t.dtype is dtype and t.get_device() == device and s[2] == 1 and
                  s[0] % 8 == 0 and s[1] % 8 == 0 and t.data_ptr() % 16 == 0,
                  "out must be two [tokens, Hkv, D] on the cache's device with rows that start on 16 bytes")
    inputs = k_cache, v_cache, k_scale, v_scale
    wants_grad = torch.is_grad_enabled() and (
        k_cache.requires_grad or v_cache.requires_grad or k_scale is not None and k_scale.requires_grad or
        v_scale is not None and v_scale.requires_grad)
    if out is not None or _dual_level() >= 0:
        _refuse_derivatives("kv_cache_read", () if out is None else (k, v), *inputs)
    ks, vs = k.stride(), v.stride()
    k_scale, v_scale, blocks = _scales(k_scale, v_scale, pages, Hkv, ps, device)
    status = _fn("vk_hip_kv_cache_read")(
        k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(), query_start, k_scale, v_scale,
        blocks, k.data_ptr(), v.data_ptr(), kind, B, tokens, Hkv, D, pages, ps, W, table_stride, out is None,
        ks[0], ks[1], vs[0], vs[1], strides[0], strides[1], strides[2], _stream(device))
    if status:
        _failed(status, "vk_hip_kv_cache_read")
    if out is not None:
        increment_version((k, v))
    elif wants_grad:
        k, v = _read_result(k, v, *inputs)
    return k, v


def paged_attention(q, k_cache, v_cache, block_table, seq_lens, *, query_start=None, max_len=None, scale=None, window=0,
                    keep_first=0, softcap=0.0, sinks=None, k_scale=None, v_scale=None, weight_sums=None, return_lse=False, out=None):
    """Attention of one new token of every sequence, q [B, Hq, D], over its cached positions, or of several.

    Query heads G g .. G g + G - 1 read key/value head g (G = Hq / Hkv).  ``scale`` defaults to
    D ** -0.5; ``window`` > 0 leaves the last so many positions and the first ``keep_first``; ``softcap`` c > 0
    bounds the scores by c tanh(s / c); ``sinks`` [Hq] float32 are scores whose value is zero.  The scales of an
    8-bit cache are [Hkv], or [pages, Hkv, blocks] as ``kv_cache_append`` has written them.  ``max_len`` bounds every
    length (default: what the table holds; a longer sequence is cut to it): the launch and its
    workspace follow it, so a tight bound is worth giving.  ``weight_sums`` [B, Hkv, positions]
    float32: every position's weights, summed over the heads of the group, are added to it; the call's
    scratch is then 4 B Hq max_len bytes, whatever the lengths are.
    Returns out [B, Hq, D], or (out, lse [B, Hq] float32).  A row that nothing is left of is 0, its
    lse -inf (its sink, where there is one).

    With ``query_start`` [B + 1] int32 q is [tokens, Hq, D], rows query_start[b] .. query_start[b + 1] - 1 the last
    tokens of sequence b, whose keys and values are in the cache already (``kv_cache_append`` takes them by the
    same query_start): each sees the positions up to its own, the window and ``keep_first`` counted from
    there.  Rows that belong to no sequence are 0 with an lse of -inf, and left as they are in ``out``.
    There are no ``weight_sums`` then."""
    (pages, Hkv, ps, D), strides, device, (B, W), table_stride = _cache(k_cache, v_cache, block_table, seq_lens)
    Hq = q.shape[1] if q.dim() == 3 else 0
    G = Hq // Hkv
    rows = B if query_start is None else q.shape[0]
    if not (q.shape == (rows, G * Hkv, D) and 0 < G <= 0x7FFFFFFF and rows <= 0x7FFFFFFF and q.get_device() == device):
        raise ValueError("q must be [B, Hq, D] (with query_start [tokens, Hq, D]) on the cache's device with Hq a "
                         "multiple of the cache's heads")
    kind = _KINDS.get((k_cache.dtype, q.dtype))
    if kind is None:
        raise ValueError("the cache's type does not take queries of this type")
    if max_len is None:
        max_len = W * ps
    if not 0 < window < max_len:      # (any other sees everything, however large it is)
        window = 0
    if keep_first:
        _need(keep_first > 0, "keep_first must not be negative")
        keep_first = min(keep_first, max_len) if window else 0
    if not 0 <= max_len <= 0x7FFFFFFF:
        _int32(max_len=max_len)
    inputs, own_out = (q, k_cache, v_cache, sinks, k_scale, v_scale), out is not None
    wants_grad = torch.is_grad_enabled() and (
        q.requires_grad or k_cache.requires_grad or v_cache.requires_grad or sinks is not None and sinks.requires_grad or
        k_scale is not None and k_scale.requires_grad or v_scale is not None and v_scale.requires_grad)
    if _dual_level() >= 0:
        _refuse_derivatives("paged_attention", (), *inputs, out)
    q = _rows(q)
    if out is None:
        out = q.new_empty((rows, Hq, D))
    else:
        _need(out.shape == q.shape and out.dtype is q.dtype and out.is_contiguous() and out.get_device() == device,
              "out must be contiguous and like q")
        # (tiles whose scales are far from 1 read their queries a second time, behind the first results)
        if query_start is not None and kind >= 2 and out.untyped_storage().data_ptr() == q.untyped_storage().data_ptr():
            q = q.clone()
    lse = q.new_empty((rows, Hq), dtype=torch.float32) if return_lse else None
    sums, sums_b, sums_h = None, 0, 0
    if weight_sums is not None:
        if not _sums_ok(weight_sums, B, Hkv, max_len, device):
            raise ValueError("weight_sums must be float32 [B, Hkv, max_len or more] with contiguous rows on the cache's device")
        sums, (sums_b, sums_h, _) = weight_sums.data_ptr(), weight_sums.stride()
    blocks = 0
    if k_scale is not None or v_scale is not None:
        k_scale, v_scale, blocks = _scales(k_scale, v_scale, pages, Hkv, ps, device)
    sink_at = None if sinks is None else _head_vector(sinks, Hq, "sinks", device)
    lse_at = None if lse is None else lse.data_ptr()
    qs, scale = q.stride(), D ** -0.5 if scale is None else scale
    if own_out:
        # (ahead of the launch: what autograd does not let be written in place is an error, and nothing has run)
        wants_grad = wants_grad or torch.is_grad_enabled() and out.requires_grad
        if wants_grad:
            _given_attention_result(out, *inputs)
        else:
            increment_version(out)
    if query_start is None:
        size = _bytes("vk_hip_paged_attention_workspace_bytes_ex", kind, B, Hkv, G, D, max_len, window, keep_first,
                      sums is not None)
        workspace = q.new_empty((size,), dtype=torch.uint8) if size else None
        name, status = "vk_hip_paged_attention_ex", _fn("vk_hip_paged_attention_ex")(
            q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(), sink_at,
            k_scale, v_scale, blocks, out.data_ptr(), lse_at, sums, kind, B, Hkv, G, D, pages, ps, W, table_stride,
            max_len, window, keep_first, scale, softcap, qs[0], qs[1], strides[0], strides[1], strides[2], sums_b,
            sums_h, None if workspace is None else workspace.data_ptr(), size, _stream(device))
    else:
        _need(sums is None, "there are no weight_sums with query_start")
        if lse is not None and own_out:
            lse.fill_(float("-inf"))
        size = _bytes("vk_hip_paged_attention_prompt_workspace_bytes", B, rows, Hkv, G, D, max_len, window, keep_first)
        workspace = q.new_empty((size,), dtype=torch.uint8) if size else None
        name, status = "vk_hip_paged_attention_prompt", _fn("vk_hip_paged_attention_prompt")(
            q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(),
            _query_start(query_start, B, device), sink_at, k_scale, v_scale, blocks, out.data_ptr(), lse_at, kind, B, rows,
            Hkv, G, D, pages, ps, W, table_stride, max_len, window, keep_first, not own_out, scale, softcap, qs[0],
            qs[1], strides[0], strides[1], strides[2], None if workspace is None else workspace.data_ptr(), size,
            _stream(device))
    if status:
        _failed(status, name)
    if wants_grad:
        if not own_out:
            out, lse = _attention_result(out, lse, *inputs)
        elif lse is not None:
            lse, _ = _attention_result(lse, None, *inputs)
    return (out, lse) if return_lse else out


def kv_cache_evict(k_cache, v_cache, block_table, seq_lens, weight_sums, budget, *, keep_first=0, keep_last=0,
                   max_len=None, sums_out=None):
    """Cuts every sequence of more than ``budget`` positions to that many, in place.

    Each key/value head keeps the first ``keep_first`` and last ``keep_last`` positions and, of the
    others, those with the largest ``weight_sums`` [B, Hkv, positions] (NaN counts as largest, ties go
    to the lowest position); their rows move in order to positions 0 .. budget - 1.  The sums move
    along, with zeros from the budget up to the old length: in place, or to ``sums_out``.
    Returns (new_lens [B] int32, kept [B, Hkv, budget] int32: the old positions, -1 beyond the new
    length).  The pages of a sequence that is cut must be its own; those behind its new length are
    free afterwards.  Rows keep the position encoding they were stored with.  Positions without a page
    are not kept; a sequence that has one among its first ``budget`` positions or its last ``keep_last``
    is left as it is, with its old length in new_lens and 0 .. budget - 1 in kept."""
    (pages, Hkv, ps, D), strides, device, (B, W), table_stride = _cache(k_cache, v_cache, block_table, seq_lens)
    if max_len is None:
        max_len = W * ps
    _int32(max_len=max_len, budget=budget, keep_first=keep_first, keep_last=keep_last)
    sums_out = weight_sums if sums_out is None else sums_out
    for name, t in (("weight_sums", weight_sums), ("sums_out", sums_out)):
        _need(_sums_ok(t, B, Hkv, max_len, device),
              f"{name} must be float32 [B, Hkv, max_len or more] with contiguous rows on the cache's device")
    new_lens = torch.empty_like(seq_lens)
    kept = seq_lens.new_empty((B, Hkv, max(budget, 0)))
    elem = k_cache.element_size()
    size = _bytes("vk_hip_kv_cache_evict_workspace_bytes", elem, B, Hkv, D, max_len, budget)
    workspace = seq_lens.new_empty((size,), dtype=torch.uint8)
    ss, so = weight_sums.stride(), sums_out.stride()
    status = _fn("vk_hip_kv_cache_evict")(
        k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(), weight_sums.data_ptr(),
        sums_out.data_ptr(), new_lens.data_ptr(), kept.data_ptr(), elem, B, Hkv, D, pages, ps, W,
        table_stride, max_len, budget, keep_first, keep_last, strides[0], strides[1], strides[2],
        ss[0], ss[1], so[0], so[1], workspace.data_ptr(), size, _stream(device))
    if status:
        _failed(status, "vk_hip_kv_cache_evict")
    return new_lens, kept
