"""CPU tests of the key-value cache's C entry points: contract violations are refused before anything is
launched, with the code and a message, and calls with nothing to do succeed."""
from __future__ import annotations

import pytest

from vkernels_amd import kv_cache as kv
from vkernels_amd import vllm_experts as ve

P = 4096          # an aligned address that nothing dereferences: every call here ends in the checks

APPEND = dict(k=P, v=P, k_cache=P, v_cache=P, block_table=P, seq_lens=P, query_start=None, k_scale=None, v_scale=None,
              kind=0, B=4, tokens=4, Hkv=2, D=64, num_pages=8, page_size=16, table_width=4, table_stride=4,
              k_stride_t=128, k_stride_h=64, v_stride_t=128, v_stride_h=64, page_stride=2048, head_stride=1024,
              slot_stride=64, stream=None)
ATTEND = dict(q=P, k_cache=P, v_cache=P, block_table=P, seq_lens=P, sinks=None, k_scale=None, v_scale=None, out=P,
              lse=None, weight_sums=None, kind=0, B=4, Hkv=2, G=4, D=64, num_pages=8, page_size=16, table_width=400,
              table_stride=400, max_len=5000, window=0, scale=0.125, softcap=0.0, q_stride_b=512, q_stride_h=64,
              page_stride=2048, head_stride=1024, slot_stride=64, sums_stride_b=0, sums_stride_h=0, workspace=P,
              workspace_bytes=1 << 40, stream=None)
EVICT = dict(k_cache=P, v_cache=P, block_table=P, seq_lens=P, weight_sums=P, sums_out=P, new_lens=2 * P, kept=P,
             elem_bytes=2, B=4, Hkv=2, D=64, num_pages=8, page_size=16, table_width=4, table_stride=4, max_len=64,
             budget=32, keep_first=4, keep_last=8, page_stride=2048, head_stride=1024, slot_stride=64,
             sums_stride_b=128, sums_stride_h=64, out_stride_b=128, out_stride_h=64, workspace=P, workspace_bytes=1 << 40,
             stream=None)
CALLS = {"vk_hip_kv_cache_append": APPEND, "vk_hip_paged_attention": ATTEND, "vk_hip_kv_cache_evict": EVICT}

CACHE = [dict(D=0), dict(D=24), dict(D=272), dict(D=-16), dict(Hkv=0), dict(num_pages=0), dict(page_size=0),
         dict(table_width=0), dict(table_stride=-1), dict(k_cache=None), dict(v_cache=None), dict(block_table=None),
         dict(seq_lens=None), dict(k_cache=P + 8), dict(v_cache=P + 2), dict(page_stride=2044), dict(head_stride=1028),
         dict(slot_stride=68), dict(slot_stride=-64), dict(slot_stride=1 << 27), dict(B=-1)]
INVALID = {
    "vk_hip_kv_cache_append": CACHE + [
        dict(k=None), dict(v=None), dict(k=P + 8), dict(k_stride_t=132), dict(v_stride_h=65), dict(tokens=3),
        dict(tokens=-1), dict(kind=2), dict(kind=2, k_scale=P), dict(k_scale=P, v_scale=P)],
    "vk_hip_paged_attention": CACHE + [
        dict(q=None), dict(out=None), dict(q=P + 4), dict(out=P + 2), dict(q_stride_b=516), dict(q_stride_h=68),
        dict(G=0), dict(max_len=-1), dict(max_len=6401), dict(softcap=-1.0), dict(softcap=float("nan")), dict(kind=3),
        dict(kind=3, v_scale=P), dict(k_scale=P, v_scale=P), dict(workspace=None), dict(workspace_bytes=16),
        dict(workspace=P + 8)],
    "vk_hip_kv_cache_evict": CACHE + [
        dict(weight_sums=None), dict(sums_out=None), dict(new_lens=None), dict(kept=None), dict(max_len=65),
        dict(max_len=-1), dict(budget=0), dict(budget=-3), dict(keep_first=-1), dict(keep_last=-1), dict(keep_first=25),
        dict(out_stride_b=64), dict(new_lens=P), dict(workspace=None), dict(workspace_bytes=4), dict(workspace=P + 2)],
}
OTHER = [
    ("vk_hip_kv_cache_append", dict(kind=4), ve.VK_ERROR_UNSUPPORTED),
    ("vk_hip_kv_cache_append", dict(B=1 << 20, tokens=1 << 20, Hkv=64, D=256, k_stride_t=1 << 14, v_stride_t=1 << 14),
     ve.VK_ERROR_OUT_OF_RANGE),
    ("vk_hip_paged_attention", dict(kind=-1), ve.VK_ERROR_UNSUPPORTED),
    ("vk_hip_paged_attention", dict(B=1 << 20, Hkv=64, G=64), ve.VK_ERROR_OUT_OF_RANGE),
    ("vk_hip_paged_attention", dict(B=1 << 20, Hkv=32, table_width=1 << 20, table_stride=1 << 20, max_len=1 << 23),
     ve.VK_ERROR_OUT_OF_RANGE),
    ("vk_hip_paged_attention", dict(B=1 << 20, Hkv=16, G=1, max_len=100), ve.VK_ERROR_OUT_OF_RANGE),
    ("vk_hip_paged_attention", dict(B=1, Hkv=1, G=1, table_width=1 << 28, table_stride=1 << 28, max_len=(1 << 31) - 64),
     ve.VK_ERROR_OUT_OF_RANGE),
    ("vk_hip_kv_cache_evict", dict(B=1, Hkv=1, table_width=1 << 28, table_stride=1 << 28, max_len=(1 << 31) - 64),
     ve.VK_ERROR_OUT_OF_RANGE),
    ("vk_hip_kv_cache_evict", dict(B=1 << 17, Hkv=64, max_len=60), ve.VK_ERROR_OUT_OF_RANGE),
    ("vk_hip_kv_cache_evict", dict(elem_bytes=4), ve.VK_ERROR_UNSUPPORTED),
    ("vk_hip_kv_cache_evict", dict(B=1 << 26, Hkv=32), ve.VK_ERROR_OUT_OF_RANGE),
    ("vk_hip_kv_cache_evict", dict(budget=1 << 28, D=256), ve.VK_ERROR_OUT_OF_RANGE),
]


@pytest.fixture(scope="module")
def lib():
    return ve.load_libvkernels_hip()


@pytest.mark.parametrize("name,change", [(n, c) for n, cs in INVALID.items() for c in cs],
                         ids=lambda x: x if isinstance(x, str) else ",".join(f"{k}={v}" for k, v in x.items()))
def test_contract_violations_are_refused(lib, name, change):
    args = dict(CALLS[name], **change)
    if "sums_out" in args and "out_stride_b" not in change:
        args["sums_out"] = args["sums_out"] and 3 * P
    lib.vk_set_last_error(0, b"")
    assert kv._fn(name)(*args.values()) == ve.VK_ERROR_INVALID_ARGUMENT
    assert ve.last_error(lib).startswith(name + ": ")


@pytest.mark.parametrize("name,change,code", OTHER)
def test_calls_beyond_what_is_supported(lib, name, change, code):
    assert kv._fn(name)(*dict(CALLS[name], **change).values()) == code
    assert ve.last_error(lib).startswith(name + ": ")


@pytest.mark.parametrize("name", list(CALLS))
def test_calls_with_nothing_to_do(lib, name):
    assert kv._fn(name)(*dict(CALLS[name], B=0, **({"tokens": 0} if "tokens" in CALLS[name] else {})).values()) == ve.VK_OK


def test_workspace_bytes(lib):
    size = kv._fn("vk_hip_paged_attention_workspace_bytes")
    assert size(0, 0, 8, 4, 64, 1000, 0, 0) == 0
    assert size(0, 64, 8, 4, 64, 100, 0, 0) == 0              # short calls need none
    plain, counted = size(0, 64, 8, 4, 128, 8192, 0, 0), size(0, 64, 8, 4, 128, 8192, 0, 1)
    assert 0 < plain < counted
    assert counted >= plain + 4 * 64 * 32 * 8192           # every score is kept
    assert size(0, 64, 8, 4, 128, 100, 0, 1) >= 4 * 64 * 32 * 100


@pytest.mark.parametrize("window", [8192 - 16, 8192, 2 ** 31 - 17, 2 ** 31 - 16, 2 ** 31 - 1, -1, -2 ** 31])
@pytest.mark.parametrize("counted", [0, 1])
def test_a_window_beyond_the_lengths_is_planned_like_none(lib, window, counted):
    """The largest integers are a usual way to say that there is no window."""
    size = kv._fn("vk_hip_paged_attention_workspace_bytes")
    for B, Hkv, G in ((64, 8, 4), (8, 8, 4), (1, 1, 40)):
        assert size(0, B, Hkv, G, 128, 8192, window, counted) == size(0, B, Hkv, G, 128, 8192, 0, counted) > 0


@pytest.mark.parametrize("name,change", [
    *((name, change) for name in ("vk_hip_kv_cache_append", "vk_hip_kv_cache_evict")
      for change in (dict(page_stride=0), dict(head_stride=0), dict(slot_stride=0))),
    ("vk_hip_paged_attention", dict(weight_sums=P, sums_stride_b=0, sums_stride_h=6400)),
    ("vk_hip_paged_attention", dict(weight_sums=P, sums_stride_b=12800, sums_stride_h=0)),
    ("vk_hip_kv_cache_evict", dict(out_stride_b=0, sums_out=3 * P)),
    ("vk_hip_kv_cache_evict", dict(out_stride_h=0, sums_out=3 * P))])
def test_what_is_written_to_must_not_be_broadcast(lib, name, change):
    """Pages, heads, positions or sums that share their memory would be written by several workgroups at once."""
    lib.vk_set_last_error(0, b"")
    args = dict(CALLS[name], **change)
    if name == "vk_hip_kv_cache_evict":
        args["sums_out"] = 3 * P
    assert kv._fn(name)(*args.values()) == ve.VK_ERROR_INVALID_ARGUMENT
    assert "broadcast" in ve.last_error(lib)
