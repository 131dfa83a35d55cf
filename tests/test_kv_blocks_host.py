"""CPU tests of the refusals of the block-scaled cache's, reading's and prompts' C entry points: nothing is launched."""
from __future__ import annotations

import pytest

from vkernels_amd import kv_cache as kv
from vkernels_amd import vllm_experts as ve

P = 4096          # an aligned address that nothing dereferences: every call here ends in the checks

APPEND = dict(k=P, v=P, k_cache=P, v_cache=P, block_table=P, seq_lens=P, query_start=None, k_scale=P, v_scale=P, scale_blocks=4,
              kind=2, B=4, tokens=4, Hkv=2, D=64, num_pages=8, page_size=16, table_width=4, table_stride=4, k_stride_t=128,
              k_stride_h=64, v_stride_t=128, v_stride_h=64, page_stride=2048, head_stride=1024, slot_stride=64, stream=None)
READ = dict(k_cache=P, v_cache=P, block_table=P, seq_lens=P, query_start=None, k_scale=P, v_scale=P, scale_blocks=4, k=P, v=P,
            kind=2, B=4, tokens=4, Hkv=2, D=64, num_pages=8, page_size=16, table_width=4, table_stride=4, clear_rest=1,
            k_stride_t=128, k_stride_h=64, v_stride_t=128, v_stride_h=64, page_stride=2048, head_stride=1024, slot_stride=64,
            stream=None)
ATTEND = dict(q=P, k_cache=P, v_cache=P, block_table=P, seq_lens=P, sinks=None, k_scale=P, v_scale=P, scale_blocks=4, out=P,
              lse=None, weight_sums=None, kind=2, B=4, Hkv=2, G=4, D=64, num_pages=8, page_size=16, table_width=400,
              table_stride=400, max_len=5000, window=0, keep_first=0, scale=0.125, softcap=0.0, q_stride_b=512, q_stride_h=64,
              page_stride=2048, head_stride=1024, slot_stride=64, sums_stride_b=0, sums_stride_h=0, workspace=P,
              workspace_bytes=1 << 40, stream=None)
PROMPT = dict(q=P, k_cache=P, v_cache=P, block_table=P, seq_lens=P, query_start=P, sinks=None, k_scale=P, v_scale=P,
              scale_blocks=4, out=P, lse=None, kind=2, B=4, tokens=20, Hkv=2, G=4, D=64, num_pages=8, page_size=16,
              table_width=400, table_stride=400, max_len=5000, window=0, keep_first=0, clear_rest=1, scale=0.125, softcap=0.0,
              q_stride_t=512, q_stride_h=64, page_stride=2048, head_stride=1024, slot_stride=64, workspace=P,
              workspace_bytes=1 << 40, stream=None)
CALLS = {"vk_hip_kv_cache_append_ex": APPEND, "vk_hip_kv_cache_read": READ, "vk_hip_paged_attention_ex": ATTEND,
         "vk_hip_paged_attention_prompt": PROMPT}

CACHE = [dict(D=0), dict(D=24), dict(D=272), dict(Hkv=0), dict(num_pages=0), dict(page_size=0), dict(table_width=0),
         dict(table_stride=-1), dict(k_cache=None), dict(v_cache=None), dict(block_table=None), dict(seq_lens=None),
         dict(k_cache=P + 8), dict(v_cache=P + 2), dict(page_stride=2044), dict(slot_stride=-64), dict(slot_stride=1 << 27),
         dict(scale_blocks=3), dict(scale_blocks=-1), dict(scale_blocks=32), dict(k_scale=None), dict(v_scale=None),
         dict(kind=0), dict(kind=0, k_scale=None, v_scale=None), dict(B=-1)]
INVALID = {
    "vk_hip_kv_cache_append_ex": CACHE + [
        dict(k=None), dict(v=P + 8), dict(k_stride_t=132), dict(tokens=3), dict(tokens=-1), dict(page_stride=0), dict(head_stride=0),
        dict(slot_stride=0)],
    "vk_hip_kv_cache_read": CACHE + [
        dict(k=None), dict(v=None), dict(k=P + 8), dict(v_stride_h=68), dict(tokens=3), dict(tokens=-1), dict(k_stride_t=0),
        dict(v_stride_h=0), dict(k_stride_t=64), dict(k_stride_h=-64), dict(B=0, tokens=5, query_start=P)],
    "vk_hip_paged_attention_ex": CACHE + [
        dict(q=None), dict(out=P + 2), dict(G=0), dict(max_len=6401), dict(keep_first=-1), dict(softcap=-1.0), dict(workspace=None),
        dict(workspace_bytes=16)],
    "vk_hip_paged_attention_prompt": CACHE + [
        dict(q=None), dict(out=None), dict(query_start=None), dict(q=P + 4), dict(out=P + 2), dict(q_stride_t=516), dict(G=0),
        dict(max_len=-1), dict(max_len=6401), dict(keep_first=-1), dict(softcap=float("nan")), dict(workspace=None),
        dict(workspace_bytes=16), dict(workspace=P + 8), dict(tokens=-1), dict(B=0)],
}
OTHER = [
    *((name, dict(kind=4), ve.VK_ERROR_UNSUPPORTED) for name in CALLS),
    ("vk_hip_kv_cache_append_ex", dict(B=1 << 20, tokens=1 << 20, Hkv=64, D=256), ve.VK_ERROR_OUT_OF_RANGE),
    ("vk_hip_kv_cache_append_ex", dict(B=1 << 24, tokens=64, query_start=P, Hkv=16), ve.VK_ERROR_OUT_OF_RANGE),
    ("vk_hip_kv_cache_read", dict(B=1 << 20, tokens=1 << 20, Hkv=64, D=256, k_stride_t=1 << 14, k_stride_h=256,
                                  v_stride_t=1 << 14, v_stride_h=256), ve.VK_ERROR_OUT_OF_RANGE),
    ("vk_hip_kv_cache_read", dict(B=1 << 24, tokens=1 << 24, Hkv=1), ve.VK_ERROR_OUT_OF_RANGE),
    ("vk_hip_paged_attention_prompt", dict(tokens=1 << 29, G=8), ve.VK_ERROR_OUT_OF_RANGE),
    ("vk_hip_paged_attention_prompt", dict(B=1 << 24), ve.VK_ERROR_OUT_OF_RANGE),
    ("vk_hip_paged_attention_prompt", dict(tokens=1 << 26, Hkv=16, G=8), ve.VK_ERROR_OUT_OF_RANGE),
    ("vk_hip_paged_attention_prompt", dict(table_width=1 << 28, table_stride=1 << 28, max_len=(1 << 31) - 64), ve.VK_ERROR_OUT_OF_RANGE),
]
NOTHING = [("vk_hip_kv_cache_append_ex", dict(B=0, tokens=0)), ("vk_hip_kv_cache_append_ex", dict(tokens=0, query_start=P)),
           ("vk_hip_kv_cache_read", dict(tokens=0, query_start=P, k=None, v=None)), ("vk_hip_kv_cache_read", dict(B=0, tokens=0)),
           ("vk_hip_paged_attention_ex", dict(B=0, q=None)), ("vk_hip_paged_attention_prompt", dict(tokens=0, q=None, out=None))]


@pytest.fixture(scope="module")
def lib():
    return ve.load_libvkernels_hip()


def _call(name, change):
    return kv._fn(name)(*dict(CALLS[name], **change).values())


@pytest.mark.parametrize("name,change", [(n, c) for n, cs in INVALID.items() for c in cs])
def test_invalid_arguments(lib, name, change):
    lib.vk_set_last_error(0, b"")
    assert _call(name, change) == ve.VK_ERROR_INVALID_ARGUMENT
    assert name in ve.last_error(lib)


@pytest.mark.parametrize("name,change,code", OTHER)
def test_other_refusals(lib, name, change, code):
    assert _call(name, change) == code


@pytest.mark.parametrize("name,change", NOTHING)
def test_nothing_to_do(lib, name, change):
    assert _call(name, change) == ve.VK_OK


def test_workspaces(lib):
    step, prompt = (kv._fn(f"vk_hip_paged_attention_{n}") for n in ("workspace_bytes_ex", "prompt_workspace_bytes"))
    assert step(0, 64, 8, 4, 128, 8192, 0, 100, 0) == step(0, 64, 8, 4, 128, 8192, 0, 0, 0) > 0
    assert step(0, 64, 8, 4, 128, 8192, 100, 4, 0) == 0 < step(0, 64, 8, 4, 128, 8192, 100, 2000, 0)
    assert step(0, 64, 8, 4, 128, 8192, 100, 2 ** 31 - 1, 0) == step(0, 64, 8, 4, 128, 8192, 0, 0, 0)
    assert step(0, 64, 8, 4, 128, 8192, 100, -1, 0) == 0
    assert prompt(1, 4096, 8, 4, 128, 16384, 0, 0) == 0 < prompt(1, 5, 8, 4, 128, 131072, 0, 0)
    assert prompt(1, 5, 8, 4, 128, 131072, 64, 4) == 0 == prompt(0, 5, 8, 4, 128, 131072, 0, 0) == prompt(1, 1 << 30, 8, 4, 128, 100, 0, 0)
