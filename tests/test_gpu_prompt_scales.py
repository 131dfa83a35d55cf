"""GPU tests of prompts' attention over 8-bit caches whose value scales are of any size, as kv_cache_append may write them
from bf16 rows: from 2^-110 to 2^100."""
from __future__ import annotations

import math

import pytest
import torch

import attention_reference as aref
import kv_reference as ref
from test_gpu_kv_window import BF16, F16, dev
from test_gpu_prompt_attention import Prompt
from vkernels_amd import kv_cache as kv

pytestmark = pytest.mark.gpu


def check(s, **kw):
    out, lse = s.call(**kw)
    torch.cuda.synchronize()
    want = aref.attention(s.q, s.k, s.v, s.table, s.lens, s.starts, k_scale=s.k_scale, v_scale=s.v_scale, weight_bits=11,
                          scale=s.D ** -0.5, **kw)
    # A weight times its scale ends at bf16's least step: each of up to 700 is off by half of that, 2^-134, times a code of
    # up to 448 (which shows where scales are near 2^-110 alone), and the result by half of it.
    out_tol = want[3][0] + 700 * 448 * 2.0 ** -134 + 2.0 ** -134
    ref.assert_attention(out, lse, (*want[:2], None, (out_tol, want[3][1], None)), s.q.dtype, "")


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("size", [2.0 ** -110, 2.0 ** -70, 2.0 ** 66, 2.0 ** 100])
@pytest.mark.parametrize("new,block", [((200, 150), 16), ((200, 150), -1), ((40, 60), 4), ((3, 5), 16)])
def test_sizes(hip_lib, D, size, new, block):
    s = Prompt([700, 600], new, 2, 4, D, 16, block, seed=D)
    s.v_scale = s.v_scale * size
    check(s, sinks=s.sinks)
    check(s, window=100, keep_first=20, softcap=20.0)


@pytest.mark.parametrize("new", [(500, 300), (3, 5)])
@pytest.mark.parametrize("q,low,high", [(BF16, 2.0 ** -100, 1.0), (F16, 2.0 ** -100, 1.0), (BF16, 1.0, 2.0 ** 100),
                                        (BF16, 2.0 ** -100, 2.0 ** 100), (BF16, 2.0 ** -60, 2.0 ** 62)])
def test_sizes_side_by_side(hip_lib, q, new, low, high):
    """64 positions of small values, 64 of large ones, and so on, with windows of 32: a row that sees one kind has a
    result of that kind, whatever the others of its tile see."""
    s = Prompt([900, 700], new, 1, 2, 64, 16, 4, q=q, seed=3)
    big = torch.zeros_like(s.v_scale)
    pages = s.table.long()
    for b, n in enumerate((900, 700)):
        for w in range(-(-n // 16)):
            big[pages[b, w]] = float(w // 4 % 2)
    s.v_scale = s.v_scale * torch.where(big > 0, high, low)
    out, lse = s.call(window=32)
    torch.cuda.synchronize()
    assert bool(torch.isfinite(out).all() and torch.isfinite(lse).all())
    queries, k, v = s.q.cpu().double(), s.k.cpu().float().double(), s.v.cpu().float().double()
    scales = [x.cpu().double().repeat_interleave(4, 2)[..., None] for x in (s.k_scale, s.v_scale)]
    k, v = k * scales[0], v * scales[1]
    half = torch.finfo(q).eps / 2
    row = 0
    for b, (n, count) in enumerate(zip((900, 700), new)):
        at = torch.arange(n)
        page = pages[b].cpu()[at // 16]
        keys, values = k[page, 0, at % 16], v[page, 0, at % 16]
        for place in range(n - count, n):
            seen = slice(max(0, place - 31), place + 1)
            score = (queries[row] @ keys[seen].t()) * 64 ** -0.5
            p = torch.softmax(score, 1)
            want, size = p @ values[seen], p @ values[seen].abs()
            # a score: D products and their sum in 32 bits (64 2^-23 of their magnitudes), its scale and its way to a power
            # of two 2^-21 of it; the weight 11 bits and, relative to them, 32 sums; the result half a step, and the least
            # step of its type
            err = 64 * 2.0 ** -23 * (queries[row].abs() @ keys[seen].abs().t()).amax() * 64 ** -0.5 + 2.0 ** -20 * score.abs().amax()
            bound = (2 * float(err) + 2.0 ** -11 + 2.0 ** -18) * size
            # (of scales that lie 2^122 apart in one window: what is 2^-40 of the row's largest value times weight may go)
            bound = bound + 2.0 ** -40 * size.amax(1, keepdim=True)
            least = 2.0 ** -25 if q is F16 else 2.0 ** -134
            got = out[row].cpu().double()
            assert bool(((got - want).abs() <= bound + half * (want.abs() + bound) + least).all()), (b, place)
            row += 1


def test_what_append_writes(hip_lib):
    """Rows near the ends of bf16 go in and come out."""
    for size in (1e30, 1e-30):
        caches = [torch.zeros((20, 2, 16, 64), dtype=torch.float8_e4m3fn, device=dev()) for _ in range(2)]
        scales = dict(zip(("k_scale", "v_scale"), (torch.zeros((20, 2, 1), device=dev()) for _ in range(2))))
        g = torch.Generator().manual_seed(2)
        k, v = (torch.randn((300, 2, 64), generator=g).to(BF16).to(dev()) for _ in range(2))
        q = torch.randn((300, 8, 64), generator=g).to(BF16).to(dev())
        table = torch.randperm(20, generator=g).to(torch.int32).to(dev())[None]
        lens = torch.tensor([300], dtype=torch.int32, device=dev())
        starts = torch.tensor([0, 300], dtype=torch.int32, device=dev())
        kv.kv_cache_append(k, v * size, *caches, table, lens, query_start=starts, **scales)
        out = kv.paged_attention(q, *caches, table, lens, query_start=starts, **scales)
        step = kv.paged_attention(q[-1:], *caches, table, lens, **scales)
        assert bool(torch.isfinite(out).all()) and bool((out != 0).any(2).all())
        # (each within its weights' 11 or 16 bits and half a step of the result)
        near = (out[-1:] - step).abs().float() / size
        assert float(near.max()) <= 2 * 2.0 ** -8 * float((step.abs().float() / size).max()) + 2.0 ** -10 * 4


def test_infinite_scales_that_are_not_seen(hip_lib):
    """Positions hidden from every row of a tile that it loads all the same: nothing of them is left."""
    s = Prompt([130], [64], 1, 2, 64, 16, 16)
    clean = s.call(window=16)
    for value in (math.inf, -math.inf, math.nan, 2.0 ** 120):
        s.v_scale[s.table[0, 0].long()] = value          # positions 0 .. 15
        out, lse = s.call(window=16)
        assert torch.equal(out, clean[0]) and torch.equal(lse, clean[1])


@pytest.mark.parametrize("ps,block", [(24, 8), (16, 1), (16, 16), (5, 5)])
@pytest.mark.parametrize("far", [0, 5, 400, 717, 899])
@pytest.mark.parametrize("window,first", [(0, 0), (64, 6), (200, 0), (64, 500)])
def test_one_block_far_from_the_others(hip_lib, ps, block, far, window, first):
    """Wherever it lies: rows that see it are what the definition says, the others as if it were not there."""
    s = Prompt([900, 130], [300, 70], 2, 4, 64, ps, block, seed=far + ps)
    clean = s.call(window=window, keep_first=first)[0].double().cpu()
    page = int(s.table[0, far // ps])
    s.v_scale[page, :, far % ps // block] *= 2.0 ** 70
    check(s, window=window, keep_first=first)
    out = s.call(window=window, keep_first=first)[0].double().cpu()
    begin, end = far // block * block, far // block * block + block
    seen = torch.tensor([any(p <= place and (not window or p > place - window or p < first) for p in range(begin, min(end, 900)))
                         for place in range(600, 900)] + [False] * 70)
    # Both calls are within their weights' 2^-11 and their scores' rounding (64 2^-23 of products that sum up to some 10,
    # twice: below 2^-11) of the largest value, and half a step of the result.
    most = float((s.v.float().cpu().nan_to_num() * 0.3).abs().max())      # (scales are e^(0.7 x) / 60, codes up to some 240)
    bound = 4 * 2.0 ** -11 * most + 2 * 2.0 ** -8 * clean.abs()
    assert bool(((out - clean).abs() <= bound)[~seen].all())
    assert not bool(seen.any()) or float(out[seen].abs().max()) > 2.0 ** 40


def test_in_a_graph(hip_lib):
    """Scales that come and go between replays of one captured call."""
    s = Prompt([700, 600], (200, 150), 2, 4, 128, 16, 16)
    ordinary = s.v_scale.clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out, lse = s.call(max_len=int(s.table.shape[1]) * 16)
    for size in (1.0, 2.0 ** 80, 1.0, 2.0 ** -80, 0.5):
        s.v_scale.copy_(ordinary * size)
        out.fill_(math.nan)
        graph.replay()
        want = s.call(max_len=int(s.table.shape[1]) * 16)
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
        check(s)


def test_results_in_the_queries_place(hip_lib):
    """Tiles that are worked on again read their queries again."""
    s = Prompt([700, 600], (200, 150), 2, 4, 64, 16, 16)
    s.v_scale = s.v_scale * 2.0 ** 80
    want = s.call()
    got = s.call(out=s.q)
    assert got[0] is s.q and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
