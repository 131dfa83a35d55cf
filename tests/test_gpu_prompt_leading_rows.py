"""GPU tests of prompts' attention where query_start does not begin at 0: the rows in front of it belong to no sequence."""
from __future__ import annotations

import math

import pytest
import torch

import attention_reference as aref
import kv_reference as ref
from test_gpu_kv_window import BF16, F16, Setup, dev
from vkernels_amd import kv_cache as kv

pytestmark = pytest.mark.gpu


def check(lens, new, lead, Hkv, G, D, ps, block, *, spare=0, q=BF16, **kw):
    s = Setup(lens, Hkv, G, D, ps, block, q=q, tokens=lead + sum(new) + spare, seed=lead + D)
    starts = (torch.tensor([0, *new]).cumsum(0) + lead).to(torch.int32).to(dev())
    args = dict(query_start=starts, k_scale=s.k_scale, v_scale=s.v_scale, return_lse=True, **kw)
    # (what new tensors are made of: nothing that could be taken for a result)
    for like in (s.q, torch.empty(s.q.shape[:2], device=dev())):
        torch.full_like(like, math.nan)
    out, lse = kv.paged_attention(s.q, s.k, s.v, s.table, s.lens, **args)
    given = torch.full_like(s.q, 3.0)
    _, given_lse = kv.paged_attention(s.q, s.k, s.v, s.table, s.lens, out=given, **args)
    torch.cuda.synchronize()
    bits = 11 if q is F16 or block else 8
    want = aref.attention(s.q, s.k, s.v, s.table, s.lens, starts, k_scale=s.k_scale, v_scale=s.v_scale, weight_bits=bits,
                          scale=D ** -0.5, **kw)
    mine = slice(lead, lead + sum(new))
    ref.assert_attention(out[mine], lse[mine], (want[0][mine], want[1][mine], None, (want[3][0][mine], want[3][1][mine], None)), q, "")
    assert torch.equal(given[mine], out[mine]) and torch.equal(given_lse, lse)
    rest = torch.ones(s.q.shape[0], dtype=torch.bool, device=dev())
    rest[mine] = False
    assert bool((out[rest] == 0).all()) and bool((lse[rest] == -math.inf).all()) and bool((given[rest] == 3).all())


@pytest.mark.parametrize("lead", [1, 7, 31, 32, 33, 100, 200])
@pytest.mark.parametrize("G", [1, 3, 33])
@pytest.mark.parametrize("lens,new", [([300, 64], [100, 33]), ([0, 40, 9], [0, 3, 1]), ([2000], [1])])
def test_rows_in_front(hip_lib, lead, G, lens, new):
    check(lens, new, lead, 2, G, 64, 16, 0, spare=2)


@pytest.mark.parametrize("block,D,q", [(0, 80, F16), (8, 128, BF16), (-1, 192, F16), (0, 256, BF16)])
@pytest.mark.parametrize("new", [(150, 70), (3, 5)])
def test_widths_and_types(hip_lib, block, D, q, new):
    check([4000, 700], new, 45, 2, 4, D, 16, block, q=q, window=500, keep_first=9)


def test_nothing_but_rows_of_no_sequence(hip_lib):
    check([50, 20], [0, 0], 70, 2, 3, 64, 16, 0)
    check([50, 20], [0, 0], 9, 2, 3, 64, 16, 0, spare=200)


def test_in_a_graph(hip_lib):
    """The same captured call with the first sequence's rows anywhere."""
    s = Setup([300, 200], 2, 4, 64, 16, 0, tokens=90)
    starts = torch.tensor([0, 30, 80], dtype=torch.int32, device=dev())
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out, lse = kv.paged_attention(s.q, s.k, s.v, s.table, s.lens, query_start=starts, return_lse=True)
    for places in ((0, 30, 80), (10, 40, 90), (60, 61, 61), (90, 90, 90), (3, 3, 70)):
        starts.copy_(torch.tensor(places, dtype=torch.int32))
        out.fill_(math.nan)
        lse.fill_(math.nan)
        graph.replay()
        want = kv.paged_attention(s.q, s.k, s.v, s.table, s.lens, query_start=starts, return_lse=True)
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
        assert bool((out[:places[0]] == 0).all() and (lse[:places[0]] == -math.inf).all())
        assert bool((out[places[-1]:] == 0).all() and (lse[places[-1]:] == -math.inf).all())
