"""Randomised calls of the key-value cache's operators: types, head layouts, widths, page sizes, lengths,
windows, caps, sinks, holes, bounds and budgets drawn together, against the definitions."""
from __future__ import annotations

import random

import pytest
import torch

import kv_reference as ref
from test_gpu_kv_cache import BF16, F16, FP8, Setup, _check_evict, dev
from vkernels_amd import kv_cache as kv

pytestmark = pytest.mark.gpu


def _setup(rng, longest, most_rows, G=True):
    cache, q = rng.choice(((BF16, BF16), (F16, F16), (FP8, BF16), (FP8, F16)))
    B, Hkv = rng.choice((1, 1, 2, 3, 5, 9, 70)), rng.choice((1, 1, 2, 3, 5))
    g = rng.choice((1, 2, 3, 4, 7, 8, 16, 19)) if G else 1
    longest = min(longest, max(40, most_rows // (B * Hkv * g)))
    lens = [rng.choice((0, 1, longest, rng.randint(1, longest), rng.randint(1, longest))) for _ in range(B)]
    lens[rng.randrange(B)] = longest
    return Setup(lens, Hkv, g, 16 * rng.randint(1, 16), rng.choice((1, 5, 8, 16, 16, 24, 32, 48, 64, 130)), cache=cache, q=q,
                 layout=rng.choice(("heads", "tokens")), seed=rng.randrange(1 << 30), peak=rng.choice((0.2, 1.0, 4.0)),
                 spare=rng.randint(1, 9))


@pytest.mark.parametrize("seed", range(60))
def test_attention(hip_lib, seed):
    rng = random.Random(seed)
    s = _setup(rng, rng.choice((60, 300, 1500, 4000)), 60000)
    longest = int(s.lens.max())
    if rng.random() < 0.3:                     # pages that are not there
        gone = torch.rand(s.table.shape, generator=torch.Generator().manual_seed(seed)) < 0.2
        s.table[gone.to(dev())] = rng.choice((-1, s.k.shape[0], 2 ** 31 - 1, -2 ** 31))
    kw = {}
    if rng.random() < 0.3:
        kw["window"] = rng.randint(1, longest + 20)
    if rng.random() < 0.3:
        kw["softcap"] = rng.choice((1.0, 15.0, 50.0))
    if rng.random() < 0.2:
        kw["scale"] = rng.choice((0.01, 0.3, -0.2))
    if rng.random() < 0.5:
        kw["max_len"] = rng.choice((longest, max(1, longest // 2), min(longest + 700, s.table.shape[1] * s.ps)))
    s.check(counted=rng.random() < 0.6, sinks=rng.random() < 0.4, what=f"seed {seed} {kw}", **kw)


@pytest.mark.parametrize("seed", range(30))
def test_append(hip_lib, seed):
    rng = random.Random(1000 + seed)
    s = _setup(rng, 200, 4000, G=False)
    lens = s.lens.cpu().tolist()
    new = None if rng.random() < 0.3 else [rng.randint(0, n) if rng.random() < 0.7 else 0 for n in lens]
    n = s.B if new is None else sum(new)
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn((n, s.Hkv, s.D), generator=g).to(s.q.dtype).to(dev()) for _ in range(2))
    starts = None if new is None else torch.tensor([0] + new).cumsum(0).to(torch.int32).to(dev())
    want = ref.append(s.k, s.v, k, v, s.table, s.lens, starts, s.k_scale, s.v_scale)
    kv.kv_cache_append(k, v, s.k, s.v, s.table, s.lens, query_start=starts, k_scale=s.k_scale, v_scale=s.v_scale)
    word = torch.uint8 if s.k.element_size() == 1 else torch.int16
    for got, exp in zip((s.k, s.v), want):
        assert torch.equal(got.cpu().contiguous().view(word), exp.contiguous().view(word))


@pytest.mark.parametrize("seed", range(40))
def test_evict(hip_lib, seed):
    rng = random.Random(2000 + seed)
    s = _setup(rng, rng.choice((100, 700, 5000, 18000)), 60000, G=False)
    longest = int(s.lens.max())
    budget = rng.randint(1, longest + 5)
    first = rng.randint(0, budget) if rng.random() < 0.7 else 0
    last = rng.randint(0, budget - first) if rng.random() < 0.7 else 0
    g = torch.Generator(device=dev()).manual_seed(seed)
    sums = torch.rand((s.B, s.Hkv, s.table.shape[1] * s.ps + rng.randint(0, 5)), device=dev(), generator=g)
    kind = rng.choice(("spread", "few", "close", "signed"))
    sums = {"spread": torch.exp(12 * sums - 6), "few": (3 * sums).floor(), "close": 1 + sums * 2 ** -20,
            "signed": sums - 0.5}[kind]
    _check_evict(s, sums, budget, first, last, in_place=rng.random() < 0.5)
