"""GPU tests of the eviction where the block table has entries that are no page: their positions are never
kept, and a sequence whose kept positions would come from or go to one is left as it is."""
from __future__ import annotations

import random

import numpy as np
import pytest
import torch

import kv_reference as ref
from test_gpu_kv_cache import BF16, F16, FP8, Setup, dev
from vkernels_amd import kv_cache as kv

pytestmark = pytest.mark.gpu


def _want(s, sums, out, budget, first, last):
    """(k, v, sums_out, new_lens, kept) by the definition, on the CPU."""
    caches = [c.detach().cpu().clone() for c in (s.k, s.v)]
    words = [c.view(torch.uint8) if c.element_size() == 1 else c for c in caches]
    table, lens, sums, out = s.table.cpu().numpy(), s.lens.cpu().tolist(), sums.cpu().numpy(), out.cpu().clone()
    kept = np.full((s.B, s.Hkv, budget), -1, dtype=np.int32)
    new_lens = []
    for b, n in enumerate(lens):
        _, _, there = ref.positions(table[b], n, s.ps, s.k.shape[0])
        cut = n > budget and there[:budget].all() and there[n - last:].all()
        new_lens.append(budget if cut else n)
        for h in range(s.Hkv):
            if not cut:
                kept[b, h, :n] = np.arange(n)[:budget]
                out[b, h, :n] = torch.from_numpy(sums[b, h, :n].copy())
                continue
            middle = np.arange(first, n - last)[there[first:n - last]]
            key = sums[b, h, middle].astype(np.float64)
            best = middle[np.lexsort((middle, -np.nan_to_num(key, nan=np.inf), ~np.isnan(key)))][:budget - first - last]
            at = np.sort(np.concatenate([np.arange(first), best, np.arange(n - last, n)]))
            assert len(at) == budget
            kept[b, h] = at
            j = np.arange(budget)
            for c in words:
                c[table[b, j // s.ps], h, j % s.ps] = c[table[b, at // s.ps], h, at % s.ps].clone()
            out[b, h, :n] = 0.0
            out[b, h, :budget] = torch.from_numpy(sums[b, h, at].copy())
    return caches[0], caches[1], out, torch.tensor(new_lens, dtype=torch.int32), torch.from_numpy(kept)


def _check(s, sums, budget, first, last, in_place):
    out = sums if in_place else torch.full_like(sums, 7.0)
    want = _want(s, sums, out, budget, first, last)
    new_lens, kept = kv.kv_cache_evict(s.k, s.v, s.table, s.lens, sums, budget, keep_first=first, keep_last=last,
                                       sums_out=None if in_place else out)
    word = torch.uint8 if s.k.element_size() == 1 else torch.int16
    assert torch.equal(new_lens.cpu(), want[3])
    assert torch.equal(kept.cpu(), want[4])
    assert torch.equal(s.k.cpu().contiguous().view(word), want[0].contiguous().view(word))
    assert torch.equal(s.v.cpu().contiguous().view(word), want[1].contiguous().view(word))
    assert torch.equal(out.cpu().view(torch.int32), want[2].view(torch.int32))


# a row's workgroup of 256 threads; of 1024, with its sums in registers and not; several workgroups a row
@pytest.mark.parametrize("n,width", [(700, None), (5000, None), (20000, None), (20000, 2100)])
@pytest.mark.parametrize("budget,first,last", [(100, 3, 20), (333, 0, 0), (64, 16, 48)])
@pytest.mark.parametrize("largest", [False, True])
def test_positions_without_a_page(hip_lib, n, width, budget, first, last, largest):
    """Holes between the new places and the last positions, in the way of either, behind the length, and
    everywhere; their sums zero, as the attention leaves them, or larger than all others."""
    s = Setup([n, n - 5, n, n - 16, n, n, n - 3, 60, n], 2, 1, 16, 16, seed=n, width=width)
    no_page = [-1, s.k.shape[0], 2 ** 31 - 1, -2 ** 31]
    behind = -(-budget // 16)
    entries = [-(-int(x) // 16) for x in s.lens]
    s.table[0, behind] = no_page[0]                                   # the first that is in nobody's way
    s.table[1, behind + 1:entries[1] - 4:2] = no_page[1]              # many of them
    s.table[2, behind - 1] = no_page[2]                               # the last new place's page
    s.table[3, 0] = no_page[3]
    s.table[4, entries[4] - 1] = no_page[0]                           # the last positions' page
    s.table[5, entries[5] - -(-last // 16) - 1] = no_page[1]          # one in front of theirs
    s.table[6, entries[6]:] = no_page[2]
    s.table[7, 1] = no_page[0]                                        # of a sequence within the budget
    s.table[8, :] = no_page[0]
    g = torch.Generator(device=dev()).manual_seed(n + budget)
    sums = torch.rand((9, 2, s.table.shape[1] * 16 + 3), device=dev(), generator=g)
    sums[6] = (3 * sums[6]).floor()
    missing = ((s.table < 0) | (s.table >= s.k.shape[0])).repeat_interleave(16, 1)
    sums[:, :, :missing.shape[1]].masked_fill_(missing[:, None], 2.0 if largest else 0.0)
    _check(s, sums, budget, first, last, in_place=largest)


@pytest.mark.parametrize("seed", range(40))
def test_random_tables_with_holes(hip_lib, seed):
    rng = random.Random(seed)
    cache, q = rng.choice(((BF16, BF16), (F16, F16), (FP8, BF16)))
    ps = rng.choice((1, 3, 8, 16, 24, 64))
    longest = rng.choice((90, 500, 2500, 9000))
    lens = [rng.choice((0, 1, longest, rng.randint(1, longest), rng.randint(1, longest))) for _ in range(rng.choice((1, 4, 9)))]
    lens[rng.randrange(len(lens))] = longest
    s = Setup(lens, rng.choice((1, 2, 3)), 1, 16 * rng.randint(1, 8), ps, cache=cache, q=q, seed=seed,
              layout=rng.choice(("heads", "tokens")),
              width=rng.choice((None, 32800 // ps + 1)) if longest < 9000 else None)
    budget = rng.randint(1, max(1, longest // 2))
    first = rng.randint(0, min(budget, 20))
    last = rng.randint(0, min(budget - first, 20))
    g = torch.Generator().manual_seed(seed)
    gone = torch.rand(s.table.shape, generator=g) < rng.choice((0.02, 0.3, 0.9))
    gone[:, :-(-budget // ps)] &= torch.rand((len(lens), 1), generator=g) < 0.2        # mostly out of the way
    for b, n in enumerate(lens):
        if rng.random() < 0.7:
            gone[b, max(0, n - last) // ps:] = False
    s.table[gone.to(dev())] = rng.choice((-1, s.k.shape[0], 2 ** 31 - 1, -2 ** 31))
    sums = torch.rand((s.B, s.Hkv, s.table.shape[1] * ps + rng.randint(0, 5)), generator=g).to(dev())
    if rng.random() < 0.4:
        sums = (3 * sums).floor()
    _check(s, sums, budget, first, last, in_place=rng.random() < 0.5)


def test_the_attention_behind_an_eviction_counts_no_stale_row(hip_lib):
    """Evict, go on from the new lengths, attend: what is seen are the rows that were kept."""
    s = Setup([400, 400, 400], 1, 2, 64, 16, seed=31)
    s.table[0, 10] = s.table[1, 2] = s.table[2, 24] = -1
    sums = torch.rand((3, 1, 400), device=dev())
    sums[0, 0, 160:176] = 9.0
    rows = [c[s.table[0].long()[kept_page], 0, kept_slot] for c in (s.k, s.v) for kept_page, kept_slot in
            [(torch.arange(400, device=dev()) // 16, torch.arange(400, device=dev()) % 16)]]
    new_lens, kept = kv.kv_cache_evict(s.k, s.v, s.table, s.lens, sums, 100, keep_first=4, keep_last=16)
    assert new_lens.tolist() == [100, 400, 400]
    assert not set(kept[0, 0].tolist()) & set(range(160, 176))
    s.lens = new_lens
    out, _, _ = s.check()
    k, v = (r[kept[0, 0].long()].double() for r in rows)
    p = torch.softmax(s.q[0].double() @ k.T * s.scale, 1)
    assert float((out[0].double() - p @ v).abs().max()) < 0.02
