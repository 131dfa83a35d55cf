"""The key-value cache operators by their definitions, in 64 bits on the CPU, one sequence and one head
at a time, and the error bounds that the kernels' arithmetic allows.  Test infrastructure."""
from __future__ import annotations

import math

import numpy as np
import torch


def host(t):
    """A tensor's values in float64 (8-bit codes as the numbers they stand for)."""
    return None if t is None else t.detach().cpu().to(torch.float32).double()


def positions(table_row, n, page_size, num_pages):
    """(page, slot, is there a page) of positions 0 .. n - 1."""
    j = np.arange(n)
    page = np.asarray(table_row)[j // page_size]
    return np.where((page >= 0) & (page < num_pages), page, 0), j % page_size, (page >= 0) & (page < num_pages)


def attention(q, k_cache, v_cache, table, lens, *, scale, window=0, softcap=0.0, sinks=None, k_scale=None,
              v_scale=None, max_len=None):
    """(out, lse, weights added per position [B, Hkv, positions], bounds): `bounds` has, of out, lse and
    the weights, what the kernel's arithmetic may be off before the result is rounded.

    A score is a sum of D products in 32 bits (error D 2^-24 of the products' magnitudes, twice for
    the order of the sum inside the matrix instruction), scaled and made a power of two's exponent
    (2^-22 of its size); the softcap's own evaluation adds 2^-20 of the cap.  Its exponential carries
    that error over as a relative one.  The weights enter the second product as two 16-bit terms:
    2^-17 of a weight, and at least 2^-25 of the largest in fp16.  Sums of n terms in 32 bits:
    sqrt(n) 2^-23 covers random signs with a margin of two; n 2^-24 is not needed."""
    q, k_cache, v_cache = host(q), host(k_cache), host(v_cache)
    B, Hq, D = q.shape
    pages, Hkv, ps, _ = k_cache.shape
    G = Hq // Hkv
    table, lens = table.cpu().numpy(), lens.cpu().numpy()
    width = table.shape[1] * ps
    out = torch.zeros(B, Hq, D, dtype=torch.float64)
    lse = torch.full((B, Hq), -math.inf, dtype=torch.float64)
    added = torch.zeros(B, Hkv, width, dtype=torch.float64)
    out_tol, lse_tol, added_tol = torch.zeros_like(out), torch.zeros_like(lse), torch.zeros_like(added)
    for b in range(B):
        n = min(max(int(lens[b]), 0), width if max_len is None else max_len)
        page, slot, there = positions(table[b], n, ps, pages)
        seen = there & (np.arange(n) >= (max(0, n - window) if window > 0 else 0))
        at = np.nonzero(seen)[0]
        for h in range(Hq):
            g = h // G
            k, v = k_cache[page[at], g, slot[at]], v_cache[page[at], g, slot[at]]
            ks = 1.0 if k_scale is None else float(k_scale[g])
            vs = 1.0 if v_scale is None else float(v_scale[g])
            s = scale * ks * (k @ q[b, h])
            err = D * 2.0 ** -23 * abs(scale) * ks * (k.abs() @ q[b, h].abs()) + 2.0 ** -22 * s.abs()
            if softcap > 0:
                s = softcap * torch.tanh(s / softcap)
                err = err + 2.0 ** -20 * softcap
            sink = None if sinks is None else float(sinks[h])
            everything = s if sink is None else torch.cat([s, torch.tensor([sink], dtype=torch.float64)])
            if everything.numel() == 0 or bool((everything == -math.inf).all()):
                continue
            top = everything.max()
            e = torch.exp(s - top)
            z = torch.exp(everything - top).sum()
            lse[b, h] = top + torch.log(z)
            p = e / z
            out[b, h] = vs * (p[:, None] * v).sum(0)
            added[b, g, at] += p
            off = float(err.max()) if err.numel() else 0.0
            off = 2 * off + 2.0 ** -17 + 2.0 ** -22 * (1 + math.sqrt(len(at))) + 2.0 ** -21 * float(top.abs())
            out_tol[b, h] = off * vs * (p[:, None] * v.abs()).sum(0) + \
                2.0 ** -25 * math.sqrt(len(at) + 1) * vs * (v.abs().amax(0) if len(at) else 0.0)
            lse_tol[b, h] = off + 2.0 ** -22 * (1 + abs(float(lse[b, h])))
            added_tol[b, g, at] += 2 * off * p + 2.0 ** -30
    return out, lse, added, (out_tol, lse_tol, added_tol)


def assert_attention(got, lse, want, dtype, what=""):
    """`got` within half a unit in the last place of its type of a value within the bound."""
    ref, ref_lse, _, (out_tol, lse_tol, _) = want
    # 8 and 11 significant bits: the last one is 2^-7 and 2^-10 of the power of two below the value
    unit = 2.0 ** -7 if dtype == torch.bfloat16 else 2.0 ** -10
    small = 2.0 ** -133 if dtype == torch.bfloat16 else 2.0 ** -24      # the least subnormal
    got = host(got)
    finite = torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), f"{what}: NaN elsewhere than in the definition"
    excess = ((got - ref).abs() - (unit / 2 * 1.01) * (ref.abs() + out_tol) - out_tol - small)[finite]
    assert excess.numel() == 0 or float(excess.max()) <= 0, f"{what}: out is {float(excess.max()):.3g} beyond its bound"
    if lse is not None:
        lse = host(lse)
        fine = torch.isfinite(ref_lse)
        assert torch.equal(lse[~fine & ~torch.isnan(ref_lse)], ref_lse[~fine & ~torch.isnan(ref_lse)]), what
        assert torch.equal(torch.isnan(lse), torch.isnan(ref_lse)), what
        off = ((lse - ref_lse).abs() - lse_tol)[fine]
        assert off.numel() == 0 or float(off.max()) <= 0, f"{what}: lse is {float(off.max()):.3g} beyond its bound"


def assert_sums(got, before, want, what=""):
    """The sums grew by the weights; each addition rounds once to 32 bits."""
    _, _, added, (_, _, tol) = want
    before, got = host(before), host(got)
    n = added.shape[2]
    assert torch.equal(got[:, :, n:], before[:, :, n:]), f"{what}: sums beyond the table changed"
    off = (got[:, :, :n] - before[:, :, :n] - added).abs() - tol - 2.0 ** -24 * (before[:, :, :n].abs() + added)
    assert float(off.max()) <= 0, f"{what}: the sums are {float(off.max()):.3g} beyond their bound"


def append(k_cache, v_cache, k, v, table, lens, starts, k_scale, v_scale):
    """The caches after the append, as tensors of the caches' type on the CPU."""
    caches = [k_cache.detach().cpu().clone(), v_cache.detach().cpu().clone()]
    pages, _, ps, _ = caches[0].shape
    table, lens = table.cpu().numpy(), lens.cpu().numpy()
    for b in range(len(lens)):
        first, last = (b, b + 1) if starts is None else (int(starts[b]), int(starts[b + 1]))
        for t in range(first, last):
            pos = int(lens[b]) - (last - t)
            if pos < 0 or pos // ps >= table.shape[1] or not 0 <= table[b, pos // ps] < pages:
                continue
            for cache, rows, scale in ((caches[0], k, k_scale), (caches[1], v, v_scale)):
                row = rows[t].cpu()
                if scale is not None:
                    # (a quotient of 32-bit numbers, rounded once to 32 bits and once to the codes)
                    row = (row.float() / scale.cpu()[:, None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
                    cache.view(torch.uint8)[table[b, pos // ps], :, pos % ps] = row.view(torch.uint8)
                else:
                    cache[table[b, pos // ps], :, pos % ps] = row
    return caches


def evict(k_cache, v_cache, table, lens, sums, sums_out, budget, first, last):
    """(k_cache, v_cache, sums_out, new_lens, kept) after the eviction, on the CPU."""
    caches = [c.detach().cpu().clone() for c in (k_cache, v_cache)]
    bytes_of = [c.view(torch.uint8) if c.element_size() == 1 else c for c in caches]
    _, Hkv, ps, _ = caches[0].shape
    table, lens, sums = table.cpu().numpy(), lens.cpu().numpy(), sums.detach().cpu().numpy()
    out = sums_out.detach().cpu().clone()
    kept = np.full((len(lens), Hkv, budget), -1, dtype=np.int32)
    for b, n in enumerate(int(x) for x in lens):
        for h in range(Hkv):
            if n <= budget:
                kept[b, h, :n] = np.arange(n)
                out[b, h, :n] = torch.from_numpy(sums[b, h, :n].copy())
                continue
            key = sums[b, h, first:n - last].astype(np.float64)
            key = np.where(np.isnan(key), np.inf, key), np.isnan(key)      # NaN above infinity
            order = np.lexsort((np.arange(len(key[0])), -key[0], ~key[1]))
            best = order[:budget - first - last] + first
            at = np.sort(np.concatenate([np.arange(first), best, np.arange(n - last, n)]))
            kept[b, h] = at
            j = np.arange(budget)
            for c in bytes_of:
                c[table[b, j // ps], h, j % ps] = c[table[b, at // ps], h, at % ps].clone()
            out[b, h, :n] = 0.0
            out[b, h, :budget] = torch.from_numpy(sums[b, h, at].copy())
    return caches[0], caches[1], out, np.minimum(lens, budget), kept
