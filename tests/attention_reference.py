"""Attention of a sequence's last tokens over its paged cache by its definition, in 64 bits on the CPU, with what
the kernels' arithmetic may be off.  Test infrastructure."""
from __future__ import annotations

import math

import torch

import kv_blocks_reference as blocks
import kv_reference as kvref


def cache_values(cache, scale):
    """[pages, Hkv, page_size, D] in 64 bits; scale None, [Hkv] or [pages, Hkv, blocks]."""
    if scale is None:
        return kvref.host(cache)
    if scale.dim() == 1:
        return kvref.host(cache) * kvref.host(scale)[:, None, None]
    return blocks.values(cache, scale)


def attention(q, k_cache, v_cache, table, lens, starts=None, *, scale, window=0, keep_first=0, softcap=0.0, sinks=None,
              k_scale=None, v_scale=None, max_len=None, weight_bits=16):
    """(out, lse, weights added per position, (bounds of the three)) of q [tokens, Hq, D]; starts None: one token
    for each sequence.  Rows that belong to no sequence are NaN.

    The bounds: a score is a sum of D products in 32 bits (D 2^-23 of the products' magnitudes), scaled and made a
    power of two's exponent, times a block's scale where there is one (2^-21 of its size); the cap's own
    evaluation 2^-20 of the cap.  Its exponential carries that over as a relative error, and the reference that it
    is taken against 2^-21 of its size.  A weight enters the second product with weight_bits significant bits: half a
    step is 2^-weight_bits of it (16: two 16-bit terms, off by 2^-17 and so inside); in fp16 at least 2^-24 / 2^15 of
    the largest, times at most 2^8 of slack, in front of the sums.  Sums of n terms in 32 bits: sqrt(n) 2^-23
    covers random signs with a margin of two, in the products of a value scale 2^-23 more."""
    q = kvref.host(q)
    k_values, v_values = cache_values(k_cache, k_scale), cache_values(v_cache, v_scale)
    tokens, Hq, D = q.shape
    pages, Hkv, ps, _ = k_values.shape
    G = Hq // Hkv
    table, lens = table.cpu().numpy(), lens.cpu().tolist()
    starts = list(range(len(lens) + 1)) if starts is None else starts.cpu().tolist()
    width = table.shape[1] * ps
    nan = math.nan
    out, lse = torch.full((tokens, Hq, D), nan, dtype=torch.float64), torch.full((tokens, Hq), nan, dtype=torch.float64)
    out_tol, lse_tol = torch.zeros_like(out), torch.zeros_like(lse)
    added = torch.zeros(len(lens), Hkv, width, dtype=torch.float64)
    added_tol = torch.zeros_like(added)
    for b, length in enumerate(lens):
        n = starts[b + 1] - starts[b]
        if n <= 0:
            continue
        length = min(max(int(length), 0), width if max_len is None else max_len)
        page, slot, there = kvref.positions(table[b], length, ps, pages)
        rows = slice(starts[b], starts[b + 1])
        place = torch.arange(length - n, length)[:, None]
        at = torch.arange(length)[None]
        seen = (at <= place) & torch.from_numpy(there)[None]
        if window > 0:
            seen &= (at > place - window) | (at < keep_first)
        for h in range(Hq):
            g = h // G
            k, v = k_values[page, g, slot], v_values[page, g, slot]
            # (what is hidden from every row may be anything)
            anyone = seen.any(0)
            k, v = torch.where(anyone[:, None], k, 0.0), torch.where(anyone[:, None], v, 0.0)
            s = scale * (q[rows, h] @ k.t())
            err = D * 2.0 ** -23 * abs(scale) * (q[rows, h].abs() @ k.abs().t()) + 2.0 ** -21 * s.abs()
            if softcap > 0:
                s = softcap * torch.tanh(s / softcap)
                err = err + 2.0 ** -20 * softcap
            s = torch.where(seen, s, -math.inf)
            extra = torch.full((n, 1), -math.inf, dtype=torch.float64) if sinks is None else \
                torch.full((n, 1), float(sinks[h]), dtype=torch.float64)
            everything = torch.cat([s, extra], 1)
            top = everything.amax(1, keepdim=True)
            ref = torch.where(torch.isinf(top) & (top < 0), 0.0, top)
            e = torch.where(seen, torch.exp(s - ref), 0.0)
            z = torch.exp(everything - ref).sum(1, keepdim=True)
            p = torch.where(z > 0, e / z, 0.0)
            lse[rows, h] = (ref + torch.log(z))[:, 0]
            out[rows, h] = p @ v
            off = torch.where(seen, err, 0.0).amax(1, keepdim=True) if length else torch.zeros(n, 1, dtype=torch.float64)
            count = math.sqrt(length + 1)
            off = 2 * off + 2.0 ** -22 * (1 + count) + 2.0 ** -21 * ref.abs()
            weight = off + 2.0 ** -weight_bits + 2.0 ** -22
            out_tol[rows, h] = weight * (p @ v.abs()) + 2.0 ** -25 * count * (v.abs().amax(0) if length else 0.0)
            lse_tol[rows, h] = off[:, 0] + 2.0 ** -22 * (1 + torch.where(torch.isinf(lse[rows, h]), 0.0, lse[rows, h].abs()))
            if n == 1:
                added[b, g, :length] += p[0]
                added_tol[b, g, :length] += 2 * (off[0] + 2.0 ** -17) * p[0] + 2.0 ** -30
    return out, lse, added, (out_tol, lse_tol, added_tol)
