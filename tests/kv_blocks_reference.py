"""8-bit caches with a scale for each block of positions by their definition: appends on the CPU, position by
position and head by head, and a cache's values in 64 bits.  Test infrastructure."""
from __future__ import annotations

import torch

FP8 = torch.float8_e4m3fn


def _codes(x):
    return x.clamp(-448.0, 448.0).to(FP8)


def append(k_cache, v_cache, k_scale, v_scale, k, v, table, lens, starts):
    """(k_cache, v_cache, k_scale, v_scale) after the append, on the CPU.  Quotients and products are rounded to
    32 bits as the operator's are, so that codes and scales have to be equal bit for bit."""
    caches = [c.detach().cpu().clone() for c in (k_cache, v_cache)]
    scales = [c.detach().cpu().clone() for c in (k_scale, v_scale)]
    pages, Hkv, ps, _ = caches[0].shape
    block = ps // scales[0].shape[2]
    table, lens = table.cpu().numpy(), lens.cpu().numpy()
    starts = None if starts is None else starts.cpu().tolist()
    for b in range(len(lens)):
        first, last = (b, b + 1) if starts is None else (starts[b], starts[b + 1])
        length = int(lens[b])
        at = max(0, length - (last - first))
        while at < length:
            begin = at // block * block
            end = min(begin + block, length)
            if begin // ps < table.shape[1] and 0 <= table[b, begin // ps] < pages:
                page, slot = int(table[b, begin // ps]), begin % ps
                for cache, scale, rows in zip(caches, scales, (k, v)):
                    mine = rows[last - (length - at):last - (length - end)].detach().cpu().float().transpose(0, 1)   # [Hkv, rows, D]
                    size = torch.where(torch.isfinite(mine), mine.abs(), 0.0).amax((1, 2))
                    s = size / 448.0
                    old = scale[page, :, slot // block]
                    if at > begin:
                        grows = ~(old >= s)          # (the old scale counts if it is larger: NaN is not)
                        s = torch.where(grows, s, old)
                        before = cache.view(torch.uint8)[page, :, slot:slot + at - begin].view(FP8).float()
                        again = _codes(before * (old / s)[:, None, None])
                        kept = torch.where(grows[:, None, None], again.view(torch.uint8), _codes(before).view(torch.uint8))
                        cache.view(torch.uint8)[page, :, slot:slot + at - begin] = kept
                    scale[page, :, slot // block] = s
                    by = torch.where(s > 0, s, 1.0)[:, None, None]
                    cache.view(torch.uint8)[page, :, slot + at - begin:slot + end - begin] = _codes(mine / by).view(torch.uint8)
            at = end
    return (*caches, *scales)


def values(cache, scale):
    """[pages, Hkv, page_size, D] in 64 bits."""
    c, s = cache.detach().cpu().float().double(), scale.detach().cpu().double()
    return c * s.repeat_interleave(c.shape[2] // s.shape[2], 2)[..., None]


def read(k_cache, v_cache, k_scale, v_scale, table, lens, starts, tokens):
    """(k, v, does a row belong to a sequence) in 64 bits on the CPU; scales [Hkv], [pages, Hkv, blocks] or None."""
    caches = []
    for c, s in ((k_cache, k_scale), (v_cache, v_scale)):
        if s is None:
            caches.append(c.detach().cpu().double())
        elif s.dim() == 1:
            caches.append(c.detach().cpu().float().double() * s.detach().cpu().double()[:, None, None])
        else:
            caches.append(values(c, s))
    pages, Hkv, ps, D = caches[0].shape
    table, lens = table.cpu().numpy(), lens.cpu().numpy()
    out = [torch.zeros(tokens, Hkv, D, dtype=torch.float64) for _ in range(2)]
    belongs = torch.zeros(tokens, dtype=torch.bool)
    for b in range(len(lens)):
        first, last = (b, b + 1) if starts is None else (int(starts[b]), int(starts[b + 1]))
        for t in range(first, last):
            belongs[t] = True
            pos = int(lens[b]) - (last - t)
            if pos < 0 or pos // ps >= table.shape[1] or not 0 <= table[b, pos // ps] < pages:
                continue
            for o, c in zip(out, caches):
                o[t] = c[table[b, pos // ps], :, pos % ps]
    return (*out, belongs)
