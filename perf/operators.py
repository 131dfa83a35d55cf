"""The key-value cache operators whose speed counts: append, the attention of one new token over the
paged cache, and eviction by accumulated attention weight, as a serving program's decode step runs
them next to the MoE layer.

Twelve listed cases and, through draw(), any other of the same ranges.  A case is

  op        "attend"  paged_attention: one new token a sequence over its cached positions
            "append"  kv_cache_append: new tokens' keys and values into the pages
            "step"    a decode step: append of one token a sequence, then the attention, counted
            "evict"   kv_cache_evict: the cache compacted to its positions of most weight
  B         sequences
  longest   positions of the longest sequence (after the append); the others are ragged below it
  Hkv, G, D key/value heads, query heads on each of them, width of a head
  ps        positions in a page
  kind      "bf16", "fp16", or "fp8": E4M3 codes with a scale for each head, queries in bf16
  layout    "heads" [pages, heads, positions, D] in memory or "tokens" [pages, positions, heads, D]
  window    attention to the last positions alone (0: all)
  softcap   scores bounded by softcap * tanh(s / softcap) (0: not)
  sinks     a learned logit per head in the softmax's sum
  counted   the weights every position received are added up ("attend"; "step" always)
  tokens    new tokens of the call ("append"; 0: one a sequence)
  budget    positions kept of each sequence ("evict"), an eighth of them the latest, four the first
"""
from __future__ import annotations

import math
import random

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp8": torch.bfloat16}


def _case(op, B, longest, heads, ps, *, kind="bf16", layout="heads", window=0, softcap=0.0, sinks=False,
          counted=False, tokens=0, budget=0, name=None):
    Hkv, G, D = heads
    case = dict(op=op, B=B, longest=longest, Hkv=Hkv, G=G, D=D, ps=ps, kind=kind, layout=layout, window=window,
                softcap=softcap, sinks=sinks, counted=counted, tokens=tokens, budget=budget)
    return case if name is None else dict(case, name=name)


def listed():
    narrow, wide = (8, 8, 64), (8, 4, 128)
    return [
        # one user's next token soon after the prompt: latency, launches, the host's work per call
        _case("attend", 1, 200, narrow, 16, sinks=True, name="attend_one_short"),
        # a decode batch in a layer with a sliding window: little to read, many sequences
        _case("attend", 64, 8192, narrow, 16, window=128, sinks=True, name="attend_window"),
        # the same batch in a layer that sees everything, the cache token by token in memory
        _case("attend", 64, 8192, narrow, 16, sinks=True, layout="tokens", name="attend_batch"),
        # one user with a very long context: all of the card on eight heads of one sequence
        _case("attend", 1, 131071, wide, 64, name="attend_one_long"),
        # a large batch on an 8-bit cache, the most memory a step reads
        _case("attend", 255, 8192, wide, 32, kind="fp8", name="attend_fp8"),
        # no shared heads, an odd head width, pages that are no power of two, capped scores
        _case("attend", 33, 3000, (20, 1, 80), 24, kind="fp16", softcap=30.0, name="attend_odd"),
        # what each position received is added up for a later eviction
        _case("attend", 64, 16384, wide, 16, counted=True, name="attend_counted"),
        # the cache's part of a decode step: the new token in, then the attention, counted
        _case("step", 32, 2048, narrow, 16, sinks=True, name="step_counted"),
        # a decode batch's new tokens into an 8-bit cache: latency
        _case("append", 255, 1024, wide, 32, kind="fp8", name="append_tokens"),
        # ragged pieces of prompts
        _case("append", 16, 2048, wide, 16, tokens=8191, name="append_prompts"),
        # the cache of a decode batch back to its budget after 256 steps
        _case("evict", 64, 2304, wide, 16, budget=2048, name="evict_steps"),
        # long prompts cut to their budget before decoding begins
        _case("evict", 4, 65536, wide, 16, budget=8192, name="evict_prompts"),
    ]


_MOST = 64 * 16384 * 8 * 128 * 2 * 2        # bytes of keys and values of the largest listed case


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """Batches and lengths spread over their logarithms, on head layouts beside the listed ones."""
    op = rng.choice(("attend",) * 6 + ("step", "step", "append", "append", "evict", "evict"))
    kind = rng.choice(("bf16", "bf16", "fp16", "fp8"))
    D = rng.choice((64, 64, 80, 96, 128, 128, 192, 256))
    Hkv, G = rng.choice((1, 2, 4, 8, 8, 16, 32)), rng.choice((1, 2, 3, 4, 5, 7, 8, 8, 12, 16, 24))
    ps = rng.choice((8, 16, 16, 24, 32, 48, 64, 128))
    B = _log_int(rng, 1, 256)
    # (half of the largest listed case's cache at most, and of its queries' scores)
    most = min(_MOST // 2 // (B * Hkv * D * 4), (1 << 28) // (B * Hkv * G), 131072)
    longest = _log_int(rng, 1, max(1, most))
    if op == "evict":
        longest = min(max(longest, 64), 65536)
        B = max(1, min(B, _MOST // 2 // (longest * Hkv * D * 4), (1 << 24) // (longest * Hkv)))
    tokens = 0
    if op == "append" and rng.random() < 0.6:
        tokens = _log_int(rng, 1, max(1, min(16384, B * longest // 2)))
    return _case(op, B, longest, (Hkv, G, D), ps, kind=kind, layout=rng.choice(("heads", "tokens")),
                 window=_log_int(rng, 1, longest) if op == "attend" and rng.random() < 0.25 else 0,
                 softcap=rng.choice((0.0, 0.0, 0.0, 20.0, 50.0)) if op in ("attend", "step") else 0.0,
                 sinks=op in ("attend", "step") and rng.random() < 0.4,
                 counted=op == "attend" and rng.random() < 0.3, tokens=tokens,
                 budget=_log_int(rng, 32, longest - 8) if op == "evict" else 0)


# ---- inputs ------------------------------------------------------------------------------------

def _lengths(case):
    """The sequences' lengths: the first the longest, the others down to an eighth of it, and in a
    batch of the attention one that is empty (a row of a padded batch); a cache that is evicted from
    is near one length (a decode batch's) or ragged (prompts)."""
    rng = random.Random(case["B"] * 131 + case["longest"])
    B, longest = case["B"], case["longest"]
    low = longest - min(16, longest // 8) if case["op"] == "evict" and longest <= 4096 else max(1, longest // 8)
    lens = [longest] + [rng.randint(low, longest) for _ in range(B - 1)]
    if case["op"] == "attend" and B >= 8:
        lens[3] = 0
    return lens


def _new_tokens(case):
    """New tokens of every sequence: one, or `tokens` spread raggedly, none longer than its sequence."""
    lens = _lengths(case)
    if not case["tokens"]:
        return [1] * len(lens)
    rng = random.Random(case["tokens"])
    share = [rng.random() + 0.1 for _ in lens]
    new = [min(n, int(case["tokens"] * s / sum(share))) for n, s in zip(lens, share)]
    short = case["tokens"] - sum(new)
    for i, n in enumerate(lens):
        more = min(short, n - new[i])
        new[i] += more
        short -= more
    return new


def _cache(case, pages, gen, dev):
    Hkv, D, ps = case["Hkv"], case["D"], case["ps"]
    order = (pages, Hkv, ps, D) if case["layout"] == "heads" else (pages, ps, Hkv, D)
    c = torch.randn(order, device=dev, generator=gen, dtype=_TYPES[case["kind"]])
    if case["kind"] == "fp8":
        c = (c * 64).to(torch.float8_e4m3fn)
    return c if case["layout"] == "heads" else c.transpose(1, 2)


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    B, Hkv, G, D, ps = (case[n] for n in ("B", "Hkv", "G", "D", "ps"))
    lens = _lengths(case)
    width = -(-case["longest"] // ps)
    need = torch.tensor([-(-n // ps) for n in lens], device=dev)
    pages = int(sum(-(-n // ps) for n in lens)) + 3
    # every sequence's pages, scattered over the cache as a server's are; -1 where it has none
    at = torch.arange(width, device=dev)[None, :]
    taken = (need.cumsum(0) - need)[:, None] + at
    shuffled = torch.randperm(pages, device=dev, generator=gen)
    table = torch.where(at < need[:, None], shuffled[taken.clamp(max=pages - 1)], -1).to(torch.int32)
    t = _TYPES[case["kind"]]
    state = dict(case=case, table=table, lens=torch.tensor(lens, dtype=torch.int32, device=dev),
                 k_cache=_cache(case, pages, gen, dev), v_cache=_cache(case, pages, gen, dev),
                 k_scale=None, v_scale=None, sinks=None, sums=None, starts=None)
    if case["kind"] == "fp8":
        state["k_scale"] = (torch.rand(Hkv, device=dev, generator=gen) + 0.5) / 64
        state["v_scale"] = (torch.rand(Hkv, device=dev, generator=gen) + 0.5) / 64
    if case["op"] in ("attend", "step"):
        # queries of 2.5 times the keys' size: a few positions take most of the weight
        state["q"] = (2.5 * torch.randn((B, Hkv * G, D), device=dev, generator=gen)).to(t)
        if case["sinks"]:
            state["sinks"] = torch.randn(Hkv * G, device=dev, generator=gen)
        if case["counted"] or case["op"] == "step":
            # what some ten steps before gave
            state["sums"] = 10 * G / case["longest"] * torch.rand((B, Hkv, width * ps), device=dev, generator=gen)
    if case["op"] in ("append", "step"):
        new = _new_tokens(case)
        state["k_new"] = torch.randn((sum(new), Hkv, D), device=dev, generator=gen).to(t)
        state["v_new"] = torch.randn((sum(new), Hkv, D), device=dev, generator=gen).to(t)
        if case["tokens"]:
            starts = [0]
            for n in new:
                starts.append(starts[-1] + n)
            state["starts"] = torch.tensor(starts, dtype=torch.int32, device=dev)
    if case["op"] == "evict":
        # sums of softmax weights: many small ones, a few large ones
        state["sums"] = torch.exp(2.0 * torch.randn((B, Hkv, width * ps), device=dev, generator=gen) - 3.0)
        state["sums_out"] = torch.zeros_like(state["sums"])
    return state


def _kept_ends(case):
    return min(4, case["budget"] // 8), case["budget"] // 8


# ---- one pass -----------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    if case["op"] == "evict":
        return (_run_evict if own else _plain_evict)(state)
    out = {}
    if case["op"] in ("append", "step"):
        (_run_append if own else _plain_append)(state)
        out = {"k_cache": state["k_cache"], "v_cache": state["v_cache"]}
    if case["op"] in ("attend", "step"):
        out["out"], out["lse"] = (_run_attend if own else _plain_attend)(state)
        if state["sums"] is not None:
            out["sums"] = state["sums"]
    return out


def _run_append(s):
    from vkernels_amd import kv_cache
    kv_cache.kv_cache_append(s["k_new"], s["v_new"], s["k_cache"], s["v_cache"], s["table"], s["lens"],
                             query_start=s["starts"], k_scale=s["k_scale"], v_scale=s["v_scale"])


def _run_attend(s):
    from vkernels_amd import kv_cache
    case = s["case"]
    return kv_cache.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"],
                                    max_len=case["longest"], window=case["window"], softcap=case["softcap"],
                                    sinks=s["sinks"], k_scale=s["k_scale"], v_scale=s["v_scale"],
                                    weight_sums=s["sums"], return_lse=True)


def _run_evict(s):
    from vkernels_amd import kv_cache
    case = s["case"]
    first, last = _kept_ends(case)
    new_lens, kept = kv_cache.kv_cache_evict(s["k_cache"], s["v_cache"], s["table"], s["lens"], s["sums"],
                                             case["budget"], keep_first=first, keep_last=last,
                                             max_len=case["longest"], sums_out=s["sums_out"])
    return {"k_cache": s["k_cache"], "v_cache": s["v_cache"], "sums": s["sums_out"], "lens": new_lens, "kept": kept}


# ---- the same in elementary operations, in 32 bits -------------------------------------------------

def _plain_append(s):
    case = s["case"]
    new, ps = s["k_new"], case["ps"]
    t = torch.arange(new.shape[0], device=new.device)
    if s["starts"] is None:
        seq, place = t, s["lens"].long() - 1
    else:
        starts, lens = s["starts"].long(), s["lens"].long()
        seq = torch.searchsorted(starts, t, right=True) - 1
        place = lens[seq] - starts[seq + 1] + t
    page, slot = s["table"][seq, place // ps].long(), place % ps
    _plain_store(s["k_cache"], s["k_new"], s["k_scale"], page, slot)
    _plain_store(s["v_cache"], s["v_new"], s["v_scale"], page, slot)


def _plain_store(cache, rows, scale, page, slot):
    if scale is None:
        cache[page, :, slot] = rows
    else:
        codes = (rows.float() / scale[:, None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
        cache.view(torch.uint8)[page, :, slot] = codes.view(torch.uint8)


def _plain_rows(cache, table):
    """[B, Hkv, positions, D] in 32 bits of every sequence's pages."""
    pages = table.long().clamp(min=0)
    rows = cache.view(torch.uint8)[pages].view(cache.dtype) if cache.dtype == torch.float8_e4m3fn else cache[pages]
    B, W, Hkv, ps, D = rows.shape
    return rows.transpose(1, 2).float().reshape(B, Hkv, W * ps, D)


def _plain_attend(s):
    case = s["case"]
    B, Hkv, G, D, ps = (case[n] for n in ("B", "Hkv", "G", "D", "ps"))
    k = _plain_rows(s["k_cache"], s["table"])
    score = s["q"].float().view(B, Hkv, G, D) @ k.transpose(2, 3)
    del k
    score *= D ** -0.5
    if s["k_scale"] is not None:
        score *= s["k_scale"].view(1, Hkv, 1, 1)
    if case["softcap"]:
        score = case["softcap"] * torch.tanh(score / case["softcap"])
    n = s["lens"].view(B, 1).long()
    at = torch.arange(score.shape[3], device=score.device).view(1, -1)
    seen = (at < n) & (s["table"].repeat_interleave(ps, 1) >= 0)
    if case["window"]:
        seen &= at >= n - case["window"]
    score.masked_fill_(~seen.view(B, 1, 1, -1), float("-inf"))
    top = score.amax(3)
    sinks = None if s["sinks"] is None else s["sinks"].view(1, Hkv, G)
    if sinks is not None:
        top = torch.maximum(top, sinks)
    top = torch.where(torch.isinf(top) & (top < 0), 0.0, top)
    weight = torch.exp(score - top[..., None])
    del score
    total = weight.sum(3)
    if sinks is not None:
        total = total + torch.exp(sinks - top)
    lse = torch.log(total) + top
    weight /= torch.where(total == 0, 1.0, total)[..., None]
    v = _plain_rows(s["v_cache"], s["table"])
    out = weight @ v
    if s["v_scale"] is not None:
        out *= s["v_scale"].view(1, Hkv, 1, 1)
    if s["sums"] is not None:
        s["sums"] += weight.sum(2)
    return out.view(B, Hkv * G, D).to(s["q"].dtype), lse.view(B, Hkv * G)


def _plain_evict(s):
    case = s["case"]
    B, Hkv, ps, budget = (case[n] for n in ("B", "Hkv", "ps", "budget"))
    first, last = _kept_ends(case)
    n = s["lens"].view(B, 1, 1).long()
    at = torch.arange(s["sums"].shape[2], device=n.device).view(1, 1, -1)
    always = (n <= budget) | (at < first) | (at >= n - last)
    order = torch.where(always, float("inf"), s["sums"]).masked_fill(at >= n, float("-inf"))
    kept = order.argsort(dim=2, descending=True, stable=True)[:, :, :budget]
    new_n = n.clamp(max=budget)
    beyond = s["sums"].shape[2]
    kept = torch.where(torch.arange(kept.shape[2], device=n.device) < new_n, kept, beyond).sort(dim=2).values
    b, h, j = torch.nonzero(kept < beyond, as_tuple=True)
    src = kept[b, h, j]
    table = s["table"].long()
    for_cache = (table[b, j // ps], h, j % ps), (table[b, src // ps], h, src % ps)
    _plain_move(s["k_cache"], *for_cache)
    _plain_move(s["v_cache"], *for_cache)
    sums = torch.where(at < n, 0.0, s["sums_out"])
    sums[b, h, j] = s["sums"][b, h, src]
    s["sums_out"].copy_(sums)
    kept = torch.nn.functional.pad(kept, (0, budget - kept.shape[2]), value=beyond)
    return {"k_cache": s["k_cache"], "v_cache": s["v_cache"], "sums": s["sums_out"],
            "lens": new_n.view(B).to(torch.int32), "kept": torch.where(kept < beyond, kept, -1).to(torch.int32)}


def _plain_move(cache, to, source):
    cache = cache.view(torch.uint8) if cache.dtype == torch.float8_e4m3fn else cache
    cache[to] = cache[source]


# ---- the definition, in 64 bits ------------------------------------------------------------------

def _exact_positions(state, b, n):
    """(pages, slots) of the first n positions of sequence b."""
    ps = state["case"]["ps"]
    j = torch.arange(n, device=state["table"].device)
    return state["table"][b].long()[j // ps], j % ps


def _exact_rows(cache, pages, slots):
    """[n, Hkv, D] of these positions."""
    if cache.dtype == torch.float8_e4m3fn:
        return cache.view(torch.uint8)[pages, :, slots].view(torch.float8_e4m3fn).double()
    return cache[pages, :, slots].double()


def _exact_append(s, caches):
    case = s["case"]
    done = 0
    for b, (n, new) in enumerate(zip(_lengths(case), _new_tokens(case))):
        pages, slots = _exact_positions(s, b, n)
        for cache, rows, scale in ((caches[0], s["k_new"], s["k_scale"]), (caches[1], s["v_new"], s["v_scale"])):
            rows = rows[done:done + new].double()
            if scale is not None:
                # the codes nearest to the quotient that 32 bits hold: that division and the
                # rounding to 8 bits are the operator's own
                rows = (rows.float() / scale[:, None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).double()
            if new:
                cache[pages[n - new:], :, slots[n - new:]] = rows
        done += new


def _exact_attend(s, caches):
    case = s["case"]
    Hkv, G, D = case["Hkv"], case["G"], case["D"]
    outs, lses = [], []
    sums = None if s["sums"] is None else s["sums"].double()
    for b, n in enumerate(_lengths(case)):
        start = max(0, n - case["window"]) if case["window"] else 0
        pages, slots = (x[start:] for x in _exact_positions(s, b, n))
        k, v = (_exact_rows(c, pages, slots).permute(1, 0, 2) for c in caches)
        if s["k_scale"] is not None:
            k, v = k * s["k_scale"].double().view(-1, 1, 1), v * s["v_scale"].double().view(-1, 1, 1)
        q = s["q"][b].double().view(Hkv, G, D) / math.sqrt(D)
        score = torch.matmul(q, k.transpose(1, 2).contiguous())
        if case["softcap"]:
            score = torch.tanh(score / case["softcap"]) * case["softcap"]
        extra = score.new_full((Hkv, G, 1), float("-inf")) if s["sinks"] is None else \
            s["sinks"].double().view(Hkv, G, 1)
        lse = torch.logsumexp(torch.cat([score, extra], 2), 2)
        share = torch.exp(score - torch.where(torch.isinf(lse), 0.0, lse)[..., None])
        outs.append(torch.matmul(share, v.contiguous()).reshape(Hkv * G, D))
        lses.append(lse.reshape(Hkv * G))
        if sums is not None:
            sums[b, :, start:n] += share.sum(1)
    got = {"out": torch.stack(outs), "lse": torch.stack(lses)}
    return got if sums is None else dict(got, sums=sums)


def _exact_evict(s):
    case = s["case"]
    budget, ps = case["budget"], case["ps"]
    first, last = _kept_ends(case)
    caches = [s["k_cache"].double(), s["v_cache"].double()]
    sums, kept = s["sums_out"].double(), torch.full((case["B"], case["Hkv"], budget), -1, dtype=torch.int32,
                                                    device=s["sums"].device)
    lens = _lengths(case)
    for b, n in enumerate(lens):
        m = min(n, budget)
        own_sums = s["sums"][b, :, :n].double()
        if n <= budget:
            sums[b, :, :n] = own_sums
            kept[b, :, :n] = torch.arange(n, dtype=torch.int32, device=sums.device)
            continue
        middle = own_sums[:, first:n - last]
        best = torch.sort(middle, dim=1, descending=True, stable=True).indices[:, :budget - first - last] + first
        ends = torch.cat([torch.arange(first), torch.arange(n - last, n)]).to(best)
        at = torch.cat([best, ends.expand(case["Hkv"], -1)], 1).sort(1).values
        heads = torch.arange(case["Hkv"], device=at.device)[:, None].expand_as(at)
        table = s["table"][b].long()
        to = torch.arange(m, device=at.device).expand_as(at)
        for c in caches:
            c[table[to // ps], heads, to % ps] = c[table[at // ps], heads, at % ps]
        sums[b, :, :n] = 0.0
        sums[b, :, :m] = own_sums.gather(1, at)
        kept[b, :, :m] = at.to(torch.int32)
    return {"k_cache": caches[0], "v_cache": caches[1], "sums": sums,
            "lens": torch.tensor([min(n, budget) for n in lens], dtype=torch.int32), "kept": kept}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "evict":
        return _exact_evict(s)
    if case["op"] == "attend":
        return _exact_attend(s, (s["k_cache"], s["v_cache"]))
    caches = [s["k_cache"].double(), s["v_cache"].double()]
    _exact_append(s, caches)
    got = {"k_cache": caches[0], "v_cache": caches[1]}
    return got if case["op"] == "append" else dict(got, **_exact_attend(s, caches))


# ---- what a pass cannot do without -----------------------------------------------------------------

def work(case):
    Hkv, G, D, B = case["Hkv"], case["G"], case["D"], case["B"]
    lens = _lengths(case)
    row = 2 * D * (1 if case["kind"] == "fp8" else 2)       # a position's key and value in one head
    moved, flops = 0, 0
    if case["op"] in ("append", "step"):
        T = sum(_new_tokens(case))
        moved += T * Hkv * (4 * D + row)
        flops += T * Hkv * 2 * D if case["kind"] == "fp8" else 0
    if case["op"] in ("attend", "step"):
        seen = sum(min(n, case["window"]) if case["window"] else n for n in lens)
        moved += seen * Hkv * row + B * Hkv * G * (4 * D + 4)
        if case["counted"] or case["op"] == "step":
            moved += seen * Hkv * 8
        flops += 4 * seen * Hkv * G * D
    if case["op"] == "evict":
        # sums in and out, and of every cut sequence the rows behind the first that goes
        moved += sum(n * Hkv * 8 for n in lens) + B * Hkv * case["budget"] * 4
        moved += sum(2 * row * Hkv * (case["budget"] - _kept_ends(case)[0]) for n in lens if n > case["budget"])
        flops += sum(n * Hkv for n in lens)
    return {"bytes": moved + 4 * B, "flops": flops}
