"""Operators of a decoder layer's attention on either side of the paged key-value cache, whose speed
counts: the norm and rotation of queries and keys, keys and values quantised as they are written and
read back, one new token's attention over a cache with a scale for each block of positions, and the
attention of several new tokens at once, over everything or over a window and the first positions.

Twelve listed cases and, through draw(), any other of the same ranges.  A case is

  op        "rotate"  qk_norm_rope: queries' and keys' RMS norm for each head, and their rotation
            "write"   kv_cache_append into a cache of E4M3 codes with a scale for each block
            "read"    kv_cache_read: positions of such a cache as ordinary rows
            "token"   paged_attention: one new token a sequence
            "prompt"  paged_attention with query_start: the new tokens of every sequence
  B         sequences ("rotate": 1)
  longest   positions of the longest sequence, the new tokens counted; the others are ragged below it
  tokens    new tokens of the call, in all ("token", and "write" with 0: one a sequence); rows that are
            read; the last `spare` of them belong to no sequence (a padded batch)
  Hkv, G, D key/value heads, query heads on each of them, width of a head
  ps, block positions in a page, and those that share a scale (0: a 16-bit cache)
  kind      "bf16" or "fp16": queries, new rows, results, and the cache where block is 0
  layout    "heads" [pages, heads, positions, D] in memory or "tokens" [pages, positions, heads, D]
  window, first   attention to the last positions and the first ones alone (0: to all)
  softcap, sinks  scores bounded by softcap * tanh(s / softcap); a learned logit for each head
  axes      axes of the positions that are rotated by (1: text; 3: time, height, width)
  turned    values of a head that are rotated;  pairs: neighbours rotate together, not halves
"""
from __future__ import annotations

import math
import random

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_FP8 = torch.float8_e4m3fn
_EPS = 1e-6


def _case(op, B, longest, heads, *, tokens=0, spare=0, ps=16, block=0, kind="bf16", layout="heads", window=0, first=0,
          softcap=0.0, sinks=False, axes=1, turned=0, pairs=False, name=None):
    Hkv, G, D = heads
    case = dict(op=op, B=B, longest=longest, tokens=tokens, spare=spare, Hkv=Hkv, G=G, D=D, ps=ps, block=block, kind=kind,
                layout=layout, window=window, first=first, softcap=softcap, sinks=sinks, axes=axes,
                turned=turned or D, pairs=pairs)
    return case if name is None else dict(case, name=name)


def listed():
    narrow, wide = (8, 8, 64), (8, 4, 128)
    return [
        # one user's next token: the smallest call, latency alone
        _case("rotate", 1, 131071, wide, tokens=1, name="rotate_one"),
        # prompts of text, images and video: three axes, an odd number of tokens
        _case("rotate", 1, 32768, wide, tokens=8191, axes=3, name="rotate_axes"),
        # a decode batch's new tokens into an 8-bit cache: latency, and blocks whose scale has to grow
        _case("write", 255, 1024, wide, ps=32, block=32, name="write_tokens"),
        # ragged pieces of prompts
        _case("write", 16, 2048, wide, tokens=8191, block=16, name="write_prompts"),
        # one prompt's cached beginning, for another user's prompt
        _case("read", 1, 1000, narrow, tokens=1000, block=16, name="read_one"),
        # a batch's whole caches, to be kept elsewhere in 16 bits
        _case("read", 16, 8192, wide, tokens=60001, spare=3, ps=64, block=16, layout="tokens", name="read_batch"),
        # one user with a very long context on an 8-bit cache
        _case("token", 1, 131071, wide, ps=64, block=64, name="token_long_8bit"),
        # a large batch on an 8-bit cache, the most memory a step reads
        _case("token", 255, 8192, wide, ps=32, block=16, name="token_batch_8bit"),
        # a decode batch in a layer with a window and first tokens that stay visible
        _case("token", 64, 8192, narrow, window=128, first=4, sinks=True, name="token_window"),
        # drafted tokens of a decode batch to be checked, on an 8-bit cache: few rows, long keys
        _case("prompt", 32, 8192, wide, tokens=32 * 5, ps=32, block=32, name="prompt_drafted"),
        # ragged prompts in a layer with a window and first tokens that stay visible
        _case("prompt", 4, 4093, narrow, tokens=8191, spare=2, window=1024, first=4, sinks=True, name="prompt_window"),
        # a piece of a long prompt over all that came before: the most products
        _case("prompt", 1, 16384, wide, tokens=4096, name="prompt_piece"),
    ]


_MOST = 255 * 8192 * 8 * 128        # values of a cache, of the largest listed case
_PRODUCTS = 4096 * 16384 * 32       # scores of the largest listed case


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def draw(rng):
    """Batches, lengths and tokens spread over their logarithms, on head layouts beside the listed ones."""
    op = rng.choice(("rotate", "rotate", "write", "write", "read", "token", "token", "token", "prompt", "prompt", "prompt"))
    kind = rng.choice(("bf16", "bf16", "fp16"))
    D = rng.choice((64, 64, 80, 96, 128, 128, 192, 256))
    Hkv, G = rng.choice((1, 2, 4, 8, 8, 16)), rng.choice((1, 2, 3, 4, 5, 7, 8, 8, 12, 16))
    if op == "rotate":
        T = _log_int(rng, 1, max(1, min(16384, (8191 * 40 * 128) // ((G + 1) * Hkv * D))))
        turned = rng.choice((D, D, D // 2 if D % 4 == 0 else D, 32))
        return _case(op, 1, rng.choice((2048, 32768, 1 << 20)), (Hkv, G, D), tokens=T, kind=kind,
                     axes=rng.choice((1, 1, 3, 4)), turned=turned, pairs=rng.random() < 0.4)
    ps = rng.choice((8, 16, 16, 24, 32, 48, 64, 128))
    block = rng.choice([b for b in (1, 4, 8, 16, 16, 32, 64, 128) if ps % b == 0])
    window = first = 0
    softcap, sinks = rng.choice((0.0, 0.0, 0.0, 30.0)), rng.random() < 0.4
    layout = rng.choice(("heads", "tokens"))
    if op in ("token", "prompt") and rng.random() < 0.4:
        block = 0
    if op == "token":
        B = _log_int(rng, 1, 256)
        longest = _log_int(rng, 1, max(1, min(_MOST // 2 // (B * Hkv * D), (1 << 28) // (B * Hkv * G), 131072)))
        tokens = 0
    elif op == "prompt":
        B = _log_int(rng, 1, 64)
        longest = _log_int(rng, 1, max(1, min(16384, _MOST // 8 // (B * Hkv * D))))
        # (a padded batch of the plain form stays within the largest listed case's scores)
        most = max(1, min(longest, _PRODUCTS // 2 // (B * Hkv * G * (longest + ps))))
        tokens = B * _log_int(rng, 1, most)
    else:
        B = _log_int(rng, 1, 256)
        longest = _log_int(rng, 1, max(1, min(32768, _MOST // 4 // (B * Hkv * D))))
        tokens = _log_int(rng, 1, B * longest)
        if op == "write":
            tokens = 0 if rng.random() < 0.4 else min(tokens, 16384)
    if op in ("token", "prompt") and rng.random() < 0.5:
        window, first = _log_int(rng, 1, longest), rng.choice((0, 1, 4, 16, 100))
    # (no more new tokens than positions, and in a ragged batch of prompts some older ones)
    held = sum(_lengths(dict(op=op, B=B, longest=longest)))
    tokens = min(tokens, max(1, held // 2) if op == "prompt" and B > 1 else held)
    spare = rng.choice((0, 0, 1, 5)) if op in ("read", "prompt") and tokens > 5 else 0
    attends = op in ("token", "prompt")
    return _case(op, B, longest, (Hkv, G, D), tokens=tokens, spare=spare, ps=ps, block=block, kind=kind, layout=layout,
                 window=window, first=first, softcap=softcap if attends else 0.0, sinks=sinks and attends)


# ---- inputs ------------------------------------------------------------------------------------

def _lengths(case):
    """The sequences' lengths: the first the longest, the others down to an eighth of it, and in a
    batch of one token each one that is empty (a row of a padded batch)."""
    rng = random.Random(case["B"] * 131 + case["longest"])
    lens = [case["longest"]] + [rng.randint(max(1, case["longest"] // 8), case["longest"]) for _ in range(case["B"] - 1)]
    if case["op"] == "token" and case["B"] >= 8:
        lens[3] = 0
    return lens


def _new_tokens(case):
    """New tokens (rows that are read) of every sequence: one, or `tokens` less the spare ones spread raggedly,
    none longer than its sequence and none much more than its part."""
    lens = _lengths(case)
    if not case["tokens"]:
        return [1] * len(lens)
    wanted = case["tokens"] - case["spare"]
    rng = random.Random(case["tokens"])
    share = [rng.random() + 1.0 for _ in lens]
    new = [min(n, int(wanted * s / sum(share))) for n, s in zip(lens, share)]
    short = wanted - sum(new)
    for most in (max(1, wanted // len(lens)), wanted):
        for i, n in enumerate(lens):
            more = min(short, n - new[i], most)
            new[i] += more
            short -= more
    return new


def _codes(case, pages, gen, dev, tame):
    """A 16-bit cache, or E4M3 codes (with a few large channels where `tame` is false, as keys have)."""
    Hkv, D, ps = case["Hkv"], case["D"], case["ps"]
    order = (pages, Hkv, ps, D) if case["layout"] == "heads" else (pages, ps, Hkv, D)
    c = torch.randn(order, device=dev, generator=gen, dtype=_TYPES[case["kind"]])
    if case["block"]:
        c = (c * (120.0 if tame else 100.0)).clamp(-448.0, 448.0).to(_FP8)
    return c if case["layout"] == "heads" else c.transpose(1, 2)


def _section(case):
    """Frequencies of each axis, the first ones of the first."""
    n, axes = case["turned"] // 2, case["axes"]
    return [n * (i + 1) // axes - n * i // axes for i in range(axes)]


def _prepare_rotate(case, gen, dev):
    T, Hkv, G, D, t = case["tokens"], case["Hkv"], case["G"], case["D"], _TYPES[case["kind"]]
    # one projection's result, of which queries and keys are the first heads
    qkv = torch.randn((T, (G + 2) * Hkv, D), device=dev, generator=gen).to(t)
    base = 1e6 if case["longest"] > 100000 else 1e4
    inv_freq = base ** (-torch.arange(0, case["turned"], 2, device=dev, dtype=torch.float64) / case["turned"])
    if case["axes"] == 1:
        start = case["longest"] - T if case["longest"] > T else 0
        positions = torch.arange(start, start + T, device=dev, dtype=torch.int32)
    else:
        positions = torch.randint(0, case["longest"], (case["axes"], T), device=dev, generator=gen, dtype=torch.int32)
    return dict(case=case, q=qkv[:, :G * Hkv], k=qkv[:, G * Hkv:(G + 1) * Hkv], positions=positions,
                inv_freq=inv_freq.float(), q_weight=(1 + 0.2 * torch.randn(D, device=dev, generator=gen)).to(t),
                k_weight=(1 + 0.2 * torch.randn(D, device=dev, generator=gen)).to(t))


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    if case["op"] == "rotate":
        return _prepare_rotate(case, gen, dev)
    B, Hkv, G, D, ps, block = (case[n] for n in ("B", "Hkv", "G", "D", "ps", "block"))
    t, lens, new = _TYPES[case["kind"]], _lengths(case), _new_tokens(case)
    width = -(-case["longest"] // ps)
    need = torch.tensor([-(-n // ps) for n in lens], device=dev)
    pages = int(sum(-(-n // ps) for n in lens)) + 3
    # every sequence's pages, scattered over the cache as a server's are; -1 where it has none
    at = torch.arange(width, device=dev)[None, :]
    taken = (need.cumsum(0) - need)[:, None] + at
    shuffled = torch.randperm(pages, device=dev, generator=gen)
    table = torch.where(at < need[:, None], shuffled[taken.clamp(max=pages - 1)], -1).to(torch.int32)
    state = dict(case=case, table=table, lens=torch.tensor(lens, dtype=torch.int32, device=dev), most_new=max(new),
                 k_cache=_codes(case, pages, gen, dev, False), v_cache=_codes(case, pages, gen, dev, True),
                 k_scale=None, v_scale=None, sinks=None, starts=None)
    if block:
        for name in ("k_scale", "v_scale"):
            # blocks of rows of about one size, some of them several times larger
            size = torch.exp(0.4 * torch.randn((pages, Hkv, ps // block), device=dev, generator=gen))
            state[name] = size / 110
    if case["op"] in ("token", "prompt"):
        # queries of 2.5 times the keys' size: a few positions take most of the weight
        rows = case["tokens"] or B
        state["q"] = (2.5 * torch.randn((rows, Hkv * G, D), device=dev, generator=gen)).to(t)
        if case["sinks"]:
            state["sinks"] = torch.randn(Hkv * G, device=dev, generator=gen)
    if case["op"] == "write":
        channels = 1 + 3 * (torch.rand((Hkv, D), device=dev, generator=gen) < 0.02)
        state["k_new"] = (channels * torch.randn((sum(new), Hkv, D), device=dev, generator=gen)).to(t)
        state["v_new"] = torch.randn((sum(new), Hkv, D), device=dev, generator=gen).to(t)
    if case["tokens"]:
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        state["starts"] = torch.tensor(starts, dtype=torch.int32, device=dev)
    return state


# ---- one pass -----------------------------------------------------------------------------------

def run(state):
    run_op = {"rotate": (_plain_rotate, _run_rotate), "write": (_plain_write, _run_write),
              "read": (_plain_read, _run_read), "token": (_plain_token, _run_token),
              "prompt": (_plain_prompt, _run_prompt)}[state["case"]["op"]]
    return run_op[1 if own else 0](state)


def _run_rotate(s):
    from vkernels_amd import rotary
    case = s["case"]
    q, k = rotary.qk_norm_rope(s["q"], s["k"], s["positions"], s["inv_freq"], q_weight=s["q_weight"], k_weight=s["k_weight"],
                               eps=_EPS, sections=None if case["axes"] == 1 else _section(case), pairs=case["pairs"])
    return {"q": q, "k": k}


def _run_write(s):
    from vkernels_amd import kv_cache
    kv_cache.kv_cache_append(s["k_new"], s["v_new"], s["k_cache"], s["v_cache"], s["table"], s["lens"],
                             query_start=s["starts"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    return {n: s[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale")}


def _run_read(s):
    from vkernels_amd import kv_cache
    k, v = kv_cache.kv_cache_read(s["k_cache"], s["v_cache"], s["table"], s["lens"], query_start=s["starts"],
                                  tokens=s["case"]["tokens"], k_scale=s["k_scale"], v_scale=s["v_scale"],
                                  dtype=_TYPES[s["case"]["kind"]])
    return {"k": k, "v": v}


def _run_token(s):
    from vkernels_amd import kv_cache
    case = s["case"]
    out, lse = kv_cache.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"],
                                        max_len=case["longest"], window=case["window"], keep_first=case["first"],
                                        softcap=case["softcap"], sinks=s["sinks"], k_scale=s["k_scale"],
                                        v_scale=s["v_scale"], return_lse=True)
    return {"out": out, "lse": lse}


def _run_prompt(s):
    from vkernels_amd import kv_cache
    case = s["case"]
    out, lse = kv_cache.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"],
                                        query_start=s["starts"], max_len=case["longest"], window=case["window"],
                                        keep_first=case["first"], softcap=case["softcap"], sinks=s["sinks"],
                                        k_scale=s["k_scale"], v_scale=s["v_scale"], return_lse=True)
    return {"out": out, "lse": lse}


# ---- the same in elementary operations, in 32 bits -------------------------------------------------

def _plain_rotate(s):
    case = s["case"]
    n = case["turned"] // 2
    axis = torch.repeat_interleave(torch.arange(case["axes"], device=s["q"].device),
                                   torch.tensor(_section(case), device=s["q"].device), output_size=n)
    # (angles of far positions lose their fraction in 32 bits)
    where = s["positions"].view(case["axes"], -1).double().t()[:, axis]
    angle = where * s["inv_freq"].double()
    cos, sin = torch.cos(angle).float()[:, None, :], torch.sin(angle).float()[:, None, :]
    return {"q": _plain_turn(case, s["q"], s["q_weight"], cos, sin), "k": _plain_turn(case, s["k"], s["k_weight"], cos, sin)}


def _plain_turn(case, rows, weight, cos, sin):
    x = rows.float()
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS) * weight.float()
    turned, rest = x[..., :case["turned"]], x[..., case["turned"]:]
    if case["pairs"]:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = turned.chunk(2, -1)
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, rest], -1).to(rows.dtype)


def _plain_places(s):
    """(sequence, position) of every new token; the rows behind the last sequence's are left out."""
    lens = s["lens"].long()
    if s["starts"] is None:
        return torch.arange(lens.shape[0], device=lens.device), lens - 1
    t = torch.arange(s["case"]["tokens"] - s["case"]["spare"], device=lens.device)
    starts = s["starts"].long()
    seq = (torch.searchsorted(starts, t, right=True) - 1).clamp(max=lens.shape[0] - 1)
    return seq, lens[seq] - starts[seq + 1] + t


def _plain_write(s):
    case = s["case"]
    ps, block = case["ps"], case["block"]
    seq, place = _plain_places(s)
    seq, place = seq[:s["k_new"].shape[0]], place[:s["k_new"].shape[0]]
    page = s["table"].long()[seq, place // ps]
    # the block that each sequence's first new token falls into, which may hold older positions
    new = torch.zeros_like(s["lens"], dtype=torch.long).index_add_(0, seq, torch.ones_like(seq))
    first = s["lens"].long() - new
    slots = first[:, None] // block * block + torch.arange(block, device=first.device)
    older = (slots < first[:, None]) & (new > 0)[:, None]
    at = (s["table"].long()[torch.arange(first.shape[0], device=first.device), (first // ps).clamp(max=s["table"].shape[1] - 1)],
          first % ps // block, slots % ps, older)
    _plain_quantise(s["k_cache"], s["k_scale"], s["k_new"], page, place % ps, at, block)
    _plain_quantise(s["v_cache"], s["v_scale"], s["v_new"], page, place % ps, at, block)
    return {n: s[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale")}


def _plain_quantise(cache, scales, rows, page, slot, at, block):
    codes = cache.view(torch.uint8)
    pages, heads, blocks = scales.shape
    x = rows.float()
    # the largest of the new rows in each block, and the old scale where the block has older positions
    size = x.abs().amax(2)
    need = torch.full((pages * blocks, heads), -1.0, device=x.device)
    which = page * blocks + slot // block
    need.scatter_reduce_(0, which[:, None].expand(-1, heads), size / 448.0, "amax")
    need = need.view(pages, blocks, heads).transpose(1, 2)
    old_page, old_block, old_slots, older = at
    has = torch.nonzero(older.any(1)).view(-1)
    old_page = old_page.clamp(min=0)
    kept = torch.zeros_like(scales)
    kept[old_page[has], :, old_block[has]] = scales[old_page[has], :, old_block[has]]
    grown = torch.maximum(need, kept)
    touched = need >= 0
    # older codes of blocks whose scale grows
    rows_at = old_page[:, None].expand_as(old_slots)
    factor = (scales[old_page, :, old_block] / grown[old_page, :, old_block])[:, None, :, None]
    before = codes[rows_at, :, old_slots]
    again = (before.view(_FP8).float() * factor).to(_FP8).view(torch.uint8)
    grows = older[:, :, None, None] & (grown[old_page, :, old_block] > scales[old_page, :, old_block])[:, None, :, None]
    b, j = torch.nonzero(older, as_tuple=True)
    codes[old_page[b], :, old_slots[b, j]] = torch.where(grows, again, before)[b, j]
    scales.copy_(torch.where(touched, grown, scales))
    by = scales[page, :, slot // block][..., None]
    codes[page, :, slot] = torch.where(by > 0, (x / by).clamp(-448.0, 448.0), 0.0).to(_FP8).view(torch.uint8)


def _plain_read(s):
    case = s["case"]
    ps, block = case["ps"], case["block"]
    seq, place = _plain_places(s)
    page, slot = s["table"].long()[seq, place // ps], place % ps
    behind = case["spare"] if case["tokens"] else 0
    return {n: torch.nn.functional.pad(
        s[n + "_cache"].view(torch.uint8)[page, :, slot].view(_FP8).float() * s[n + "_scale"][page, :, slot // block][..., None],
        (0, 0, 0, 0, 0, behind)).to(_TYPES[case["kind"]]) for n in ("k", "v")}


def _plain_rows(cache, scales, table):
    """[B, Hkv, positions, D] in 32 bits of every sequence's pages."""
    pages = table.long().clamp(min=0)
    if scales is None:
        rows = cache[pages].transpose(1, 2).float()
    else:
        rows = cache.view(torch.uint8)[pages].view(_FP8).transpose(1, 2).float()
        rows *= scales[pages].repeat_interleave(cache.shape[2] // scales.shape[2], 3).transpose(1, 2)[..., None]
    B, Hkv, W, ps, D = rows.shape
    return rows.reshape(B, Hkv, W * ps, D)


def _plain_softmax(s, score, seen):
    """Weights in the scores' place (zeros in a row that sees nothing), and the log of their sum."""
    case = s["case"]
    if case["softcap"]:
        score = case["softcap"] * torch.tanh(score / case["softcap"])
    score = score.masked_fill_(~seen, float("-inf"))
    top = score.amax(-1)
    sinks = None if s["sinks"] is None else s["sinks"].view(1, case["Hkv"], case["G"], *[1] * (top.dim() - 3))
    if sinks is not None:
        top = torch.maximum(top, sinks)
    top = torch.where(torch.isinf(top) & (top < 0), 0.0, top)
    weight = score.sub_(top[..., None]).exp_()
    total = weight.sum(-1)
    if sinks is not None:
        total = total + torch.exp(sinks - top)
    weight /= torch.where(total == 0, 1.0, total)[..., None]
    return weight, torch.log(total) + top


def _plain_seen(case, at, place):
    """Whether a query at `place` sees position `at`."""
    seen = at <= place
    if case["window"]:
        seen = seen & ((at > place - case["window"]) | (at < case["first"]))
    return seen


def _plain_token(s):
    case = s["case"]
    B, Hkv, G, D = (case[n] for n in ("B", "Hkv", "G", "D"))
    k = _plain_rows(s["k_cache"], s["k_scale"], s["table"])
    score = s["q"].float().view(B, Hkv, G, D) @ k.transpose(2, 3)
    del k
    score *= D ** -0.5
    at = torch.arange(score.shape[3], device=score.device)
    seen = _plain_seen(case, at, s["lens"].long().view(B, 1, 1, 1) - 1)
    weight, lse = _plain_softmax(s, score, seen)
    out = weight @ _plain_rows(s["v_cache"], s["v_scale"], s["table"])
    return {"out": out.view(B, Hkv * G, D).to(s["q"].dtype), "lse": lse.view(B, Hkv * G)}


def _plain_prompt(s):
    case = s["case"]
    B, Hkv, G, D = (case[n] for n in ("B", "Hkv", "G", "D"))
    n, rows = s["most_new"], case["tokens"]
    starts = s["starts"].long()
    i = torch.arange(n, device=starts.device)
    token = (starts[:-1, None] + i).clamp(max=rows - 1)                          # [B, n]
    place = s["lens"].long()[:, None] - (starts[1:] - starts[:-1])[:, None] + i
    q = s["q"].float()[token].view(B, n, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * n, D)
    k = _plain_rows(s["k_cache"], s["k_scale"], s["table"])
    score = (q @ k.transpose(2, 3)).view(B, Hkv, G, n, -1)
    del k
    score *= D ** -0.5
    at = torch.arange(score.shape[4], device=score.device)
    seen = _plain_seen(case, at, place.view(B, 1, 1, n, 1))
    weight, lse = _plain_softmax(s, score, seen)
    out = weight.view(B, Hkv, G * n, -1) @ _plain_rows(s["v_cache"], s["v_scale"], s["table"])
    out = out.view(B, Hkv, G, n, D).permute(0, 3, 1, 2, 4).reshape(B, n, Hkv * G, D)
    lse = lse.view(B, Hkv, G, n).permute(0, 3, 1, 2).reshape(B, n, Hkv * G)
    b, j = torch.nonzero(i < (starts[1:] - starts[:-1])[:, None], as_tuple=True)
    whole, whole_lse = s["q"].new_zeros(s["q"].shape), lse.new_full((rows, Hkv * G), float("-inf"))
    whole[token[b, j]], whole_lse[token[b, j]] = out[b, j].to(s["q"].dtype), lse[b, j]
    return {"out": whole, "lse": whole_lse}


# ---- the definition, in 64 bits ------------------------------------------------------------------

def _exact_rotate(s):
    """Every pair as a complex number times e^(i angle)."""
    case = s["case"]
    n = case["turned"] // 2
    of = [axis for axis, count in enumerate(_section(case)) for _ in range(count)]
    p = s["positions"].double().view(case["axes"], -1)
    angle = torch.stack([p[axis] * float(f) for axis, f in zip(of, s["inv_freq"].tolist())], 1)[:, None, :]
    unit = torch.polar(torch.ones_like(angle), angle)
    index = torch.arange(case["turned"], device=p.device)
    index = index.view(n, 2) if case["pairs"] else index.view(2, n).t().contiguous()
    got = {}
    for name in ("q", "k"):
        x = s[name].double()
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / case["D"] + _EPS) * s[name + "_weight"].double()
        y = torch.complex(x[..., index[:, 0]], x[..., index[:, 1]]) * unit
        out = x.clone()
        out[..., index[:, 0]], out[..., index[:, 1]] = y.real, y.imag
        got[name] = out
    return got


def _exact_positions(s, b, lo, hi):
    """(pages, slots) of positions lo .. hi - 1 of sequence b."""
    j = torch.arange(lo, hi, device=s["table"].device)
    return s["table"][b].long()[j // s["case"]["ps"]], j % s["case"]["ps"]


def _exact_rows(s, name, b, lo, hi):
    """[positions, Hkv, D] of a sequence."""
    pages, slots = _exact_positions(s, b, lo, hi)
    cache, scales = s[name + "_cache"], s[name + "_scale"]
    if scales is None:
        return cache[pages, :, slots].double()
    codes = cache.view(torch.uint8)[pages, :, slots].view(_FP8).double()
    return codes * scales[pages, :, slots // s["case"]["block"]].double()[..., None]


def _to_codes(x):
    """The nearest E4M3 values of numbers in 64 bits."""
    return x.clamp(-448.0, 448.0).float().to(_FP8).double()


def _exact_write(s):
    """Sequence by sequence and block by block.  (Scales are held in 32 bits: a quotient rounded once.)"""
    case = s["case"]
    ps, block = case["ps"], case["block"]
    new, lens = _new_tokens(case), _lengths(case)
    if sum(-(-n // block) + 1 for n in new) > 3000:
        return None
    got = {}
    for name in ("k", "v"):
        cache, scales = s[name + "_cache"].double(), s[name + "_scale"].clone()
        done = 0
        for b, (n, length) in enumerate(zip(new, lens)):
            rows = s[name + "_new"][done:done + n].double()
            done += n
            at = length - n
            while at < length:
                begin = at // block * block
                end = min(begin + block, length)
                page, slot, j = int(s["table"][b, begin // ps]), begin % ps, begin % ps // block
                mine = rows[at - (length - n):end - (length - n)]                   # [rows, Hkv, D]
                scale = (mine.abs().amax((0, 2)) / 448).float()
                if at > begin:
                    old = scales[page, :, j]
                    scale = torch.maximum(old, scale)
                    older = cache[page, :, slot:slot + at - begin]
                    cache[page, :, slot:slot + at - begin] = _to_codes(older * (old.double() / scale.double())[:, None, None])
                by = scale.double()[None, :, None]
                codes = _to_codes(torch.where(by > 0, mine / by, 0.0))
                cache[page, :, slot + at - begin:slot + end - begin] = codes.transpose(0, 1)
                scales[page, :, j] = scale
                at = end
        got[name + "_cache"], got[name + "_scale"] = cache, scales.double()
    return got


def _exact_read(s):
    case = s["case"]
    got = {}
    for name in ("k", "v"):
        rows = [_exact_rows(s, name, b, length - n, length)
                for b, (n, length) in enumerate(zip(_new_tokens(case), _lengths(case)))]
        rows = torch.cat(rows)
        got[name] = torch.cat([rows, rows.new_zeros((case["tokens"] - rows.shape[0], *rows.shape[1:]))])
    return got


def _exact_attend(s):
    """A sequence, a head and a few hundred queries at a time."""
    case = s["case"]
    Hkv, G, D = case["Hkv"], case["G"], case["D"]
    rows = s["q"].shape[0]
    out = torch.zeros((rows, Hkv * G, D), dtype=torch.float64, device=s["q"].device)
    lse = torch.full((rows, Hkv * G), -math.inf, dtype=torch.float64, device=s["q"].device)
    done = 0
    for b, (n, length) in enumerate(zip(_new_tokens(case), _lengths(case))):
        begin, done = done, done + n
        k, v = (_exact_rows(s, name, b, 0, length) for name in ("k", "v"))
        at = torch.arange(length, device=k.device)
        for g in range(Hkv):
            kg, vg = k[:, g].t().contiguous(), v[:, g].contiguous()
            for i in range(0, n, 512):
                m = min(512, n - i)
                heads = slice(G * g, G * g + G)
                q = s["q"][begin + i:begin + i + m, heads].double().reshape(m * G, D) / math.sqrt(D)
                score = (q @ kg).view(m, G, length)
                if case["softcap"]:
                    score = torch.tanh(score / case["softcap"]) * case["softcap"]
                place = torch.arange(length - n + i, length - n + i + m, device=k.device).view(m, 1, 1)
                hidden = at > place
                if case["window"]:
                    hidden |= (at <= place - case["window"]) & (at >= case["first"])
                score = score.masked_fill(hidden, -math.inf)
                extra = score.new_full((1, G, 1), -math.inf) if s["sinks"] is None else s["sinks"][heads].double().view(1, G, 1)
                total = torch.logsumexp(torch.cat([score, extra.expand(m, G, 1)], 2), 2)
                share = torch.exp(score - torch.where(torch.isinf(total), 0.0, total)[..., None])
                out[begin + i:begin + i + m, heads] = (share.view(m * G, length) @ vg).view(m, G, D)
                lse[begin + i:begin + i + m, heads] = total
    return {"out": out, "lse": lse}


def exact(case, seed):
    return {"rotate": _exact_rotate, "write": _exact_write, "read": _exact_read, "token": _exact_attend,
            "prompt": _exact_attend}[case["op"]](prepare(case, seed))


# ---- what a pass cannot do without -----------------------------------------------------------------

def _visible(case, length, n):
    """(positions of a sequence that any of its last n queries sees, pairs of a query and a position)."""
    w, f = case["window"], case["first"]
    if not w:
        return length, n * length - n * (n - 1) // 2
    lows = [max(0, place + 1 - w) for place in range(length - n, length)]
    pairs = sum(place + 1 - low + min(f, low) for place, low in zip(range(length - n, length), lows))
    return (length - lows[0] + min(f, lows[0]) if n else 0), pairs


def work(case):
    Hkv, G, D = case["Hkv"], case["G"], case["D"]
    if case["op"] == "rotate":
        rows = case["tokens"] * (G + 1) * Hkv
        return {"bytes": rows * D * 4 + 4 * case["tokens"] * case["axes"], "flops": rows * (4 * D + 3 * case["turned"])}
    row = 2 * D * (1 if case["block"] else 2)       # a position's key and value in one head
    lens, new = _lengths(case), _new_tokens(case)
    T, scale = sum(new), 8 / case["block"] if case["block"] else 0
    if case["op"] == "write":
        return {"bytes": int(T * Hkv * (4 * D + row + scale)), "flops": T * Hkv * 4 * D}
    if case["op"] == "read":
        return {"bytes": int(T * Hkv * (4 * D + row + scale)), "flops": T * Hkv * 2 * D}
    seen = [_visible(case, length, min(n, length)) for length, n in zip(lens, new)]
    q = T * Hkv * G * (4 * D + 4)
    return {"bytes": int(sum(a for a, _ in seen) * Hkv * (row + scale)) + q,
            "flops": 4 * D * Hkv * G * sum(b for _, b in seen)}
