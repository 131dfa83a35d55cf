"""GPU tests of the attention of several new tokens of every sequence against the definition in 64 bits."""
from __future__ import annotations

import math

import pytest
import torch

import attention_reference as aref
import kv_reference as ref
from test_gpu_kv_window import BF16, F16, FP8, Setup, dev
from vkernels_amd import kv_cache as kv

pytestmark = pytest.mark.gpu


class Prompt(Setup):
    def __init__(self, lens, new, *args, spare=0, **kw):
        super().__init__(lens, *args, tokens=sum(new) + spare, **kw)
        self.new = list(new)
        self.starts = torch.tensor([0, *new]).cumsum(0).to(torch.int32).to(dev())

    def call(self, **kw):
        return kv.paged_attention(self.q, self.k, self.v, self.table, self.lens, query_start=self.starts, return_lse=True,
                                  **dict(dict(k_scale=self.k_scale, v_scale=self.v_scale), **kw))

    def check(self, *, sinks=False, what="", got=None, **kw):
        kw = dict(kw, sinks=self.sinks if sinks else None)
        out, lse = got if got is not None else self.call(**kw)
        torch.cuda.synchronize()
        # (bf16 has 8 significant bits, fp16 11; weights of 8-bit caches are fp16)
        bits = 11 if self.q.dtype is F16 or self.block else 8
        want = aref.attention(self.q, self.k, self.v, self.table, self.lens, self.starts, k_scale=self.k_scale,
                              v_scale=self.v_scale, weight_bits=bits, **dict(kw, scale=kw.get("scale", self.D ** -0.5)))
        n = sum(self.new)
        mine = tuple(x[:n] for x in want[:2])
        ref.assert_attention(out[:n], lse[:n], (*mine, None, (want[3][0][:n], want[3][1][:n], None)), self.q.dtype, what)
        if out.shape[0] > n:
            assert bool((out[n:] == 0).all()) and bool((lse[n:] == -math.inf).all())
        return out, lse


LENS = [0, 1, 5, 64, 65, 130, 300, 33]
NEW = [0, 1, 5, 17, 65, 1, 129, 0]


@pytest.mark.parametrize("D", [16, 48, 64, 80, 96, 112, 128, 160, 192, 240, 256])
@pytest.mark.parametrize("q", [BF16, F16])
@pytest.mark.parametrize("block,ps", [(0, 16), (0, 24), (-1, 16), (8, 16), (24, 24), (1, 5)])
def test_widths_and_types(hip_lib, D, q, block, ps):
    Prompt(LENS, NEW, 2, 3, D, ps, block, q=q, seed=D + ps, spare=2).check(sinks=True)


@pytest.mark.parametrize("Hkv,G", [(1, 1), (3, 1), (1, 2), (8, 8), (1, 7), (2, 33), (1, 70), (1, 129), (1, 260), (16, 1)])
def test_head_layouts(hip_lib, Hkv, G):
    Prompt([200, 3, 70, 129], [150, 3, 1, 128], Hkv, G, 64, 16, 0, seed=G).check()


@pytest.mark.parametrize("window", [1, 2, 17, 64, 100, 200])
@pytest.mark.parametrize("first", [0, 1, 4, 63, 64, 65, 150, 100000])
def test_windows_with_first_positions(hip_lib, window, first):
    Prompt([500, 130, 64, 3], [300, 130, 1, 2], 2, 4, 64, 16, 0, seed=window + first).check(window=window, keep_first=first, sinks=True)


@pytest.mark.parametrize("window,first", [(0, 0), (300, 10), (1500, 700)])
@pytest.mark.parametrize("block,D", [(0, 64), (0, 128), (16, 128), (-1, 192)])
@pytest.mark.parametrize("q", [BF16, F16])
def test_few_tokens_on_long_sequences(hip_lib, window, first, block, D, q):
    """Tiles whose positions several workgroups share."""
    Prompt([5000, 1, 2200, 700, 0], [3, 1, 8, 20, 0], 2, 4, D, 16, block, q=q, seed=D, spare=1).check(window=window, keep_first=first, sinks=True)


@pytest.mark.parametrize("window,first", [(0, 0), (300, 70)])
@pytest.mark.parametrize("block,ps,D", [(16, 16, 256), (-1, 16, 160), (8, 24, 208), (1, 5, 240), (16, 16, 144), (16, 16, 192), (4, 16, 112)])
@pytest.mark.parametrize("q", [BF16, F16])
def test_few_tokens_over_codes_of_every_width(hip_lib, window, first, block, ps, D, q):
    Prompt([3000, 1, 700, 90, 0], [3, 1, 8, 12, 0], 2, 4, D, ps, block, q=q, seed=D, spare=1).check(window=window, keep_first=first, sinks=True)
    Prompt([300, 33, 64], [1, 2, 16], 1, 5, D, ps, block, q=q, seed=D + 1, layout="tokens").check(softcap=20.0)


@pytest.mark.parametrize("new", [(200, 150), (3, 5)])
@pytest.mark.parametrize("q,size", [(BF16, 2.0 ** -54), (BF16, 2.0 ** 60), (BF16, 1.0), (F16, 2.0 ** -6), (F16, 2.0 ** 5), (F16, -1.0)])
@pytest.mark.parametrize("block", [-1, 4, 16])
def test_value_scales_of_any_size(hip_lib, new, q, size, block):
    """The weights' reference follows them: all far from 1, below it, blocks of zeros and blocks 2^12 apart."""
    s = Prompt([700, 600], new, 2, 4, 128, 16, block, q=q, seed=5)
    s.v_scale = s.v_scale * size
    if block > 0:
        kind = torch.randint(0, 3, s.v_scale.shape, generator=torch.Generator().manual_seed(1)).to(dev())
        s.v_scale = torch.where(kind == 0, s.v_scale, torch.where(kind == 1, s.v_scale * 2.0 ** -12, 0.0))
    s.check(sinks=True)
    s.check(window=100, keep_first=20)


def test_parts_that_see_nothing(hip_lib):
    """Far more room than positions: shares behind every position, and sequences without any."""
    s = Prompt([40, 9, 0], [4, 9, 0], 1, 1, 64, 16, 0)
    s.table = torch.cat([s.table, torch.full((3, 4000), -1, dtype=torch.int32, device=dev())], 1)
    s.check()
    s.check(max_len=33)


@pytest.mark.parametrize("kw", [dict(softcap=20.0), dict(softcap=1e-3), dict(scale=0.3), dict(scale=-0.2), dict(scale=0.0),
                                dict(softcap=5.0, scale=-1.0), dict(softcap=math.inf)])
@pytest.mark.parametrize("block", [0, 8])
def test_scales_and_caps(hip_lib, kw, block):
    s = Prompt([300, 50], [100, 50], 2, 4, 64, 16, block)
    out, lse = s.call(sinks=s.sinks, **kw)
    kw = dict(kw, softcap=0.0 if kw.get("softcap") == math.inf else kw.get("softcap", 0.0))
    s.check(got=(out, lse), sinks=True, **kw)


def test_one_token_each_is_the_step(hip_lib):
    s = Prompt([900, 33, 1, 2000], [1, 1, 1, 1], 2, 8, 128, 16, 0)
    out, lse = s.check(sinks=True, window=500, keep_first=4)
    step, step_lse = kv.paged_attention(s.q, s.k, s.v, s.table, s.lens, sinks=s.sinks, window=500, keep_first=4, return_lse=True)
    assert bool(((lse - step_lse).abs() < 1e-4).all()) and bool(((out - step).abs().float() < 0.05).all())


def test_holes(hip_lib):
    """Entries that are no page leave their positions out; tokens that see nothing else are 0."""
    for ps in (16, 24):
        s = Prompt([300, 100, 40], [200, 100, 40], 2, 4, 64, ps, 0)
        s.table[0, 2], s.table[0, 5], s.table[2, 0] = -1, s.k.shape[0], 2147483647
        out, lse = s.check()
        assert bool((out[300:300 + ps] == 0).all() and (lse[300:300 + ps] == -math.inf).all())


@pytest.mark.parametrize("block,q", [(0, BF16), (0, F16), (8, BF16), (16, F16), (-1, BF16)])
@pytest.mark.parametrize("window,first", [(0, 0), (50, 3)])
def test_what_a_token_does_not_see_may_be_anything(hip_lib, block, q, window, first):
    """NaN and infinities in keys, values and scales at positions that some tokens of a tile see and others do not: rows
    that see them are NaN or infinite as the definition says, all others as if they were not there."""
    s = Prompt([200, 70, 333], [150, 70, 5], 2, 3, 80, 16, block, q=q, seed=5)
    clean = s.call(window=window, keep_first=first)
    touched = {0: (60, 140, 199), 1: (20, 21), 2: (331,)}
    for b, at in touched.items():
        for i, pos in enumerate(at):
            page, slot = int(s.table[b, pos // 16]), pos % 16
            if block:
                codes = s.v.view(torch.uint8)
                codes[page, i % 2, slot, (7 * pos) % 80] = 0xFF          # a NaN
                s.k.view(torch.uint8)[page, 1, slot, 3] = 0x7F
            else:
                s.v[page, i % 2, slot, (7 * pos) % 80] = (math.inf, -math.inf, math.nan)[i]
                s.v[page, i % 2, slot, (7 * pos + 1) % 80] = math.nan
                s.k[page, 1, slot, 3] = math.inf if i else math.nan
    out, lse = s.call(window=window, keep_first=first)
    torch.cuda.synchronize()
    row = 0
    for b, (length, n) in enumerate(zip((200, 70, 333), s.new)):
        for i in range(n):
            place = length - n + i
            sees = [p for p in touched[b] if p <= place and (not window or p > place - window or p < first)]
            if not sees:
                assert torch.equal(out[row], clean[0][row]) and torch.equal(lse[row], clean[1][row]), (b, i)
            else:
                # the value's own head and column, and with it every column of the heads whose keys are no numbers
                for j, p in enumerate(touched[b]):
                    if p in sees:
                        assert not bool(torch.isfinite(out[row, (j % 2) * 3:(j % 2) * 3 + 3, (7 * p) % 80]).any()), (b, i, p)
                assert bool(torch.isfinite(lse[row, :3]).all())
                kept = [d for d in range(80) if d not in {(7 * p + e) % 80 for p in touched[b] for e in (0, 1)}]
                assert torch.equal(out[row, :3, kept], clean[0][row, :3, kept]), (b, i)
            row += 1


def test_scales_that_a_token_does_not_see_may_be_anything(hip_lib):
    s = Prompt([64], [40], 1, 2, 64, 16, 4)
    clean = s.call(window=10)
    s.k_scale[s.table[0, 3].long(), 0, 3], s.v_scale[s.table[0, 3].long(), 0, 3] = math.inf, math.nan       # positions 60 .. 63
    s.k_scale[s.table[0, 0].long(), 0, 1], s.v_scale[s.table[0, 0].long(), 0, 1] = math.nan, math.inf       # 4 .. 7
    out, lse = s.call(window=10)
    assert torch.equal(out[:36], clean[0][:36]) and torch.equal(lse[:36], clean[1][:36])
    assert not bool(torch.isfinite(out[36:]).any())
    # one token: the same scales in front of its window
    lens = torch.tensor([60], dtype=torch.int32, device=dev())
    args = s.q[:1], s.k, s.v, s.table, lens
    for window, first in ((10, 0), (10, 3), (52, 4)):
        got = kv.paged_attention(*args, window=window, keep_first=first, k_scale=s.k_scale, v_scale=s.v_scale)
        assert bool(torch.isfinite(got).all())


def test_more_tokens_than_positions(hip_lib):
    """Tokens in front of a sequence's first position see nothing (a length that a bound has cut, or a wrong one)."""
    s = Prompt([30, 10], [30, 10], 2, 4, 64, 16, 0)
    s.lens -= 7
    s.check(sinks=True)
    s.check(max_len=5)


def test_given_results_keep_the_rows_behind(hip_lib):
    s = Prompt([90, 20], [40, 20], 2, 4, 80, 16, 0, spare=9)
    out = torch.full_like(s.q, 3.0)
    got, lse = s.call(out=out)
    assert got is out and bool((out[60:] == 3).all()) and bool((lse[60:] == -math.inf).all())
    assert torch.equal(out[:60], s.check()[0][:60])


@pytest.mark.parametrize("layout", ["heads", "tokens"])
def test_strides(hip_lib, layout):
    g = torch.Generator().manual_seed(1)
    for block in (0, 8):
        s = Prompt([200, 64], [70, 33], 4, 2, 64, 16, block, layout=layout)
        wide = torch.randn((103, 16, 64), generator=g).to(BF16).to(dev())
        s.q = wide[:, 2:10]
        s.check()
        s.q = torch.randn((103, 8, 67), generator=g).to(BF16).to(dev())[:, :, 2:66]
        s.check()
        s.q = wide[:1, :8].expand(103, 8, 64)
        s.check()
        s.table = s.table.repeat(1, 2)[:, :s.table.shape[1]]
        s.check()


def test_many_sequences(hip_lib):
    g = torch.Generator().manual_seed(9)
    lens = torch.randint(0, 90, (300,), generator=g).tolist()
    new = [int(torch.randint(0, n + 1, (1,), generator=g)) for n in lens]
    Prompt(lens, new, 1, 3, 64, 16, 0, spare=40).check()


def test_longer_prompts(hip_lib):
    Prompt([1500, 1100], [1500, 700], 1, 2, 128, 16, 0).check()
    Prompt([1500, 1100], [1500, 700], 1, 2, 64, 32, 32, q=F16).check(window=700, keep_first=100)


@pytest.mark.parametrize("q", [BF16, F16])
@pytest.mark.parametrize("block", [0, 16])
def test_many_small_weights_beside_a_large_one(hip_lib, q, block):
    """A sink far above every score: the weights that are left are small, and many."""
    s = Prompt([3000], [40], 1, 2, 64, 16, block, q=q, peak=0.05)
    s.sinks = torch.full((2,), 14.0, device=dev())
    s.check(sinks=True)


def test_streams_and_graphs(hip_lib):
    s = Prompt([300, 2000], [5, 9], 2, 4, 128, 16, 16)
    t = Prompt([300, 200], [150, 90], 2, 4, 128, 16, 0)
    for p in (s, t):
        want = p.call()
        side = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            got = p.call()
        side.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, lse = p.call(max_len=int(p.table.shape[1]) * 16)
        for i in range(3):
            p.q.mul_(-0.9)
            p.lens -= 3
            graph.replay()
            eager = p.call(max_len=int(p.table.shape[1]) * 16)
            torch.cuda.synchronize()
            assert torch.equal(out, eager[0]) and torch.equal(lse, eager[1])
            p.check(got=(out, lse))


def test_runs_give_the_same_bits(hip_lib):
    s = Prompt([3000, 900], [6, 300], 2, 4, 128, 16, 0)
    first = s.call()
    for _ in range(3):
        again = s.call()
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_append_then_attend(hip_lib):
    """A prompt in pieces: what each piece gives is what the whole gives."""
    g = torch.Generator().manual_seed(4)
    n, Hkv, G, D = 200, 2, 4, 64
    q, k, v = (torch.randn((n, h, D), generator=g).to(BF16).to(dev()) for h in (Hkv * G, Hkv, Hkv))
    for scales in (False, True):
        t = FP8 if scales else BF16
        caches = [torch.zeros((14, Hkv, 16, D), dtype=t, device=dev()) for _ in range(2)]
        kw = {}
        if scales:
            kw = dict(zip(("k_scale", "v_scale"), (torch.zeros((14, Hkv, 1), device=dev()) for _ in range(2))))
        table = torch.randperm(14, generator=g).to(torch.int32).to(dev())[None]
        for lo, hi in ((0, 64), (64, 65), (65, 180), (180, 200)):
            lens = torch.tensor([hi], dtype=torch.int32, device=dev())
            starts = torch.tensor([0, hi - lo], dtype=torch.int32, device=dev())
            kv.kv_cache_append(k[lo:hi], v[lo:hi], *caches, table, lens, query_start=starts, **kw)
            out, lse = kv.paged_attention(q[lo:hi], *caches, table, lens, query_start=starts, return_lse=True, **kw)
            want = aref.attention(q[lo:hi], *caches, table, lens, starts, scale=D ** -0.5, weight_bits=8, **kw)
            ref.assert_attention(out, lse, want, BF16, f"{lo}:{hi}")


@pytest.mark.parametrize("seed", range(40))
def test_random_calls(hip_lib, seed):
    g = torch.Generator().manual_seed(1000 + seed)
    pick = lambda *x: x[int(torch.randint(0, len(x), (1,), generator=g))]      # noqa: E731
    ps = pick(1, 5, 8, 16, 16, 24, 32, 64)
    block = pick(0, 0, 0, -1, *[b for b in (1, 2, 4, 8, 16, 32, 64) if ps % b == 0])
    B, D = pick(1, 2, 3, 9), pick(16, 64, 64, 80, 96, 128, 128, 144, 192, 256)
    most = pick(5, 70, 300, 900)
    lens = torch.randint(0, most + 1, (B,), generator=g).tolist()
    new = [min(n, int(torch.randint(0, pick(2, 6, 60, 300), (1,), generator=g))) for n in lens]
    s = Prompt(lens, new, pick(1, 2, 3, 8), pick(1, 2, 3, 5, 8, 17), D, ps, block, q=pick(BF16, F16), seed=seed,
               layout=pick("heads", "tokens"), spare=pick(0, 0, 1, 4))
    if sum(new) == 0 and s.q.shape[0] == 0:
        assert s.call()[0].shape[0] == 0
        return
    window = pick(0, 0, 1, 10, 64, 100, 500)
    s.check(window=window, keep_first=pick(0, 1, 4, 70), softcap=pick(0.0, 0.0, 15.0), sinks=pick(False, True), what=str(seed))


def test_nothing_and_refusals(hip_lib):
    s = Prompt([40, 30], [4, 3], 2, 4, 64, 16, 8)
    empty = kv.paged_attention(s.q[:0], s.k, s.v, s.table, s.lens, query_start=s.starts * 0, k_scale=s.k_scale, v_scale=s.v_scale)
    assert empty.shape == (0, 8, 64)
    args = s.q, s.k, s.v, s.table, s.lens
    both = dict(k_scale=s.k_scale, v_scale=s.v_scale, query_start=s.starts)
    sums = torch.zeros((2, 2, 48), device=dev())
    for bad in (dict(weight_sums=sums), dict(query_start=s.starts[:2]), dict(query_start=s.starts.long()), dict(query_start=s.starts.cpu()),
                dict(keep_first=-1, window=5), dict(out=s.q[:, :4]), dict(sinks=s.sinks[:4])):
        with pytest.raises(ValueError):
            kv.paged_attention(*args, **dict(both, **bad))
    for bad in (dict(softcap=-1.0), dict(softcap=math.nan), dict(max_len=49)):
        with pytest.raises(RuntimeError):
            kv.paged_attention(*args, **dict(both, **bad))
    q = s.q.clone().requires_grad_()
    out = kv.paged_attention(q, *args[1:], **both)
    with pytest.raises(RuntimeError, match="no backward"):
        out.float().sum().backward()


@pytest.mark.parametrize("D,q", [(64, F16), (128, F16), (192, F16), (128, BF16)])
@pytest.mark.parametrize("new", [(3, 5), (200, 150)])
@pytest.mark.parametrize("drop", [9, 17, 24, 30])
@pytest.mark.parametrize("every", [0, 64, 1000])
def test_weights_far_below_those_of_values_that_are_zero(hip_lib, D, q, new, drop, every):
    """One position (or every so many) has nearly all of the weight and a value of zero: the others are the result."""
    s = Prompt([8000, 6000], new, 1, 2, D, 16, 0, q=q)
    large = torch.arange(s.table.shape[1] * 16) % every == 0 if every else torch.arange(s.table.shape[1] * 16) == 40
    s.q.zero_()
    s.k.zero_()
    s.v.fill_(8.0)
    s.q[..., 0] = 1.0
    for b in range(2):
        pages = s.table[b][s.table[b] >= 0].long()
        at = large.view(-1, 16)[:len(pages)].to(dev())
        k, v = s.k[pages], s.v[pages]           # [W, 1, 16, D]
        k[..., 0] = torch.where(at[:, None], float(drop), 0.0).to(k.dtype)
        v[at[:, None]] = 0.0
        s.k[pages], s.v[pages] = k, v
    out, lse = s.call(scale=1.0)
    # scores are exact; a weight is rounded once to 16 bits and so is the result; the exponent's product with log2(e) is off by
    # 2^-24 of up to 2^6, a move of the reference by 2^-22, twice for every large position; in fp16 a weight may also be off by
    # 2^-18 of the largest among its 32 positions (which is 2^-7 or more, and a half step 2^-25 or less)
    moves = 2 * (1 if not every else 8000 / every)
    tol = 2 * torch.finfo(q).eps / 2 + 2.0 ** -18 + moves * 2.0 ** -22
    row = 0
    for b, (length, n) in enumerate(zip((8000, 6000), new)):
        for p in range(length - n, length):
            spikes = int(large[:p + 1].sum())
            beside = 0 if q is BF16 else int((large[:8000].view(-1, 32).any(1).repeat_interleave(32) & ~large[:8000])[:p + 1].sum())
            off = beside * min(math.exp(-drop), 2.0 ** -18) / ((p + 1 - spikes) * math.exp(-drop))
            want = 8.0 * (p + 1 - spikes) * math.exp(-drop) / (spikes + (p + 1 - spikes) * math.exp(-drop))
            got = out[row].double()
            assert float((got - want).abs().max()) <= (tol + off) * want + 2.0 ** -25, (b, p)
            row += 1
