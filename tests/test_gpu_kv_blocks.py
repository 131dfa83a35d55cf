"""GPU tests of 8-bit caches with a scale for each block of positions: appends bit for bit against the
definition in 32 bits, and reading caches of every kind back."""
from __future__ import annotations

import math

import pytest
import torch

import kv_blocks_reference as ref
from vkernels_amd import kv_cache as kv

pytestmark = pytest.mark.gpu

BF16, F16, FP8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def dev():
    return torch.device("cuda", 0)


class Cache:
    """An empty cache of scattered pages; what nobody has written is NaN, scales included."""

    def __init__(self, lens, Hkv, D, ps, block, *, layout="heads", seed=1, spare=3, width=None):
        g = self.g = torch.Generator().manual_seed(seed)
        self.lens_host, self.Hkv, self.D, self.ps, self.block = list(lens), Hkv, D, ps, block
        need = [-(-n // ps) for n in lens]
        pages = sum(need) + spare
        order = torch.randperm(pages, generator=g).to(torch.int32)
        self.table = torch.full((len(lens), max(1, max(need))), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.table = self.table.to(dev())[:, :width]
        self.order = order[at:]
        caches = [torch.full((pages, Hkv, ps, D), 0x7F, dtype=torch.uint8).view(FP8).to(dev()) for _ in range(2)]
        if layout == "tokens":
            caches = [c.view(torch.uint8).transpose(1, 2).contiguous().transpose(1, 2).view(FP8) for c in caches]
        self.k, self.v = caches
        self.ks, self.vs = (torch.full((pages, Hkv, ps // block), math.nan, device=dev()) for _ in range(2))

    def rows(self, n, dtype=BF16, size=1.0):
        return [(size * torch.randn((n, self.Hkv, self.D), generator=self.g)).to(dtype).to(dev()) for _ in range(2)]

    def append(self, lens, counts=None, *, dtype=BF16, size=1.0, rows=None, spare=0, check=True):
        """lens count the new tokens; counts: how many of them each sequence has (None: one each)."""
        lens = torch.tensor(lens, dtype=torch.int32, device=dev())
        starts = None if counts is None else torch.tensor([0, *counts]).cumsum(0).to(torch.int32).to(dev())
        k, v = rows if rows is not None else self.rows((len(lens) if counts is None else sum(counts)) + spare, dtype, size)
        want = ref.append(self.k, self.v, self.ks, self.vs, k, v, self.table, lens, starts)
        kv.kv_cache_append(k, v, self.k, self.v, self.table, lens, query_start=starts, k_scale=self.ks, v_scale=self.vs)
        torch.cuda.synchronize()
        if check:
            self.equal(want)
        return k, v

    def equal(self, want):
        for name, got, w in zip(("k scale", "v scale"), (self.ks, self.vs), want[2:]):
            assert torch.equal(got.cpu().view(torch.int32), w.view(torch.int32)), name
        for name, got, w in zip(("k", "v"), (self.k, self.v), want[:2]):
            a, b = got.cpu().contiguous().view(torch.uint8), w.contiguous().view(torch.uint8)
            # (a NaN is a NaN of either sign)
            a, b = (torch.where(x & 0x7F == 0x7F, 0x7F, x) for x in (a, b))
            assert torch.equal(a, b), f"{name}: {int((a != b).sum())} codes differ"


@pytest.mark.parametrize("D", [16, 48, 64, 80, 96, 128, 192, 256])
@pytest.mark.parametrize("ps,block", [(16, 16), (16, 1), (24, 8), (48, 48), (128, 128), (5, 5), (6, 2)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_prompts_and_steps(hip_lib, D, ps, block, dtype):
    """Ragged pieces of prompts, then steps of one token, each larger than the last so that scales grow."""
    final = [70, 1, 0, 33, 200, 17]
    c = Cache([n + 20 for n in final], 3, D, ps, block, seed=D + ps)
    half = [n // 3 for n in final]
    c.append(half, half, dtype=dtype)
    c.append(final, [n - m for n, m in zip(final, half)], dtype=dtype, size=1.7)
    lens = list(final)
    for i in range(5):
        lens = [n + 1 for n in lens]
        c.append(lens, dtype=dtype, size=(0.5, 3.0, 1.0, 9.0, 0.01)[i])


@pytest.mark.parametrize("B", [1, 2, 63, 65, 300])
@pytest.mark.parametrize("layout", ["heads", "tokens"])
def test_batches(hip_lib, B, layout):
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, 40, (B,), generator=g).tolist()
    c = Cache([n + 4 for n in lens], 2, 64, 16, 8, layout=layout, seed=B)
    new = [int(torch.randint(0, n + 1, (1,), generator=g)) for n in lens]
    c.append([n - m for n, m in zip(lens, new)], [n - m for n, m in zip(lens, new)])
    c.append(lens, new, size=2.0)
    c.append([n + 1 for n in lens])
    c.append([n + 4 for n in lens], [3] * B, spare=5)        # rows behind the last sequence


def test_one_token_calls_with_rows_of_a_padded_batch(hip_lib):
    """A sequence of length 0 takes no token; nothing of its row of the table is touched."""
    c = Cache([10, 10, 10], 2, 64, 16, 4)
    c.append([3, 0, 5], [3, 0, 5])
    c.append([4, 0, 6])


def test_quotients_are_rounded_as_divisions(hip_lib):
    """Scales of every kind of significand, all ones among them, over the types' range; values near the borders between
    codes: a quotient that is off by its last bit would give another code there."""
    g = torch.Generator().manual_seed(11)
    n, D = 4096, 256
    for dtype, low, high in ((BF16, -100, 100), (F16, -9, 4)):
        size = torch.exp2(torch.randint(low, high, (n, 1, 1), generator=g).double()) * (1 + torch.rand((n, 1, 1), generator=g).double())
        border = torch.randint(8, 16, (n, 1, D), generator=g).double() + 0.5        # between two significands of a code
        x = size * border / 16 * torch.exp2(-torch.randint(0, 12, (n, 1, D), generator=g).double()) * (1 + 2e-3 * torch.randn((n, 1, D), generator=g).double())
        x = (x * torch.sign(torch.randn((n, 1, D), generator=g).double())).to(dtype)
        x[:, :, :1] = (448 * size).clamp(max=6e4 if dtype is F16 else 3e38).to(dtype)
        c = Cache([n], 1, D, 16, 1)
        lens, starts = torch.tensor([n], dtype=torch.int32, device=dev()), torch.tensor([0, n], dtype=torch.int32, device=dev())
        rows = x.to(dev())
        kv.kv_cache_append(rows, rows, c.k, c.v, c.table, lens, query_start=starts, k_scale=c.ks, v_scale=c.vs)
        page, slot = c.table[0].long()[torch.arange(n, device=dev()) // 16], torch.arange(n, device=dev()) % 16
        scale = x.float().abs().amax((1, 2)) / 448.0
        assert torch.equal(c.ks[page, 0, slot].cpu(), scale)
        want = (x.float() / scale[:, None, None]).clamp(-448, 448).to(FP8).view(torch.uint8)
        for got in (c.k, c.v):
            assert torch.equal(got.view(torch.uint8)[page, :, slot].cpu(), want)


def test_zeros_and_tiny_values(hip_lib):
    c = Cache([40], 2, 64, 16, 8)
    zeros = [torch.zeros((3, 2, 64), dtype=BF16, device=dev()) for _ in range(2)]
    c.append([3], [3], rows=zeros)
    assert bool((c.ks[c.table[0, 0].long(), :, 0] == 0).all())
    tiny = [torch.full((2, 2, 64), x, dtype=BF16, device=dev()) for x in (9.2e-41, -1.2e-38)]
    c.append([5], [2], rows=tiny)
    assert bool((c.ks[c.table[0, 0].long(), :, 0] > 0).all())
    c.append([6], [1], size=1e30)
    c.append([7], [1], rows=[torch.full((1, 2, 64), 3.38e38, dtype=BF16, device=dev())] * 2)


def test_infinities_and_nan_do_not_count(hip_lib):
    c = Cache([40], 2, 64, 16, 16)
    k, v = c.rows(9)
    k[2, 0, 5], k[4, 1, 9], v[3, 1, 2] = math.inf, -math.inf, math.nan
    v[8, 0] = math.nan
    c.append([9], [9], rows=(k, v))
    page = int(c.table[0, 0])
    codes = c.k.cpu().float()
    assert codes[page, 0, 2, 5] == 448 and codes[page, 1, 4, 9] == -448 and bool(torch.isfinite(c.ks[page]).all())
    assert bool(torch.isnan(c.v.cpu().float()[page, 0, 8]).all())
    c.append([12], [3], size=50.0)          # NaN codes stay NaN when the scale grows
    assert bool(torch.isnan(c.v.cpu().float()[page, 0, 8]).all())
    assert not bool(torch.isnan(c.v.cpu().float()[page, 0, 7]).any())


def test_values_stay_near(hip_lib):
    """A code is off by half a step, 2^-4 of the value or 2^-10 of the scale; a block whose scale grew m times
    has rounded m + 1 times, each time by half a step of a value that is near already."""
    c = Cache([64], 4, 128, 16, 16)
    rows = [c.append([i + 1], [1], size=1.0 + i % 16)[0] for i in range(64)]
    want = torch.cat(rows).cpu().double()
    got = kv.kv_cache_read(c.k, c.v, c.table, torch.tensor([64], dtype=torch.int32, device=dev()), tokens=64,
                           query_start=torch.tensor([0, 64], dtype=torch.int32, device=dev()), k_scale=c.ks, v_scale=c.vs)[0]
    scale = c.ks.cpu().double()[c.table[0].long().cpu()].squeeze(-1).repeat_interleave(16, 0)[:64]
    times = 17.0
    assert bool(((got.cpu().double() - want).abs() <= (times * 2.0 ** -4 * want.abs() + times * 2.0 ** -10 * scale[..., None]) * 1.1).all())
    # rows that were written in one call have rounded once
    c = Cache([64], 4, 128, 16, 16)
    k, _ = c.append([64], [64])
    got = kv.kv_cache_read(c.k, c.v, c.table, torch.tensor([64], dtype=torch.int32, device=dev()), tokens=64,
                           query_start=torch.tensor([0, 64], dtype=torch.int32, device=dev()), k_scale=c.ks, v_scale=c.vs)[0]
    scale = c.ks.cpu().double()[c.table[0].long().cpu()].squeeze(-1).repeat_interleave(16, 0)[:64]
    want = k.cpu().double()
    # (and once to bfloat16; 2^-22 for the quotient and the product)
    bound = (2.0 ** -4 + 2.0 ** -22) * want.abs() + 2.0 ** -10 * scale[..., None]
    assert bool(((got.cpu().double() - want).abs() <= bound + 2.0 ** -8 * (want.abs() + bound)).all())


def test_holes_and_short_tables(hip_lib):
    """Entries outside [0, pages) and positions beyond the table are skipped."""
    c = Cache([100, 60], 2, 64, 16, 16, width=5)
    c.table[0, 1], c.table[0, 3], c.table[1, 0] = -1, c.k.shape[0], 2147483647
    c.append([100, 60], [100, 60])
    c.append([101, 61])


def test_more_new_tokens_than_positions(hip_lib):
    """Rows in front of a sequence's first position are skipped."""
    c = Cache([20, 8], 2, 64, 8, 4)
    c.append([5, 8], [9, 3], size=1.0)


def test_rewritten_positions(hip_lib):
    """A length that went back: positions behind it are new rows again."""
    c = Cache([48], 2, 96, 16, 16)
    c.append([30], [30])
    c.append([20], [3], size=4.0)
    c.append([16], [1])
    c.append([17], [1], size=0.1)      # begins a block: its old scale does not count
    page = int(c.table[0, 1])
    assert bool((c.ks[page] < 0.1).all())


def test_strides_of_rows_and_broadcast_tables(hip_lib):
    g = torch.Generator().manual_seed(5)
    c = Cache([40, 40], 4, 64, 16, 8)
    qkv = torch.randn((24, 20, 64), generator=g).to(BF16).to(dev())
    c.append([11, 13], [11, 13], rows=(qkv[:, 8:12], qkv[:, 12:16]))
    odd = torch.randn((8, 4, 67), generator=g).to(BF16).to(dev())
    c.append([15, 17], [4, 4], rows=(odd[:, :, 1:65], odd[:, :, 3:]))


def test_append_in_a_graph_and_on_a_stream(hip_lib):
    c = Cache([64, 64], 2, 128, 16, 16)
    c.append([30, 20], [30, 20])
    lens = torch.tensor([30, 20], dtype=torch.int32, device=dev())
    k, v = c.rows(2)
    before = [t.clone() for t in (c.k, c.v, c.ks, c.vs)]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        kv.kv_cache_append(k, v, c.k, c.v, c.table, lens, k_scale=c.ks, v_scale=c.vs)
    for t, b in zip((c.k, c.v, c.ks, c.vs), before):
        assert torch.equal(t.view(torch.uint8), b.view(torch.uint8))
    for i in range(4):
        lens += 1
        k.copy_(torch.randn(k.shape, generator=c.g).to(BF16) * (1 + i))
        v.copy_(torch.randn(v.shape, generator=c.g).to(BF16) * (1 + i))
        torch.cuda.synchronize()
        want = ref.append(c.k, c.v, c.ks, c.vs, k, v, c.table, lens, None)
        graph.replay()
        torch.cuda.synchronize()
        c.equal(want)


# ---- reading back -----------------------------------------------------------------------------------

def check_read(k, v, table, lens, counts, ks, vs, dtype, spare=0, out=None):
    lens = torch.tensor(lens, dtype=torch.int32, device=dev())
    starts = None if counts is None else torch.tensor([0, *counts]).cumsum(0).to(torch.int32).to(dev())
    tokens = len(lens) if counts is None else sum(counts) + spare
    before = None if out is None else [t.clone() for t in out]
    got = kv.kv_cache_read(k, v, table, lens, query_start=starts, tokens=tokens, k_scale=ks, v_scale=vs, dtype=dtype, out=out)
    want = ref.read(k, v, ks, vs, table, lens, starts, tokens)
    half = torch.finfo(got[0].dtype).eps / 2
    # (a product rounded to 32 bits and once more; the least steps of the types)
    for i in range(2):
        w, g = want[i], got[i].cpu().double()
        if before is not None:
            w = torch.where(want[2][:, None, None], w, before[i].cpu().double())
        if ks is None:
            assert torch.equal(g, w)
        else:
            least = 2.0 ** -134 if dtype is BF16 else 2.0 ** -25
            assert bool(((g - w).abs() <= (half + 2.0 ** -23) * w.abs() + least).all())
    return got


@pytest.mark.parametrize("D", [16, 80, 128, 256])
@pytest.mark.parametrize("kind", ["bf16", "fp16", "head", "block"])
@pytest.mark.parametrize("layout", ["heads", "tokens"])
def test_read_kinds(hip_lib, D, kind, layout):
    g = torch.Generator().manual_seed(D)
    lens, Hkv, ps = [37, 0, 5, 130, 1], 3, 24
    c = Cache(lens, Hkv, D, ps, 8, layout=layout, seed=D)
    k, v, ks, vs = c.k, c.v, None, None
    if kind in ("bf16", "fp16"):
        t = BF16 if kind == "bf16" else F16
        k, v = (torch.randn(c.k.shape, generator=g).to(t).to(dev()) for _ in range(2))
        if layout == "tokens":
            k, v = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v))
        types = [t]
    else:
        for x in (k, v):
            x.copy_((torch.randn(c.k.shape, generator=g) * 100).clamp(-448, 448).to(FP8))
        ks, vs = (torch.rand(Hkv if kind == "head" else c.ks.shape, generator=g).to(dev()) + 0.1 for _ in range(2))
        types = [BF16, F16]
    for dtype in types:
        check_read(k, v, c.table, lens, lens, ks, vs, dtype)
        check_read(k, v, c.table, lens, [n // 2 for n in lens], ks, vs, dtype, spare=3)
        check_read(k, v, c.table, [37, 4, 5, 130, 1], None, ks, vs, dtype)       # (one without a page)
        room = [torch.full((sum(lens) + 4, Hkv + 1, D + 8), 5.0, dtype=dtype, device=dev()) for _ in range(2)]
        check_read(k, v, c.table, lens, lens, ks, vs, dtype, spare=4, out=[r[:, :Hkv, :D] for r in room])
        assert all(bool((r[:, Hkv] == 5).all() and (r[:, :, D:] == 5).all() and (r[-4:] == 5).all()) for r in room)


def test_read_holes(hip_lib):
    c = Cache([100, 60], 2, 64, 16, 16, width=5)
    c.append([100, 60], [100, 60])
    c.table[0, 1], c.table[1, 0] = -1, c.k.shape[0]
    check_read(c.k, c.v, c.table, [100, 60], [100, 60], c.ks, c.vs, BF16)
    check_read(c.k, c.v, c.table, [5, 60], [9, 3], c.ks, c.vs, BF16)        # more rows than positions


def test_nothing_to_read(hip_lib):
    c = Cache([10, 10], 2, 64, 16, 16)
    starts = torch.zeros(3, dtype=torch.int32, device=dev())
    lens = torch.tensor([3, 4], dtype=torch.int32, device=dev())
    k, v = kv.kv_cache_read(c.k, c.v, c.table, lens, query_start=starts, tokens=0, k_scale=c.ks, v_scale=c.vs)
    assert k.shape == v.shape == (0, 2, 64)
    k, v = kv.kv_cache_read(c.k, c.v, c.table, lens, query_start=starts, tokens=3, k_scale=c.ks, v_scale=c.vs)
    assert bool((k == 0).all() and (v == 0).all())


def test_a_backward_pass_is_an_error(hip_lib):
    c = Cache([10], 2, 64, 16, 4)
    wide = [torch.zeros(c.k.shape, dtype=BF16, device=dev(), requires_grad=True) for _ in range(2)]
    lens = torch.tensor([5], dtype=torch.int32, device=dev())
    k, v = kv.kv_cache_read(*wide, c.table, lens)
    with pytest.raises(RuntimeError, match="kv_cache_read has no backward"):
        (k.float().sum() + v.float().sum()).backward()
    with torch.no_grad():
        assert not kv.kv_cache_read(*wide, c.table, lens)[0].requires_grad


def test_refusals(hip_lib):
    c = Cache([10, 10], 2, 64, 16, 4)
    lens = torch.tensor([3, 4], dtype=torch.int32, device=dev())
    k, v = c.rows(2)
    pages = c.k.shape[0]
    for ks, vs in ((c.ks[:-1], c.vs), (c.ks[:, :, :3].contiguous(), c.vs[:, :, :3].contiguous()), (c.ks.double(), c.vs.double()),
                   (c.ks, None), (c.ks, c.vs[:, :, :2].contiguous()), (c.ks.transpose(1, 2), c.vs), (c.ks.cpu(), c.vs.cpu()),
                   (c.ks[:1].expand(pages, 2, 4), c.vs), (c.ks[0, :, 0].contiguous(), c.vs), (c.ks[:, :, :0], c.vs[:, :, :0])):
        with pytest.raises((ValueError, RuntimeError)):
            kv.kv_cache_append(k, v, c.k, c.v, c.table, lens, k_scale=ks, v_scale=vs)
        with pytest.raises((ValueError, RuntimeError)):
            kv.kv_cache_read(c.k, c.v, c.table, lens, k_scale=ks, v_scale=vs)
    wide = [torch.zeros((pages, 2, 16, 64), dtype=BF16, device=dev()) for _ in range(2)]
    with pytest.raises(RuntimeError):
        kv.kv_cache_append(k, v, *wide, c.table, lens, k_scale=c.ks, v_scale=c.vs)
    with pytest.raises(RuntimeError):
        kv.kv_cache_read(*wide, c.table, lens, k_scale=c.ks, v_scale=c.vs)
    starts = torch.tensor([0, 1, 2], dtype=torch.int32, device=dev())
    for bad in (dict(query_start=starts), dict(tokens=3), dict(dtype=torch.float32), dict(query_start=starts.long(), tokens=2),
                dict(query_start=starts, tokens=-1), dict(out=(k, v[:1])), dict(out=(k, v.half())),
                dict(out=(k, torch.zeros((2, 2, 68), dtype=BF16, device=dev())[..., :64]))):
        with pytest.raises(ValueError):
            kv.kv_cache_read(c.k, c.v, c.table, lens, k_scale=c.ks, v_scale=c.vs, **bad)
    with pytest.raises(RuntimeError):
        kv.kv_cache_read(c.k, c.v, c.table, lens, k_scale=c.ks, v_scale=c.vs, out=(k, v[:1].expand(2, 2, 64)))
