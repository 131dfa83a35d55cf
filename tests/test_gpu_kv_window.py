"""GPU tests of one new token's attention over a window and the first positions, and over 8-bit caches with a scale for
each block of positions."""
from __future__ import annotations

import math

import pytest
import torch

import attention_reference as aref
import kv_reference as ref
from vkernels_amd import kv_cache as kv

pytestmark = pytest.mark.gpu

BF16, F16, FP8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def dev():
    return torch.device("cuda", 0)


class Setup:
    """A cache with the sequences' pages scattered over it; what is no position is NaN, scales included.  block 0: of
    the queries' type; -1: 8 bits with a scale for each head."""

    def __init__(self, lens, Hkv, G, D, ps, block, *, q=BF16, layout="heads", seed=1, peak=2.0, tokens=None, spread=0.7):
        g = torch.Generator().manual_seed(seed)
        self.B, self.Hkv, self.G, self.D, self.ps, self.block = len(lens), Hkv, G, D, ps, block
        need = [-(-n // ps) for n in lens]
        pages = sum(need) + 2
        order = torch.randperm(pages, generator=g)
        self.table = torch.full((self.B, max(1, max(need))), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n].to(torch.int32)
            at += n
        caches, scales = [], []
        for _ in range(2):
            c = torch.full((pages, Hkv, ps, D), math.nan)
            s = torch.full((pages, Hkv, max(1, ps // block) if block > 0 else 1), math.nan)
            for b, n in enumerate(lens):
                j = torch.arange(n)
                c[self.table[b].long()[j // ps], :, j % ps] = torch.randn((n, Hkv, D), generator=g)
                if block > 0:
                    used = torch.arange(0, n, block)
                    s[self.table[b].long()[used // ps], :, used % ps // block] = \
                        torch.exp(spread * torch.randn((len(used), Hkv), generator=g)) / 60
            caches.append((c * 60 if block else c).to(FP8 if block else q))
            scales.append(s if block > 0 else torch.rand(Hkv, generator=g) * 0.02 + 0.01 if block else None)
        if layout == "tokens":
            caches = [c.transpose(1, 2).contiguous().transpose(1, 2) for c in caches]
        self.k, self.v = (c.to(dev()) for c in caches)
        self.k_scale, self.v_scale = (None if s is None else s.to(dev()) for s in scales)
        self.lens = torch.tensor(lens, dtype=torch.int32, device=dev())
        self.table = self.table.to(dev())
        rows = self.B if tokens is None else tokens
        self.q = (peak * torch.randn((rows, Hkv * G, D), generator=g)).to(q).to(dev())
        self.sinks = torch.randn(Hkv * G, generator=g).to(dev())

    def check(self, *, counted=False, sinks=False, what="", **kw):
        sums = before = None
        if counted:
            sums = torch.rand((self.B, self.Hkv, self.table.shape[1] * self.ps + 3), device=dev())
            before = sums.clone()
        both = dict(kw, sinks=self.sinks if sinks else None, k_scale=self.k_scale, v_scale=self.v_scale)
        out, lse = kv.paged_attention(self.q, self.k, self.v, self.table, self.lens, weight_sums=sums, return_lse=True, **both)
        want = aref.attention(self.q, self.k, self.v, self.table, self.lens, **dict(both, scale=kw.get("scale", self.D ** -0.5)))
        ref.assert_attention(out, lse, want, self.q.dtype, what)
        if counted:
            ref.assert_sums(sums, before, want, what)
        return out, lse, sums


LENGTHS = [0, 1, 15, 16, 17, 31, 33, 127, 128, 129, 300, 700]


@pytest.mark.parametrize("window", [1, 2, 16, 100, 128, 300])
@pytest.mark.parametrize("first", [0, 1, 4, 16, 100, 127, 128, 129, 250, 100000])
@pytest.mark.parametrize("ps", [16, 24])
def test_windows_with_first_positions(hip_lib, window, first, ps):
    Setup(LENGTHS, 2, 4, 64, ps, 0, seed=window + first).check(counted=True, sinks=True, window=window, keep_first=first)


@pytest.mark.parametrize("lens", [[9000], [2500, 0, 3, 1400, 1101, 40]])
@pytest.mark.parametrize("window,first", [(1030, 4), (1500, 700), (2047, 129), (700, 1000), (64, 2000), (1, 1)])
@pytest.mark.parametrize("G", [8, 33])
def test_long_sequences(hip_lib, lens, window, first, G):
    """Shares of several workgroups that begin among the first positions, in the window, or at its edge."""
    Setup(lens, 2, G, 64, 16, 0, seed=window).check(counted=True, window=window, keep_first=first)


def test_first_positions_without_a_window_change_nothing(hip_lib):
    s = Setup([300, 40, 1200], 2, 8, 128, 16, 0)
    args = s.q, s.k, s.v, s.table, s.lens
    plain = kv.paged_attention(*args)
    assert torch.equal(plain, kv.paged_attention(*args, keep_first=4))
    assert torch.equal(plain, kv.paged_attention(*args, keep_first=4, window=2 ** 31 - 1))
    assert torch.equal(plain, kv.paged_attention(*args, keep_first=2 ** 40, window=2 ** 40))
    assert torch.equal(kv.paged_attention(*args, window=100), kv.paged_attention(*args, window=100, keep_first=0))


def test_what_lies_between_may_be_anything(hip_lib):
    """Positions between the first ones and the window are NaN, or have no page."""
    for block, ps in ((0, 16), (0, 24), (8, 16), (8, 24)):
        s = Setup([900, 333], 2, 4, 64, ps, block, seed=ps)
        for b, n in enumerate((900, 333)):
            j = torch.arange(5, n - 150, device=dev())
            for c in (s.k, s.v):
                c.view(torch.uint8 if block else torch.int16)[s.table[b].long()[j // ps], :, j % ps] = 0x7F if block else 0x7FFF
            s.table[b, 100 // ps + 1:(n - 150) // ps] = -7
        out, lse, _ = s.check(window=150, keep_first=5)
        assert bool(torch.isfinite(out).all() and torch.isfinite(lse).all())


@pytest.mark.parametrize("D", [16, 48, 64, 80, 128, 160, 192, 240, 256])
@pytest.mark.parametrize("q", [BF16, F16])
@pytest.mark.parametrize("ps,block", [(16, 16), (16, 1), (32, 8), (64, 32), (24, 24), (24, 6), (5, 1)])
def test_block_scales(hip_lib, D, q, ps, block):
    Setup([0, 1, 15, 33, 130, 700], 2, 4, D, ps, block, q=q, seed=D + ps).check(counted=True, sinks=True)


@pytest.mark.parametrize("lens", [[9000], [1, 2500, 0, 3001, 17]])
@pytest.mark.parametrize("Hkv,G", [(1, 1), (2, 8), (1, 24), (3, 40)])
@pytest.mark.parametrize("layout", ["heads", "tokens"])
def test_block_scales_of_long_sequences(hip_lib, lens, Hkv, G, layout):
    Setup(lens, Hkv, G, 128, 32, 16, seed=G, layout=layout).check(counted=True)


@pytest.mark.parametrize("q", [BF16, F16])
def test_block_scales_far_apart(hip_lib, q):
    """Scales over ten powers of ten, and blocks of scale 0."""
    s = Setup([400, 1500], 2, 4, 64, 16, 8, q=q, spread=0.1)
    for t in (s.k_scale, s.v_scale):
        t[::3] *= 1e-7
        t[1::7] = 0.0
    s.v_scale[::5] *= 1000.0
    s.check(softcap=30.0)


def test_equal_block_scales_are_a_head_scale(hip_lib):
    s = Setup([700, 33, 2000], 3, 5, 128, 16, -1)
    args = s.q, s.k, s.v, s.table, s.lens
    want = kv.paged_attention(*args, k_scale=s.k_scale, v_scale=s.v_scale).cpu().double()
    wide = [t[None, :, None].expand(s.k.shape[0], 3, 4).contiguous() for t in (s.k_scale, s.v_scale)]
    got = kv.paged_attention(*args, k_scale=wide[0], v_scale=wide[1]).cpu().double()
    # (each is its own rounding, half a step, from values that differ by 32-bit roundings)
    assert bool(((got - want).abs() <= 2.0 ** -7 * want.abs() + 2.0 ** -16).all())


def test_append_then_attend_in_a_graph(hip_lib):
    """A decode step with block scales, a window and first positions, captured and replayed as lengths grow."""
    s = Setup([200, 340], 2, 4, 128, 16, 16)
    s.table = torch.cat([s.table, torch.full((2, 2), -1, dtype=torch.int32, device=dev())], 1)
    s.table[0, 13], s.table[0, 14], s.table[1, 22] = s.k.shape[0] - 1, -1, s.k.shape[0] - 2
    spare = sorted(set(range(s.k.shape[0])) - set(s.table.flatten().tolist()))
    for b, i in ((0, 13), (1, 22)):
        if spare:
            s.table[b, i] = spare.pop()
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn((2, 2, 128), generator=g).to(BF16).to(dev()) for _ in range(2))

    def step():
        kv.kv_cache_append(k, v, s.k, s.v, s.table, s.lens, k_scale=s.k_scale, v_scale=s.v_scale)
        return kv.paged_attention(s.q, s.k, s.v, s.table, s.lens, window=100, keep_first=4, k_scale=s.k_scale,
                                  v_scale=s.v_scale, return_lse=True)

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = step()
    for i in range(4):
        s.lens += 1
        k.copy_(torch.randn(k.shape, generator=g).to(BF16) * (i + 1))
        graph.replay()
        torch.cuda.synchronize()
        want = aref.attention(s.q, s.k, s.v, s.table, s.lens, scale=128 ** -0.5, window=100, keep_first=4, k_scale=s.k_scale,
                              v_scale=s.v_scale)
        ref.assert_attention(out, lse, want, BF16, f"replay {i}")


def test_refusals(hip_lib):
    s = Setup([40], 2, 4, 64, 16, 8)
    args = s.q, s.k, s.v, s.table, s.lens
    both = dict(k_scale=s.k_scale, v_scale=s.v_scale)
    with pytest.raises(ValueError):
        kv.paged_attention(*args, window=3, keep_first=-1, **both)
    for bad in (dict(k_scale=s.k_scale[:, :, 0], v_scale=s.v_scale[:, :, 0]), dict(k_scale=s.k_scale, v_scale=None),
                dict(k_scale=s.k_scale[:-1], v_scale=s.v_scale), dict(k_scale=s.k_scale.half(), v_scale=s.v_scale.half()),
                dict(k_scale=s.k_scale.repeat(1, 1, 2)[:, :, :3].contiguous(), v_scale=s.v_scale.repeat(1, 1, 2)[:, :, :3].contiguous())):
        with pytest.raises((ValueError, RuntimeError)):
            kv.paged_attention(*args, **bad)
