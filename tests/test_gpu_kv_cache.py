"""GPU tests of the key-value cache's operators against their definitions in 64 bits: head layouts, types,
lengths from nothing to several shares of a workgroup, pages of any size, windows, capped scores,
sinks, pages that are not there, what lies beyond a length, strides, streams and graphs."""
from __future__ import annotations

import math

import pytest
import torch

import kv_reference as ref
from vkernels_amd import kv_cache as kv

pytestmark = pytest.mark.gpu

BF16, F16, FP8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def dev():
    return torch.device("cuda", 0)


class Setup:
    """A cache with the sequences' pages scattered over it, everything that is not a position NaN."""

    def __init__(self, lens, Hkv, G, D, ps, *, cache=BF16, q=BF16, layout="heads", seed=1, peak=2.0, width=None,
                 spare=2):
        g = torch.Generator().manual_seed(seed)
        self.B, self.Hkv, self.G, self.D, self.ps = len(lens), Hkv, G, D, ps
        need = [-(-n // ps) for n in lens]
        width = max(1, max(need)) if width is None else width
        pages = sum(need) + spare
        order = torch.randperm(pages, generator=g)
        self.table = torch.full((self.B, width), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n].to(torch.int32)
            at += n
        self.lens = torch.tensor(lens, dtype=torch.int32)
        caches = []
        for _ in range(2):
            c = torch.full((pages, Hkv, ps, D), math.nan)
            for b, n in enumerate(lens):
                j = torch.arange(n)
                c[self.table[b].long()[j // ps], :, j % ps] = torch.randn((n, Hkv, D), generator=g)
            caches.append(c)
        self.k_scale = self.v_scale = None
        if cache == FP8:
            self.k_scale, self.v_scale = (torch.rand(Hkv, generator=g) * 0.02 + 0.01 for _ in range(2))
            caches = [c * 60 for c in caches]
        caches = [c.to(cache) for c in caches]
        if layout == "tokens":
            caches = [c.transpose(1, 2).contiguous().transpose(1, 2) for c in caches]
        self.k, self.v = (c.to(dev()) for c in caches)
        if layout == "tokens":
            assert self.k.stride(1) == D or 1 in (Hkv, ps)      # (a single head or position has any stride)
        self.q = (peak * torch.randn((self.B, Hkv * G, D), generator=g)).to(q).to(dev())
        self.sinks = torch.randn(Hkv * G, generator=g)
        self.scale = D ** -0.5
        self.to_device()

    def to_device(self):
        for name in ("table", "lens", "k_scale", "v_scale", "sinks"):
            t = getattr(self, name)
            setattr(self, name, None if t is None else t.to(dev()))

    def args(self):
        return self.q, self.k, self.v, self.table, self.lens

    def check(self, *, counted=False, what="", sinks=False, **kw):
        sums = before = None
        if counted:
            sums = torch.rand((self.B, self.Hkv, self.table.shape[1] * self.ps + 3), device=dev())
            before = sums.clone()
        both = dict(kw, sinks=self.sinks if sinks else None, k_scale=self.k_scale, v_scale=self.v_scale)
        out, lse = kv.paged_attention(*self.args(), weight_sums=sums, return_lse=True, **both)
        want = ref.attention(*self.args(), **dict(both, scale=kw.get("scale", self.scale)))
        ref.assert_attention(out, lse, want, self.q.dtype, what)
        if counted:
            ref.assert_sums(sums, before, want, what)
        return out, lse, sums


# ---- attention ----------------------------------------------------------------------------------

# one wavefront's tile is 32 positions, a workgroup's 128; calls that see more than 1024 are shared out
LENGTHS = [0, 1, 15, 16, 17, 31, 33, 127, 128, 129, 300]


@pytest.mark.parametrize("D", [16, 48, 64, 80, 96, 112, 128, 160, 192, 240, 256])
@pytest.mark.parametrize("cache,q", [(BF16, BF16), (F16, F16), (FP8, BF16), (FP8, F16)])
def test_head_widths_and_types(hip_lib, D, cache, q):
    for lens, ps in ((LENGTHS, 16), ([700, 1, 0, 1033], 24)):
        Setup(lens, 2, 4, D, ps, cache=cache, q=q, seed=D).check(counted=True, what=f"D {D} ps {ps}")


@pytest.mark.parametrize("Hkv,G", [(1, 1), (3, 1), (2, 2), (1, 7), (2, 8), (1, 15), (2, 16), (1, 17), (2, 33), (1, 70)])
@pytest.mark.parametrize("long", [False, True])
def test_head_layouts(hip_lib, Hkv, G, long):
    lens = [650, 5, 1300] if long else [40, 0, 130]
    Setup(lens, Hkv, G, 64, 16, seed=Hkv * 100 + G).check(counted=True, sinks=True)


@pytest.mark.parametrize("Hkv,G,D", [(1, 24, 64), (3, 40, 64), (1, 128, 128), (1, 250, 64), (1, 256, 192), (1, 260, 64), (2, 272, 16), (1, 273, 64)])
@pytest.mark.parametrize("lens,window", [([9000], 0), ([1, 2500, 0, 3001, 17], 0), ([5000, 1300, 4999], 2000), ([40, 3, 1030], 1025)])
def test_head_tiles_that_share_a_stream(hip_lib, Hkv, G, D, lens, window):
    """Up to 16 tiles of heads each have workgroups of their own (a number that does not divide the grid
    among them, and one tile more than that)."""
    Setup(lens, Hkv, G, D, 16, seed=G + len(lens)).check(counted=True, sinks=True, window=window)


@pytest.mark.parametrize("ps", [1, 2, 3, 7, 8, 16, 17, 24, 32, 48, 64, 100, 256, 1000])
@pytest.mark.parametrize("layout", ["heads", "tokens"])
def test_page_sizes_and_layouts(hip_lib, ps, layout):
    Setup([ps, ps + 1, max(1, ps - 1), 3 * ps, 1201], 2, 3, 64, ps, layout=layout, seed=ps).check(counted=True)
    Setup([200, 31, 77], 2, 3, 80, ps, layout=layout, seed=ps, cache=FP8).check(counted=True)


@pytest.mark.parametrize("window", [1, 15, 16, 17, 100, 128, 129, 500, 5000])
@pytest.mark.parametrize("ps", [16, 10])
def test_windows(hip_lib, window, ps):
    Setup([1, 16, 17, 129, 500, 1100, 0], 2, 4, 64, ps, seed=window).check(window=window, counted=True)


@pytest.mark.parametrize("cache", [BF16, FP8])
@pytest.mark.parametrize("softcap,scale", [(20.0, None), (0.5, 1.0), (50.0, 0.003), (0.0, 0.7), (5.0, -0.1)])
def test_capped_and_scaled_scores(hip_lib, softcap, scale, cache):
    s = Setup([1, 40, 777], 2, 4, 96, 16, seed=7, cache=cache)
    kw = {} if scale is None else {"scale": scale}
    s.check(softcap=softcap, counted=True, sinks=True, **kw)


def test_many_sequences_share_the_workgroups(hip_lib):
    """More sequences than a workgroup has threads, ragged, some empty: several items a workgroup, items
    over several workgroups, and the scan over more than one sequence a thread."""
    g = torch.Generator().manual_seed(3)
    lens = torch.randint(0, 90, (700,), generator=g).tolist()
    lens[0], lens[350], lens[699] = 900, 2500, 1111
    Setup(lens, 1, 2, 64, 16, seed=11).check(counted=True)


@pytest.mark.parametrize("L", [513, 1024, 1025, 4096, 20000])
def test_one_long_sequence(hip_lib, L):
    for peak in (0.3, 6.0):
        Setup([L], 2, 4, 128, 64, seed=L, peak=peak).check(counted=True, sinks=True)


def test_a_bound_above_the_lengths_changes_nothing_but_the_split(hip_lib):
    """Short sequences in a call whose max_len says they might be long (a captured graph's), and lengths
    that max_len cuts."""
    s = Setup([100, 3, 0, 64], 2, 4, 64, 16, width=400)
    s.check(counted=True)
    s.check(max_len=130, counted=True)
    s.check(max_len=50, counted=True)
    s.check(max_len=0, counted=True)


def test_pages_that_are_not_there(hip_lib):
    """Entries outside [0, pages) leave their positions out, whole sequences included."""
    for ps in (16, 12):
        for lens in ([200, 200, 90, 200], [1300, 700, 90, 40]):
            s = Setup(lens, 2, 4, 64, ps, seed=5)
            table = s.table.clone()
            table[0, 0] = -1
            table[0, 3] = s.k.shape[0]
            table[1, :] = -7
            table[2, -1] = 2 ** 31 - 1
            table[3, 1::2] = -1
            s.table = table
            out, lse, _ = s.check(counted=True)
            assert torch.all(out[1] == 0) and torch.all(lse[1] == -math.inf)
            out, lse, _ = s.check(sinks=True)
            assert torch.all(out[1] == 0) and torch.equal(lse[1].cpu(), s.sinks.cpu())


def test_scores_of_infinity_and_nan(hip_lib):
    """What is stored at positions that count is computed with as the definition says: a score of -inf
    gets no weight, a row of nothing else is 0, +inf or NaN make the row NaN; other rows are not
    touched."""
    for n in (40, 1200):
        s = Setup([n, n, n, n], 1, 1, 64, 16, seed=9)
        s.q.zero_()
        s.q[:, :, 0] = 1.0
        page = s.table.long()
        s.k[page[0, 0], 0, 3, 0] = -math.inf                   # one position of weight 0
        s.k[page[1]] = 0.0
        s.k[page[1], :, :, 0] = -math.inf                      # all of them
        s.k[page[2, 1], 0, 2, 0] = math.inf
        s.v[page[3, 1], 0, 5, 7] = math.nan                    # a value: its column alone
        out, lse, sums = s.check()
        assert torch.all(out[1] == 0) and torch.all(lse[1] == -math.inf)
        assert torch.all(torch.isnan(out[2]))
        assert torch.isnan(out[3, 0, 7]) and int(torch.isnan(out[3]).sum()) == 1
        lowest = torch.finfo(BF16).min
        s.k[page[0], :, :, 0] = lowest                         # all alike, and the lowest there is
        s.k[page[0, 2], 0, 1, 0] = 0.0
        out, _, _ = s.check()
        assert torch.equal(out[0, 0], s.v[page[0, 2], 0, 1])


@pytest.mark.parametrize("cache", [BF16, F16])
def test_an_infinite_value_stays_in_its_column(hip_lib, cache):
    for n in (40, 1200):
        s = Setup([n, n], 1, 4, 64, 16, seed=10, cache=cache, q=cache)
        want = kv.paged_attention(*s.args())
        s.v[s.table[0, 1].long(), 0, 2, 9] = math.inf
        got = kv.paged_attention(*s.args())
        assert not bool(torch.isfinite(got[0, :, 9]).any())
        got[0, :, 9] = want[0, :, 9]
        assert torch.equal(got, want)


def test_large_scores_and_rising_maxima(hip_lib):
    """The reference of the exponentials moves many times, in both directions of the scores' order."""
    for flip in (False, True):
        s = Setup([1500, 600], 1, 4, 64, 16, seed=4)
        ramp = torch.linspace(-300, 300, 1500, device=dev())
        ramp = ramp.flip(0) if flip else ramp
        s.q.zero_()
        s.q[:, :, 0] = torch.tensor([8.0, 1.0, 0.1, -2.0], device=dev()).to(BF16)
        for b in range(2):
            n = int(s.lens[b])
            j = torch.arange(n, device=dev())
            s.k[s.table[b].long()[j // 16], 0, j % 16, 0] = ramp[:n].to(BF16)
        s.check(counted=True)


def test_strided_queries_tables_and_sums(hip_lib):
    s = Setup([100, 1140, 3], 2, 4, 64, 16, seed=6)
    want, want_lse, _ = s.check()
    fused = torch.randn((3, 8 + 4, 64), device=dev()).to(BF16)       # queries as part of a fused projection
    fused[:, :8] = s.q
    s.q = fused[:, :8]
    wide = torch.full((3, s.table.shape[1] + 5), 10 ** 6, dtype=torch.int32, device=dev())
    wide[:, 2:-3] = s.table
    s.table = wide[:, 2:-3]
    n = s.table.shape[1] * 16
    out, lse = kv.paged_attention(*s.args(), return_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    odd = torch.empty(3 * 8 * 64 + 1, dtype=BF16, device=dev())[1:].view(3, 8, 64)     # rows off 16 bytes
    odd.copy_(s.q)
    assert torch.equal(kv.paged_attention(odd, *s.args()[1:]), want)
    turned = s.q.transpose(1, 2).contiguous().transpose(1, 2)                          # D not contiguous
    assert torch.equal(kv.paged_attention(turned, *s.args()[1:]), want)
    plain = torch.zeros((3, 2, n), device=dev())
    kv.paged_attention(*s.args(), weight_sums=plain)
    big = torch.zeros((3, 5, n + 11), device=dev())
    kv.paged_attention(*s.args(), weight_sums=big[:, 1:4:2, 1:])
    assert torch.equal(big[:, 1:4:2, 1:1 + n], plain) and float(big[:, ::2].abs().sum()) == 0
    assert float(big[:, :, 0].abs().sum()) == 0 and float(big[:, :, 1 + n:].abs().sum()) == 0
    out = torch.full_like(want, math.nan)
    assert kv.paged_attention(*s.args(), out=out) is out and torch.equal(out, want)


def test_broadcast_tables_queries_and_rows(hip_lib):
    """One row of the table for all sequences (a shared prompt), one query for all heads, one key for all heads."""
    s = Setup([1500], 2, 4, 64, 16, seed=16)
    table, lens = s.table.expand(3, -1), torch.tensor([1500, 0, 77], dtype=torch.int32, device=dev())
    q = torch.randn((3, 1, 64), device=dev()).to(BF16)
    want = kv.paged_attention(q.repeat(1, 8, 1), s.k, s.v, table.contiguous(), lens)
    assert torch.equal(kv.paged_attention(q.expand(-1, 8, -1), s.k, s.v, table, lens), want)
    few = Setup([40, 17, 3], 2, 1, 64, 16, seed=3)
    row = torch.randn((3, 1, 64), device=dev()).to(BF16).expand(-1, 2, -1)
    after = ref.append(few.k, few.v, row, -row, few.table, few.lens, None, None, None)
    kv.kv_cache_append(row, -row, few.k, few.v, few.table, few.lens)
    assert all(torch.equal(a.cpu().view(torch.int16), b.view(torch.int16)) for a, b in zip((few.k, few.v), after))
    with pytest.raises(ValueError):      # sums that heads would share cannot be added to
        kv.paged_attention(*s.args(), weight_sums=torch.zeros((1, 1, 1504), device=dev()).expand(-1, 2, -1))


def test_results_do_not_depend_on_the_run(hip_lib):
    s = Setup([900, 30, 2222, 0, 511], 2, 8, 128, 16, seed=8)
    runs = []
    for _ in range(4):
        sums = torch.zeros((5, 2, s.table.shape[1] * 16), device=dev())
        out, lse = kv.paged_attention(*s.args(), weight_sums=sums, return_lse=True)
        runs.append((out.view(torch.int16), lse, sums))
    for r in runs[1:]:
        assert all(torch.equal(x, y) for x, y in zip(r, runs[0]))


def test_offsets_beyond_32_bits(hip_lib):
    """A cache of more than 2^32 bytes and 2^31 elements, pages at its two ends."""
    pages, Hkv, ps, D = 17000, 8, 128, 128
    k = torch.zeros((pages, Hkv, ps, D), dtype=BF16, device=dev())
    v = torch.zeros_like(k)
    assert k.numel() > 2 ** 31
    table = torch.tensor([[pages - 1, 0, pages - 2, pages // 2, 1, 16384]], dtype=torch.int32, device=dev())
    g = torch.Generator(device=dev()).manual_seed(1)
    for p in table[0].tolist():
        k[p] = torch.randn((Hkv, ps, D), device=dev(), generator=g).to(BF16)
        v[p] = torch.randn((Hkv, ps, D), device=dev(), generator=g).to(BF16)
    lens = torch.tensor([6 * ps - 5], dtype=torch.int32, device=dev())
    q = torch.randn((1, Hkv, D), device=dev(), generator=g).to(BF16)
    out, lse = kv.paged_attention(q, k, v, table, lens, return_lse=True)
    few = table[0].long()
    small = torch.arange(6, dtype=torch.int32, device=dev())[None]
    want = ref.attention(q, k[few], v[few], small, lens, scale=D ** -0.5)
    ref.assert_attention(out, lse, want, BF16)
    rows = torch.randn((1, Hkv, D), device=dev(), generator=g).to(BF16)
    lens += 1
    kv.kv_cache_append(rows, -rows, k, v, table, lens)
    assert torch.equal(k[16384, :, ps - 5], rows[0]) and torch.equal(v[16384, :, ps - 5], -rows[0])
    sums = torch.rand((1, Hkv, 6 * ps), device=dev(), generator=g)
    want = ref.evict(k[few], v[few], small, lens, sums, sums, 200, 2, 30)
    new_lens, kept = kv.kv_cache_evict(k, v, table, lens, sums, 200, keep_first=2, keep_last=30)
    assert torch.equal(kept.cpu(), torch.from_numpy(want[4])) and torch.equal(k[few].cpu(), want[0])
    assert torch.equal(v[few].cpu(), want[1]) and torch.equal(sums.cpu(), want[2])


# ---- append -----------------------------------------------------------------------------------------

@pytest.mark.parametrize("cache,q", [(BF16, BF16), (F16, F16), (FP8, BF16), (FP8, F16)])
@pytest.mark.parametrize("ps,layout", [(16, "heads"), (7, "tokens")])
@pytest.mark.parametrize("new", [None, [3, 0, 20, 1, 0, 0, 65, 2]])
@pytest.mark.parametrize("D", [16, 80, 128])
def test_append(hip_lib, cache, q, ps, layout, new, D):
    lens = [5, 0, 20, 1, 9, 33, 100, 17]
    s = Setup(lens, 3, 1, D, ps, cache=cache, q=q, layout=layout, seed=D + ps)
    starts = None if new is None else torch.tensor([0] + new).cumsum(0).to(torch.int32).to(dev())
    n = 8 if new is None else sum(new)
    g = torch.Generator().manual_seed(2)
    k, v = (torch.randn((n, 3, D), generator=g).to(q).to(dev()) for _ in range(2))
    if cache == FP8:      # beyond the range, subnormal codes, ties, NaN and infinity
        k[0, 0, :8] = torch.tensor([1e4, -1e4, math.inf, -math.inf, math.nan, 1e-6, -1e-6, 0.0]).to(q).to(dev())
        k[-1] *= 1e-3
        s.k_scale[1], s.v_scale[1] = 1.0, 1.0
    want = ref.append(s.k, s.v, k, v, s.table, s.lens, starts, s.k_scale, s.v_scale)
    kv.kv_cache_append(k, v, s.k, s.v, s.table, s.lens, query_start=starts, k_scale=s.k_scale, v_scale=s.v_scale)
    for got, exp in zip((s.k, s.v), want):
        word = torch.uint8 if cache == FP8 else torch.int16
        got, exp = got.cpu().contiguous(), exp.contiguous()
        same = (got.view(word) == exp.view(word)) | (torch.isnan(got.float()) & torch.isnan(exp.float()))
        assert bool(same.all())


def test_append_skips_what_has_no_place(hip_lib):
    s = Setup([40, 40, 40], 2, 1, 64, 16, seed=3)
    s.table[0, 2] = -1
    s.table[1, 2] = s.k.shape[0]
    s.lens[2] = 1000                          # beyond the table
    before = s.k.clone()
    rows = torch.ones((3, 2, 64), dtype=BF16, device=dev())
    kv.kv_cache_append(rows, rows, s.k, s.v, s.table, s.lens)
    assert torch.equal(s.k.view(torch.int16), before.view(torch.int16))


def test_append_from_slices_of_a_fused_projection(hip_lib):
    s = Setup([40, 17, 3], 2, 1, 64, 16, seed=3)
    fused = torch.randn((3, 8 + 2 + 2, 64), device=dev()).to(BF16)
    want = ref.append(s.k, s.v, fused[:, 8:10], fused[:, 10:], s.table, s.lens, None, None, None)
    kv.kv_cache_append(fused[:, 8:10], fused[:, 10:], s.k, s.v, s.table, s.lens)
    assert all(torch.equal(a.cpu().view(torch.int16), b.view(torch.int16)) for a, b in zip((s.k, s.v), want))


def test_calls_without_sequences_or_tokens(hip_lib):
    s = Setup([40, 3], 2, 4, 64, 16)
    before = s.k.clone()
    none = torch.zeros((0, 2, 64), dtype=BF16, device=dev())
    kv.kv_cache_append(none, none, s.k, s.v, s.table[:0], s.lens[:0])
    kv.kv_cache_append(none, none, s.k, s.v, s.table, s.lens, query_start=torch.zeros(3, dtype=torch.int32, device=dev()))
    out, lse = kv.paged_attention(s.q[:0], s.k, s.v, s.table[:0], s.lens[:0], return_lse=True)
    assert out.shape == (0, 8, 64) and lse.shape == (0, 8)
    new_lens, kept = kv.kv_cache_evict(s.k, s.v, s.table[:0], s.lens[:0], torch.zeros((0, 2, 48), device=dev()), 8)
    assert new_lens.shape == (0,) and kept.shape == (0, 2, 8)
    assert torch.equal(s.k.view(torch.int16), before.view(torch.int16))


def test_append_of_a_stretch_of_the_tokens(hip_lib):
    """query_start that begins behind token 0 and ends before the last: the tokens outside go nowhere."""
    s = Setup([40, 20, 9], 2, 1, 64, 16, seed=5)
    rows = torch.randn((30, 2, 64), device=dev()).to(BF16)
    starts = torch.tensor([6, 14, 14, 23], dtype=torch.int32, device=dev())
    want = ref.append(s.k, s.v, rows, -rows, s.table, s.lens, starts.cpu(), None, None)
    kv.kv_cache_append(rows, -rows, s.k, s.v, s.table, s.lens, query_start=starts)
    assert all(torch.equal(a.cpu().view(torch.int16), b.view(torch.int16)) for a, b in zip((s.k, s.v), want))


def test_append_many_sequences_of_few_tokens(hip_lib):
    """More sequences than the search's 64 candidates, many of them without a token."""
    g = torch.Generator().manual_seed(1)
    new = (torch.randint(0, 5, (5000,), generator=g) - 2).clamp(min=0)
    lens = new + torch.randint(0, 9, (5000,), generator=g)
    s = Setup(lens.tolist(), 1, 1, 16, 16, seed=3)
    starts = torch.cat([torch.zeros(1, dtype=torch.long), new.cumsum(0)]).to(torch.int32).to(dev())
    k = torch.randn((int(new.sum()), 1, 16), generator=g).to(BF16).to(dev())
    want = ref.append(s.k, s.v, k, -k, s.table, s.lens, starts.cpu(), None, None)
    kv.kv_cache_append(k, -k, s.k, s.v, s.table, s.lens, query_start=starts)
    assert all(torch.equal(a.cpu().view(torch.int16), b.view(torch.int16)) for a, b in zip((s.k, s.v), want))


# ---- eviction --------------------------------------------------------------------------------------

def _check_evict(s, sums, budget, first, last, in_place=False):
    out = sums if in_place else torch.full_like(sums, 7.0)
    want = ref.evict(s.k, s.v, s.table, s.lens, sums, out, budget, first, last)
    new_lens, kept = kv.kv_cache_evict(s.k, s.v, s.table, s.lens, sums, budget, keep_first=first, keep_last=last,
                                       sums_out=None if in_place else out)
    word = torch.uint8 if s.k.element_size() == 1 else torch.int16
    assert torch.equal(kept.cpu(), torch.from_numpy(want[4]))
    assert torch.equal(new_lens.cpu(), torch.from_numpy(want[3]).to(torch.int32))
    assert torch.equal(s.k.cpu().contiguous().view(word), want[0].contiguous().view(word))
    assert torch.equal(s.v.cpu().contiguous().view(word), want[1].contiguous().view(word))
    assert torch.equal(out.cpu().view(torch.int32), want[2].view(torch.int32))


@pytest.mark.parametrize("cache,D", [(BF16, 64), (F16, 80), (FP8, 16), (FP8, 256), (BF16, 256)])
@pytest.mark.parametrize("budget,first,last", [(1, 0, 0), (1, 0, 1), (33, 4, 8), (64, 64, 0), (64, 0, 64), (200, 3, 100),
                                               (699, 0, 0)])
@pytest.mark.parametrize("in_place", [False, True])
def test_evict(hip_lib, cache, D, budget, first, last, in_place):
    s = Setup([700, 64, 0, 1, 65, 201, 350], 2, 1, D, 16, cache=cache, seed=D + budget)
    sums = torch.exp(2 * torch.randn((7, 2, s.table.shape[1] * 16 + 5), device=dev(),
                                     generator=torch.Generator(device=dev()).manual_seed(budget)))
    _check_evict(s, sums, budget, first, last, in_place)


@pytest.mark.parametrize("ps,layout", [(1, "heads"), (10, "tokens"), (24, "heads"), (512, "tokens")])
def test_evict_page_sizes(hip_lib, ps, layout):
    s = Setup([1500, 300, 77], 2, 1, 64, ps, layout=layout, seed=ps)
    sums = torch.rand((3, 2, s.table.shape[1] * ps), device=dev())
    _check_evict(s, sums, 77, 5, 11)


def test_evict_ties_zeros_and_odd_values(hip_lib):
    """Equal sums go to the lowest positions, -0 is 0, infinities and NaN have their order, whole rows of one
    value, sums below nothing."""
    s = Setup([500] * 6, 1, 1, 16, 16, seed=2)
    sums = torch.zeros((6, 1, s.table.shape[1] * 16), device=dev())
    sums[0, 0, ::2] = -0.0
    sums[1, 0] = torch.randint(0, 3, sums[1, 0].shape, device=dev()).float()
    sums[2, 0] = torch.randn(sums[2, 0].shape, device=dev())
    sums[2, 0, 5:400:7] = math.inf
    sums[2, 0, 6:400:7] = -math.inf
    sums[3, 0] = 1.0
    sums[3, 0, 100:130] = math.nan
    sums[4, 0] = torch.randn(sums[4, 0].shape, device=dev()) * 1e-42      # subnormal
    sums[5, 0] = 3.4e38
    _check_evict(s, sums, 50, 2, 9)


@pytest.mark.parametrize("budget,first,last", [(4097, 1, 64), (8999, 0, 0), (300, 100, 200), (9001, 9001, 0), (5, 0, 2)])
@pytest.mark.parametrize("kind", ["close", "spread", "ties", "zero"])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("width", [None, 2100])
def test_evict_long(hip_lib, budget, first, last, kind, in_place, width):
    """Rows that a workgroup does not hold in registers, and (a table of more than 32768 positions) rows that
    several workgroups share: keys that agree in their leading digits, that do not, few values."""
    s = Setup([20000, 9000, 100, 8193], 1, 1, 16, 16, seed=2, width=width)
    g = torch.Generator(device=dev()).manual_seed(budget)
    sums = torch.rand((4, 1, s.table.shape[1] * 16), device=dev(), generator=g)
    sums = {"close": 1 + 2e-4 * sums, "spread": torch.exp(40 * sums - 20), "ties": (5 * sums).floor(),
            "zero": 0 * sums}[kind]
    _check_evict(s, sums, budget, first, last, in_place)


@pytest.mark.parametrize("rows,longest", [(129, 9000), (40, 12288), (256, 40000), (65, 32769), (64, 32769), (40, 32768)])
def test_evict_many_rows(hip_lib, rows, longest):
    """A workgroup for each of many rows longer than it holds in registers, and the rule's edges."""
    g = torch.Generator().manual_seed(rows)
    lens = torch.randint(1, 200, (rows,), generator=g).tolist()
    lens[0], lens[rows // 2], lens[-1] = longest, 8193, longest - 777
    s = Setup(lens, 1, 1, 16, 16, seed=2)
    sums = torch.exp(3 * torch.randn((rows, 1, s.table.shape[1] * 16), device=dev()))
    _check_evict(s, sums, 150, 3, 40, in_place=True)


@pytest.mark.parametrize("rows,longest,budget", [(1100, 8192, 511), (1100, 8208, 512), (600, 4800, 513), (600, 4816, 90), (5, 2048, 512), (5, 2064, 513)])
@pytest.mark.parametrize("kind", ["spread", "close", "ties"])
def test_evict_rows_of_a_small_workgroup(hip_lib, rows, longest, budget, kind):
    """The edges of the rules on a row's workgroup: positions to rows, and bytes of a head's kept rows."""
    g = torch.Generator().manual_seed(rows + longest)
    lens = torch.randint(1, 900, (rows,), generator=g).tolist()
    lens[0], lens[rows // 2], lens[-1] = longest, min(longest, 4100), longest - 7
    s = Setup(lens, 1, 1, 16, 16, seed=2)
    sums = torch.rand((rows, 1, s.table.shape[1] * 16), device=dev())
    sums = {"close": 1 + 2e-4 * sums, "spread": torch.exp(40 * sums - 20), "ties": (5 * sums).floor()}[kind]
    _check_evict(s, sums, budget, 3, 40, in_place=kind != "close")


@pytest.mark.parametrize("cache,D", [(FP8, 16), (FP8, 64), (BF16, 128)])
def test_evict_in_many_batches_of_rows_that_share_lines(hip_lib, cache, D):
    """Several batches of rows a head, which wait for each other, and heads whose rows lie in the same lines."""
    s = Setup([12000, 9000, 8500], 4, 1, D, 24, cache=cache, layout="tokens", seed=D)
    g = torch.Generator(device=dev()).manual_seed(D)
    sums = torch.rand((3, 4, s.table.shape[1] * 24), device=dev(), generator=g)
    sums[1, :, :3000] = 0.0                     # nearly all of the first rows go: every row moves far
    _check_evict(s, sums, 8500, 3, 60, in_place=True)


def test_evict_twice_in_place(hip_lib):
    """As a server does: evict, go on from the new lengths, evict again."""
    s = Setup([600, 80, 400], 2, 1, 64, 16, seed=12)
    sums = torch.rand((3, 2, s.table.shape[1] * 16), device=dev())
    _check_evict(s, sums, 300, 4, 32, in_place=True)
    s.lens = s.lens.clamp(max=300)
    _check_evict(s, sums, 100, 4, 32, in_place=True)


# ---- together, streams, graphs --------------------------------------------------------------------------

def test_calls_on_a_stream_of_their_own(hip_lib):
    """Work on another stream than the default, with the same calls at the same time on a second one."""
    s = Setup([1200, 64, 700], 2, 4, 64, 16, seed=13)
    sums = torch.zeros((3, 2, s.table.shape[1] * 16), device=dev())
    want, lse = kv.paged_attention(*s.args(), weight_sums=sums, return_lse=True)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(5):
        for st in streams:
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                mine = torch.zeros_like(sums)
                got.append((kv.paged_attention(*s.args(), weight_sums=mine), mine))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) and torch.equal(m, sums) for o, m in got)


def test_a_decode_step_under_graph_capture(hip_lib):
    """Append, counted attention and eviction captured once and replayed on new contents and lengths
    within the captured bounds; every replay gives what the eager calls give."""
    s = Setup([700, 40, 333], 2, 4, 64, 16, seed=14, width=50)
    cap = 50 * 16
    k, v = (torch.zeros((3, 2, 64), dtype=BF16, device=dev()) for _ in range(2))
    start = [t.clone() for t in (s.k, s.v)]
    sums = torch.zeros((3, 2, cap), device=dev())

    def step():
        kv.kv_cache_append(k, v, s.k, s.v, s.table, s.lens)
        out, lse = kv.paged_attention(*s.args(), weight_sums=sums, return_lse=True, max_len=cap)
        new_lens, kept = kv.kv_cache_evict(s.k, s.v, s.table, s.lens, sums, 128, keep_first=4, keep_last=16)
        return out, lse, new_lens, kept

    def reset(i):
        g = torch.Generator(device=dev()).manual_seed(i)
        s.k.copy_(start[0])
        s.v.copy_(start[1])
        for t in (k, v, s.q):
            t.copy_(torch.randn(t.shape, device=dev(), generator=g).to(BF16))
        s.lens.copy_(torch.tensor([700 - 131 * i, 40 - 13 * i, 333 - 5 * i], dtype=torch.int32))
        sums.copy_(torch.rand(sums.shape, device=dev(), generator=g))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        reset(0)
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured = step()
    for i in (0, 1, 2, 3, 0):
        reset(i)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (*captured, sums, s.k.view(torch.int16), s.v.view(torch.int16))]
        reset(i)
        eager = step()
        torch.cuda.synchronize()
        for x, y in zip(got, (*eager, sums, s.k.view(torch.int16), s.v.view(torch.int16))):
            assert torch.equal(x, y), i


def test_python_refusals(hip_lib):
    s = Setup([40, 3], 2, 4, 64, 16)
    sums = torch.zeros((2, 2, 48), device=dev())
    rows = torch.zeros((2, 2, 64), dtype=BF16, device=dev())
    bad = [
        lambda: kv.paged_attention(s.q.to(F16), *s.args()[1:]),
        lambda: kv.paged_attention(s.q[:1], *s.args()[1:]),
        lambda: kv.paged_attention(s.q[:, :3], *s.args()[1:]),
        lambda: kv.paged_attention(s.q.cpu(), *s.args()[1:]),
        lambda: kv.paged_attention(s.q, s.k, s.v.transpose(1, 2).contiguous().transpose(1, 2), s.table, s.lens),
        lambda: kv.paged_attention(s.q, s.k, s.v, s.table.long(), s.lens),
        lambda: kv.paged_attention(s.q, s.k, s.v, s.table, s.lens[:1]),
        lambda: kv.paged_attention(*s.args(), sinks=s.sinks[:3]),
        lambda: kv.paged_attention(*s.args(), weight_sums=sums[:, :, :20]),
        lambda: kv.paged_attention(*s.args(), out=torch.empty((2, 8, 64), device=dev())),
        lambda: kv.kv_cache_append(rows[:1], rows[:1], s.k, s.v, s.table, s.lens),
        lambda: kv.kv_cache_append(rows.float(), rows.float(), s.k, s.v, s.table, s.lens),
        lambda: kv.kv_cache_append(rows, rows, s.k, s.v, s.table, s.lens, query_start=s.lens),
        lambda: kv.kv_cache_evict(s.k, s.v, s.table, s.lens, sums[:, :1], 4),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")
    for call in (lambda: kv.paged_attention(*s.args(), max_len=10 ** 6),
                 lambda: kv.paged_attention(*s.args(), softcap=-1.0),
                 lambda: kv.kv_cache_evict(s.k, s.v, s.table, s.lens, sums, 0),
                 lambda: kv.kv_cache_evict(s.k, s.v, s.table, s.lens, sums, 8, keep_first=5, keep_last=4)):
        with pytest.raises(RuntimeError, match="vk_hip_"):
            call()
