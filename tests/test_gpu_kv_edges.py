"""GPU tests of the key-value cache's operators at the ends of what their arguments may be, against the
definitions."""
from __future__ import annotations

import pytest
import torch

import kv_reference as ref
from test_gpu_kv_cache import BF16, F16, FP8, Setup, dev
from vkernels_amd import kv_cache as kv

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window", [2 ** 31 - 17, 2 ** 31 - 16, 2 ** 31 - 1])
@pytest.mark.parametrize("lens", [[40, 0, 130], [1300, 5, 2500]])
def test_a_window_beyond_every_length(hip_lib, window, lens):
    """The largest integers as a window are no window: the same split, results and sums."""
    s = Setup(lens, 2, 4, 64, 16, seed=21)
    out, lse, _ = s.check(window=window, counted=True, sinks=True)
    want, want_lse, _ = s.check(counted=True, sinks=True)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("cache,q", [(BF16, BF16), (F16, F16), (FP8, BF16), (FP8, F16)])
@pytest.mark.parametrize("n", [33, 40, 1200, 20000])
@pytest.mark.parametrize("where", ["first", "last", "every 32"])
def test_many_small_weights_beside_a_large_one(hip_lib, cache, q, n, where):
    """One position takes nearly all the weight and has a value of zero (or of one), all others are `gap`
    nats below it and alike: what they add up to is the result (or part of it), to the result's own
    rounding.  Or every tile of 32 has such a position.

    Scores are single products, exact.  A weight is off by 2^-24 of its exponent in powers of two (less
    than 64) twice and by 2^-22 of the exponential, and bf16 keeps 2^-17 of it; a lane adds up fewer than
    64 tiles one after the other; numerator and sum: below 2^-15 of the result in all, its rounding aside."""
    s = Setup([n] * 6, 1, 1, 64, 16, cache=cache, q=q, seed=n)
    at = {"first": [0], "last": [n - 1], "every 32": list(range(5, n, 32))}[where]
    gaps = torch.tensor([8.0, 12.0, 16.0, 18.0, 20.0, 16.0])
    s.q.zero_()
    s.q[:, :, 0] = 1.0
    if s.k_scale is not None:
        s.k_scale, s.v_scale = torch.ones_like(s.k_scale), torch.ones_like(s.v_scale)
    j = torch.arange(n, device=dev())
    for b, gap in enumerate(gaps.tolist()):
        rows, values = torch.zeros((n, 1, 64), device=dev()), torch.ones((n, 1, 64), device=dev())
        rows[:, 0, 0] = -gap
        rows[at] = 0.0
        if b < 5:
            values[:, 0, ::2] += torch.rand((n, 32), device=dev(), generator=torch.Generator(device=dev()).manual_seed(b))
            values[at] = 0.0
        page = s.table[b].long()[j // 16]
        for c, x in ((s.k, rows), (s.v, values)):
            if c.element_size() == 1:
                c.view(torch.uint8)[page, :, j % 16] = x.to(c.dtype).view(torch.uint8)
            else:
                c[page, :, j % 16] = x.to(c.dtype)
    out = kv.paged_attention(*s.args(), scale=1.0, k_scale=s.k_scale, v_scale=s.v_scale)
    want = ref.attention(*s.args(), scale=1.0, k_scale=s.k_scale, v_scale=s.v_scale)[0]
    unit, small = (2.0 ** -7, 2.0 ** -133) if q == BF16 else (2.0 ** -10, 2.0 ** -24)
    off = (ref.host(out) - want).abs() - (unit / 2 + 2.0 ** -15) * want - small / 2
    assert float(off.max()) <= 0, [float(x) for x in off.amax((1, 2))]


def test_sizes_beyond_32_bits_are_not_cut_to_them(hip_lib):
    """max_len, budget and what is always kept are refused, windows of any size are none."""
    s = Setup([200, 150], 2, 4, 64, 16, seed=23)
    sums = torch.rand((2, 2, 208), device=dev())
    before = [t.clone() for t in (s.k, s.v, sums)]
    for n in (2 ** 31, 2 ** 32, 2 ** 32 + 100, -2 ** 32 + 100, 2 ** 63 - 1, 2 ** 64 + 100):
        for call in (lambda: kv.paged_attention(*s.args(), max_len=n),
                     lambda: kv.paged_attention(*s.args(), max_len=n, weight_sums=sums),
                     lambda: kv.kv_cache_evict(*s.args()[1:], sums, 100, max_len=n),
                     lambda: kv.kv_cache_evict(*s.args()[1:], sums, n),
                     lambda: kv.kv_cache_evict(*s.args()[1:], sums, 100, keep_first=n),
                     lambda: kv.kv_cache_evict(*s.args()[1:], sums, 100, keep_last=n)):
            with pytest.raises(ValueError):
                call()
    assert all(torch.equal(a.view(torch.int8), b.view(torch.int8)) for a, b in zip(before, (s.k, s.v, sums)))
    want = kv.paged_attention(*s.args())
    for window in (2 ** 31, 2 ** 32 + 5, 2 ** 63 - 1, 2 ** 64 + 5, -2 ** 32 + 5, -1):
        assert torch.equal(kv.paged_attention(*s.args(), window=window), want), window


def test_a_table_of_more_positions_than_32_bits_count(hip_lib):
    """Its default bound is refused (it would be cut to 0 positions), a bound that is given is taken."""
    s = Setup([200, 150], 1, 4, 16, 128, seed=24)
    wide = s.table[:, :1].expand(-1, 1).repeat(1, 1 << 24)
    wide[:, :s.table.shape[1]] = s.table
    want = kv.paged_attention(*s.args())
    with pytest.raises(ValueError, match="max_len"):
        kv.paged_attention(s.q, s.k, s.v, wide, s.lens)
    assert torch.equal(kv.paged_attention(s.q, s.k, s.v, wide, s.lens, max_len=256), want)
    with pytest.raises(ValueError, match="max_len"):
        kv.kv_cache_evict(s.k, s.v, wide, s.lens, torch.rand((2, 1, 256), device=dev()), 100)


@pytest.mark.parametrize("pitch", [(65, 65), (64, 67), (129, 64)])
def test_rows_of_odd_strides_in_dimensions_of_size_one(hip_lib, pitch):
    """One sequence and one head out of a buffer of an odd pitch: contiguous, and its strides are no multiple
    of 16 bytes all the same."""
    s = Setup([90], 1, 1, 64, 16, seed=25)
    want = kv.paged_attention(*s.args())
    s.q = torch.empty(200, dtype=BF16, device=dev()).as_strided((1, 1, 64), (*pitch, 1)).copy_(s.q)
    assert s.q.is_contiguous() and s.q.data_ptr() % 16 == 0 and s.q.stride() == (*pitch, 1)
    assert torch.equal(kv.paged_attention(*s.args()), want)
    after = ref.append(s.k, s.v, s.q, -s.q, s.table, s.lens, None, None, None)
    kv.kv_cache_append(s.q, (-s.q).as_strided((1, 1, 64), (*pitch, 1)), s.k, s.v, s.table, s.lens)
    assert all(torch.equal(a.cpu().view(torch.int16), b.view(torch.int16)) for a, b in zip((s.k, s.v), after))


def test_rows_of_one_head_out_of_an_odd_pitch(hip_lib):
    """Several sequences of one head whose strides over the heads are odd, and one sequence of several heads
    whose stride over the sequences is."""
    for B, Hq, strides in ((3, 1, (128, 65)), (1, 4, (259, 64))):
        s = Setup([90] * B, 1, Hq, 64, 16, seed=26)
        want = kv.paged_attention(*s.args())
        s.q = torch.empty(1000, dtype=BF16, device=dev()).as_strided((B, Hq, 64), (*strides, 1)).copy_(s.q)
        assert torch.equal(kv.paged_attention(*s.args()), want)


@pytest.mark.parametrize("cache,q", [(BF16, BF16), (FP8, F16)])
def test_caps_of_any_size(hip_lib, cache, q):
    """Infinity and caps that no score comes near change nothing; under the least caps all scores are alike."""
    s = Setup([60, 1200], 2, 4, 64, 16, cache=cache, q=q, seed=27)
    scales = dict(k_scale=s.k_scale, v_scale=s.v_scale)
    want = kv.paged_attention(*s.args(), **scales)
    for softcap in (float("inf"), 1e300, 3.4e38, 2.5e38, 1e38, 2.0 ** 100):
        assert torch.equal(kv.paged_attention(*s.args(), softcap=softcap, **scales), want), softcap
    # the two ways to a score differ by 2^-20 of it at most, scores here are below 32: 2^-15 of a weight, and
    # the result's last place (8 or 11 bits) once for either
    size = kv.paged_attention(s.q, s.k, (s.v.float().abs()).to(cache), s.table, s.lens, **scales).float()
    unit = 2.0 ** -7 if q == BF16 else 2.0 ** -10
    for softcap in (1e29, 1e20, 1e9):
        got = kv.paged_attention(*s.args(), softcap=softcap, **scales)
        assert float(((got.float() - want.float()).abs() - 2 * (unit + 2.0 ** -15) * size).max()) <= 0, softcap
    zero = torch.zeros_like(s.q)
    want = kv.paged_attention(zero, *s.args()[1:], **scales)
    for softcap in (1e-44, 1e-38, 1e-30, 1e-20):
        assert torch.equal(kv.paged_attention(*s.args(), softcap=softcap, **scales), want), softcap


@pytest.mark.parametrize("which", ["q", "sinks", "k_cache"])
def test_a_backward_pass_is_an_error(hip_lib, which):
    """The results are those of inference, and what would be a gradient of nothing raises."""
    s = Setup([60, 1200], 2, 4, 64, 16, seed=28)
    want, want_lse = kv.paged_attention(*s.args(), sinks=s.sinks, return_lse=True)
    assert not want.requires_grad and not want_lse.requires_grad
    {"q": s.q, "sinks": s.sinks, "k_cache": s.k}[which].requires_grad_()
    out, lse = kv.paged_attention(*s.args(), sinks=s.sinks, return_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    for result in (out, lse, kv.paged_attention(*s.args(), sinks=s.sinks)):
        with pytest.raises(RuntimeError, match="no backward"):
            result.float().sum().backward()
    mine = torch.empty_like(want)
    assert kv.paged_attention(*s.args(), sinks=s.sinks, out=mine) is mine and torch.equal(mine, want)
    for off in (torch.no_grad, torch.inference_mode):
        with off():
            out = kv.paged_attention(*s.args(), sinks=s.sinks)
            assert not out.requires_grad and torch.equal(out, want)
