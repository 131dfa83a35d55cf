"""GPU tests of the norm and rotation of queries and keys against the definition in 64 bits."""
from __future__ import annotations

import math

import pytest
import torch

from vkernels_amd.rotary import qk_norm_rope

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def dev():
    return torch.device("cuda", 0)


def definition(x, positions, inv_freq, weight, eps, sections, pairs, factor):
    """(result, size of every value's pair) in 64 bits, on the CPU."""
    x = x.detach().cpu().double()
    T, H, D = x.shape
    R = inv_freq.shape[0]
    if eps is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + torch.tensor(eps, dtype=F32).double())
        if weight is not None:
            x = x * weight.cpu().double()
    p = positions.cpu().double().view(-1, T)
    of = [i for i, n in enumerate([R] if sections is None else sections) for _ in range(n)]
    angle = (p[of] * inv_freq.cpu().double()[:, None]).t()[:, None, :]
    cos, sin = torch.cos(angle) * factor, torch.sin(angle) * factor
    first = torch.arange(R) * 2 if pairs else torch.arange(R)
    second = first + (1 if pairs else R)
    out, size = x.clone(), x.abs()
    a, b = x[..., first], x[..., second]
    out[..., first], out[..., second] = a * cos - b * sin, b * cos + a * sin
    size[..., first] = size[..., second] = torch.hypot(a, b) * abs(factor)
    return out, size


def check(q, k, positions, inv_freq, *, out=None, what="", **kw):
    """The sum of squares in 32 bits is off by D 2^-24 at most, its root by half of that and 2^-22; three products
    2^-24 each; a fraction of a turn cut to 32 bits, its sine and cosine 2^-21 of the pair's size together; the
    rotation's products and sum 3 2^-24: less than D 2^-25 + 2^-20 in all, then half a step of the type."""
    q0, k0 = q.clone(), k.clone()
    got = qk_norm_rope(q, k, positions, inv_freq, out=out, **kw)
    torch.cuda.synchronize()
    for name, x, y in (("q", q0, got[0]), ("k", k0, got[1])):
        want, size = definition(x, positions, inv_freq, kw.get(name + "_weight"), kw.get("eps", 1e-6),
                                kw.get("sections"), kw.get("pairs", False), kw.get("factor", 1.0))
        assert y.dtype is x.dtype and y.shape == x.shape
        tol = size * (x.shape[2] * 2.0 ** -25 + 2.0 ** -20)
        half = torch.finfo(x.dtype).eps / 2
        least = 2.0 ** -134 if x.dtype is BF16 else 2.0 ** -25
        y = y.detach().cpu().double()
        assert torch.equal(torch.isnan(y), torch.isnan(want)), f"{what} {name}: NaN elsewhere"
        off = ((y - want).abs() - half * (want.abs() + tol) - tol - least)[torch.isfinite(want)]
        assert off.numel() == 0 or float(off.max()) <= 0, f"{what} {name}: {float(off.max()):.3g} beyond its bound"
    return got


def inputs(T, Hq, Hkv, D, dtype=BF16, seed=0, extra=0):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn((T, Hq + 2 * Hkv + extra, D), generator=g).to(dtype).to(dev())
    return qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], g


def freqs(R, base=10000.0):
    return (base ** (-torch.arange(R, dtype=torch.float64) / R)).float().to(dev())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("D,turned", [(16, 16), (16, 8), (48, 48), (64, 64), (64, 24), (80, 80), (80, 40), (96, 48), (112, 112),
                                      (128, 128), (128, 32), (192, 192), (240, 120), (256, 256), (256, 8), (256, 248)])
def test_widths(hip_lib, D, turned, pairs, dtype):
    q, k, g = inputs(37, 5, 2, D, dtype, seed=D + turned)
    w = [(1 + 0.3 * torch.randn(D, generator=g)).to(dtype).to(dev()) for _ in range(2)]
    p = torch.randint(0, 5000, (37,), generator=g, dtype=torch.int32).to(dev())
    check(q, k, p, freqs(turned // 2), q_weight=w[0], k_weight=w[1], pairs=pairs)


@pytest.mark.parametrize("T", [1, 2, 3, 63, 257, 1025, 4099])
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (7, 1), (64, 8), (33, 3)])
def test_tokens_and_heads(hip_lib, T, Hq, Hkv):
    """Heads split among wavefronts where tokens are few, all of a wavefront's where they are many."""
    q, k, g = inputs(T, Hq, Hkv, 64, seed=T + Hq)
    check(q, k, torch.arange(T, dtype=torch.int32, device=dev()), freqs(32), q_weight=torch.rand(64, generator=g).to(dev()),
          k_weight=torch.rand(64, generator=g).to(dev()))


@pytest.mark.parametrize("sections", [(16, 24, 24), (64, 0), (0, 64), (0, 0, 1, 63), (64,), (10, 30, 10, 14)])
@pytest.mark.parametrize("pairs", [False, True])
def test_axes(hip_lib, sections, pairs):
    q, k, g = inputs(131, 4, 2, 128)
    p = torch.randint(0, 1 << 20, (len(sections), 140), generator=g, dtype=torch.int32).to(dev())
    check(q, k, p[:, 4:135], freqs(64), sections=sections, pairs=pairs)


def test_far_positions(hip_lib):
    """Positions up to the ends of 32 bits, negative ones too, at a frequency of 1 and beyond."""
    q, k, _ = inputs(7, 3, 1, 64, F16)
    p = torch.tensor([0, 1, 1 << 20, (1 << 24) + 1, 2147483647, -2147483648, -12345], dtype=torch.int32, device=dev())
    check(q, k, p, freqs(32))
    check(q, k, p, torch.linspace(0, 3.0, 32, device=dev()), factor=0.7)


@pytest.mark.parametrize("q_weight,k_weight", [(True, False), (False, True), (False, False)])
@pytest.mark.parametrize("f32", [False, True])
def test_weights_on_one_side(hip_lib, q_weight, k_weight, f32):
    q, k, g = inputs(9, 4, 4, 96, F16)
    w = (torch.rand(97, generator=g) + 0.5).to(F32 if f32 else F16).to(dev())[1:]        # (does not start on 16 bytes)
    check(q, k, torch.arange(9, dtype=torch.int32, device=dev()), freqs(48), q_weight=w if q_weight else None,
          k_weight=w if k_weight else None, eps=1e-3)


def test_without_norm(hip_lib):
    q, k, _ = inputs(50, 6, 2, 80)
    check(q, k, torch.arange(50, dtype=torch.int32, device=dev()), freqs(40), eps=None)


def test_in_place_and_given_results(hip_lib):
    q, k, _ = inputs(300, 8, 2, 128, extra=1)
    whole = q._base
    before = whole.clone()
    p = torch.arange(300, dtype=torch.int32, device=dev())
    apart = qk_norm_rope(q, k, p, freqs(64))
    got = check(q, k, p, freqs(64), out=(q, k))
    assert got[0] is q and got[1] is k and torch.equal(q, apart[0]) and torch.equal(k, apart[1])
    assert torch.equal(whole[:, 10:], before[:, 10:])          # values and what lies beside them
    room = torch.full((300, 20, 136), 7.0, dtype=BF16, device=dev())
    check(before[:, :8], before[:, 8:10], p, freqs(64), out=(room[:, 1:9, :128], room[:, 11:13, :128]))
    assert bool((room[:, :, 128:] == 7).all() and (room[:, 0] == 7).all() and (room[:, 9:11] == 7).all())


def test_strides_and_alignment(hip_lib):
    """Heads before tokens in memory, rows that do not start on 16 bytes, a broadcast token, odd strides of
    dimensions of size 1."""
    g = torch.Generator().manual_seed(3)
    p = torch.arange(21, dtype=torch.int32, device=dev())
    by_head = torch.randn((5, 21, 64), generator=g).to(BF16).to(dev())
    check(by_head[:4].transpose(0, 1), by_head[4:].transpose(0, 1), p, freqs(32))
    odd = torch.randn((21, 5, 67), generator=g).to(BF16).to(dev())
    check(odd[:, :4, 1:65], odd[:, 4:, 3:], p, freqs(32))
    one = torch.randn((1, 5, 64), generator=g).to(BF16).to(dev()).expand(21, 5, 64)
    check(one[:, :4], one[:, 4:], p, freqs(32))
    x = torch.randn((64 * 7 + 1,), generator=g).to(BF16).to(dev())
    check(x.as_strided((1, 1, 64), (3, 5, 1)), x.as_strided((1, 1, 64), (1, 1, 1), 64), p[:1], freqs(32))


def test_rows_of_zeros_infinities_and_nan_stay_to_themselves(hip_lib):
    q, k, _ = inputs(12, 4, 2, 64)
    q, k = q.clone(), k.clone()
    q[3, 1] = 0
    q[4, 2, 5] = math.inf
    k[5, 0, 60] = math.nan
    p = torch.arange(12, dtype=torch.int32, device=dev())
    got = check(q, k, p, freqs(32))
    assert bool((got[0][3, 1] == 0).all())
    # values beside the rotation see nothing of each other
    k[5, 0, 60], k[6, 1, 50] = 1.0, math.inf
    got = qk_norm_rope(q, k, p, freqs(8), eps=None)
    assert bool(torch.isfinite(got[1][6, 1, :50]).all()) and got[1][6, 1, 50] == math.inf and bool(torch.isfinite(got[1][6, 1, 51:]).all())


def test_streams_and_graphs(hip_lib):
    q, k, g = inputs(65, 8, 2, 128)
    q, k = q.clone(), k.clone()
    p = torch.arange(65, dtype=torch.int32, device=dev())
    f = freqs(64)
    out = torch.empty_like(q), torch.empty_like(k)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        qk_norm_rope(q, k, p, f, out=out)
    side.synchronize()
    want = qk_norm_rope(q, k, p, f)
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = qk_norm_rope(q, k, p, f)
    for i in range(3):
        q.mul_(-0.5)
        p.add_(100)
        graph.replay()
        want = qk_norm_rope(q, k, p, f)
        torch.cuda.synchronize()
        assert torch.equal(captured[0], want[0]) and torch.equal(captured[1], want[1])


def test_no_tokens_and_no_gradient(hip_lib):
    f = freqs(32)
    q, k = qk_norm_rope(torch.empty((0, 4, 64), dtype=BF16, device=dev()), torch.empty((0, 2, 64), dtype=BF16, device=dev()),
                        torch.empty(0, dtype=torch.int32, device=dev()), f)
    assert q.shape == (0, 4, 64) and k.shape == (0, 2, 64)
    q, k, _ = inputs(5, 4, 2, 64)
    q = q.clone().requires_grad_()
    p = torch.arange(5, dtype=torch.int32, device=dev())
    a, b = qk_norm_rope(q, k, p, f)
    with pytest.raises(RuntimeError, match="no backward"):
        (a.float().sum() + b.float().sum()).backward()
    with torch.no_grad():
        assert not qk_norm_rope(q, k, p, f)[0].requires_grad


def test_refusals(hip_lib):
    q, k, _ = inputs(5, 4, 2, 64)
    p, f = torch.arange(5, dtype=torch.int32, device=dev()), freqs(32)
    w = torch.ones(64, device=dev())
    for bad in (dict(q=q[:4]), dict(k=k[..., :48]), dict(k=k.half()), dict(q=q.float(), k=k.float()), dict(positions=p.long()),
                dict(positions=p[:4]), dict(positions=p.cpu()), dict(inv_freq=f.double()), dict(inv_freq=freqs(33)),
                dict(inv_freq=f[::2]), dict(sections=(16, 16)), dict(positions=p.expand(2, 5), sections=(16, 15)),
                dict(positions=p.expand(5, 5), sections=(10, 10, 10, 1, 1)), dict(positions=p.expand(2, 5), sections=(33, -1)),
                dict(q_weight=w[:32]), dict(q_weight=w, k_weight=w.to(BF16)), dict(q_weight=w.half()),
                dict(q_weight=w, eps=None), dict(out=(torch.empty_like(k), k)), dict(out=(q, k[:, :1].expand(5, 2, 64)[..., ::1].half())),
                dict(q=q[:, :0])):
        args = dict(q=q, k=k, positions=p, inv_freq=f, **{n: v for n, v in bad.items() if n not in ("q", "k", "positions", "inv_freq")})
        args.update(bad)
        with pytest.raises(ValueError):
            qk_norm_rope(args.pop("q"), args.pop("k"), args.pop("positions"), args.pop("inv_freq"), **args)
    for bad in (dict(inv_freq=f[:31]), dict(inv_freq=f[:0]), dict(eps=-1.0), dict(eps=math.nan),
                dict(out=(q, k[:, :1].expand(5, 2, 64))), dict(out=(q[:1].expand(5, 4, 64), k))):
        with pytest.raises(RuntimeError, match="vk_hip_qk_norm_rope failed"):
            qk_norm_rope(q, k, p, **dict(dict(inv_freq=f), **bad))
