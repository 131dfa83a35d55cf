"""Norm and rotation, block-scaled cache, prompts' attention, window and reading back together, as a decode layer runs
them: every attention against the definition on what the layer's cache holds, and what it holds against the keys that
went in."""
from __future__ import annotations

import pytest
import torch

import attention_reference as aref
import kv_reference as ref
from test_gpu_rotary import definition
from vkernels_amd import synth
from vkernels_amd import vllm_experts as ve
from vkernels_amd.decode_layer import DecodeLayer, _example

pytestmark = pytest.mark.gpu

BF16, FP8 = torch.bfloat16, torch.float8_e4m3fn


def dev():
    return torch.device("cuda", 0)


def _layer(D=64, **kw):
    cfg = synth.CONFIGS["c0"]
    w = synth.make_weights(cfg.E, cfg.H, cfg.I, 3, device=dev())
    experts = ve.FusedExperts(w.w13, w.w13_scale, w.w2, w.w2_scale)
    gen = torch.Generator(device=dev()).manual_seed(5)

    def normal(*shape, std=1.0):
        return (torch.randn(shape, device=dev(), generator=gen) * std).to(BF16)

    heads, kv_heads = 4, 2
    layer = DecodeLayer(experts, normal(cfg.H, (heads + 2 * kv_heads) * D, std=cfg.H ** -0.5), normal(heads * D, cfg.H, std=0.02),
                        normal(cfg.H, cfg.E, std=cfg.H ** -0.5), kv_heads=kv_heads, head_dim=D, top_k=cfg.top_k, sequences=3,
                        pages=60, max_positions=400, sinks=torch.randn(heads, device=dev(), generator=gen), **kw)
    return layer, normal, cfg


ROTARY = dict(inv_freq=1e4 ** -(torch.arange(0, 64, 2) / 64))


@pytest.mark.parametrize("options", [
    dict(), dict(window=20, window_first=3), dict(cache_dtype=FP8, scale_blocks=1), dict(cache_dtype=FP8, scale_blocks=16, window=33),
    dict(sections=(8, 12, 12)), dict(pairs=True, cache_dtype=FP8, scale_blocks=4)])
def test_prompts_and_steps(hip_lib, options):
    rotary = dict(ROTARY, inv_freq=ROTARY["inv_freq"].to(dev()), eps=1e-5,
                  **{n: options.pop(n) for n in ("sections", "pairs") if n in options})
    layer, normal, cfg = _layer(rotary=rotary, **options)
    keys = [[] for _ in range(3)]                 # what went in, in 64 bits
    seen = [0, 0, 0]
    turned = dict(weight=None, eps=1e-5, sections=rotary.get("sections"), pairs=rotary.get("pairs", False), factor=1.0)

    def turn(x, positions):
        p = torch.tensor(positions, dtype=torch.int32)
        if turned["sections"] is not None:
            p = p.expand(3, -1)
        return definition(x, p, rotary["inv_freq"], **turned)[0]

    def check(out, q, k, counts):
        positions = [seen[b] + i for b, n in enumerate(counts) for i in range(n)]
        want_k = turn(k, positions)
        at = 0
        for b, n in enumerate(counts):
            keys[b] += list(want_k[at:at + n])
            at += n
            seen[b] += n
        assert layer.positions.tolist() == seen == layer.lens
        got_k, _ = layer.read()
        got_k = got_k.cpu().double()
        held = torch.stack([row for rows in keys for row in rows])
        # bf16 rounds by 2^-8; codes once more by 2^-4 of a value or 2^-10 of the block's scale, a few times where it
        # grew, and a block's scale is at most its largest value / 448
        tol = (2.0 ** -4 * 4 if layer.k_cache.dtype is FP8 else 2.0 ** -7) * held.abs() + 2.0 ** -6 * 8.0 / 448 + 2.0 ** -9
        assert bool(((got_k - held).abs() <= tol).all())
        # the attention, from what the cache holds and the queries as they are rounded
        starts = torch.tensor([0, *counts]).cumsum(0)
        q_turned = turn(q, positions).to(BF16)
        want = aref.attention(q_turned, layer.k_cache, layer.v_cache, layer.table, layer.lens_dev, starts, scale=64 ** -0.5,
                              sinks=layer.sinks.cpu(), weight_bits=8, **layer.sees,
                              **{n: None if s is None else s.cpu() for n, s in layer.scales.items()})
        # (a query's own rounding may fall the other way where its value lies at a border: half a step of 2^-8 moves a
        # score by up to 2^-8 of sum |q k| / 8, a row's result by as much of its values)
        got, exact = out.cpu().double(), want[0]
        assert float((got - exact).norm() / exact.norm()) < 2.0 ** -7

    for counts in ([30, 5, 0], [0, 40, 17], [3, 1, 64]):
        n = sum(counts)
        q, k, v = normal(n, 4, 64), normal(n, 2, 64), normal(n, 2, 64)
        check(layer.prefill(k, v, counts, q=q), q, k, counts)
    for _ in range(6):
        q, k, v = normal(3, 4, 64), normal(3, 2, 64), normal(3, 2, 64)
        check(layer.attend(q, k, v), q, k, [1, 1, 1])
    hidden = normal(3, cfg.H)
    for _ in range(3):
        hidden = layer.step(hidden)
    assert bool(torch.isfinite(hidden.float()).all()) and layer.positions.tolist() == layer.lens == [n + 3 for n in seen]


def test_prompts_attention_without_rotation(hip_lib):
    layer, normal, _ = _layer()
    q, k, v = normal(50, 4, 64), normal(50, 2, 64), normal(50, 2, 64)
    out = layer.prefill(k, v, [20, 0, 30], q=q)
    want = aref.attention(q, layer.k_cache, layer.v_cache, layer.table, layer.lens_dev, torch.tensor([0, 20, 20, 50]),
                          scale=64 ** -0.5, sinks=layer.sinks.cpu(), weight_bits=8)
    ref.assert_attention(out, None, want, BF16)
    got_k, got_v = layer.read()
    assert torch.equal(got_k, k) and torch.equal(got_v, v)


def test_a_refused_prompt_leaves_the_layer_as_it_was(hip_lib):
    layer, normal, _ = _layer(cache_dtype=FP8, scale_blocks=1)
    q, k, v = normal(50, 4, 64), normal(50, 2, 64), normal(50, 2, 64)
    layer.prefill(k, v, [20, 0, 30], q=q)
    before = [t.clone() for t in (layer.k_cache.view(torch.uint8), layer.scales["k_scale"])]
    for bad in (q[:, :3], q.half(), q[:49]):
        with pytest.raises(ValueError):
            layer.prefill(k, v, [20, 0, 30], q=bad)
    with pytest.raises(ValueError):
        layer.attend(q[:3, :2], k[:3], v[:3])
    assert layer.lens == [20, 0, 30] == layer.positions.tolist()
    assert torch.equal(before[0], layer.k_cache.view(torch.uint8)) and torch.equal(before[1], layer.scales["k_scale"])


def test_queries_and_keys_of_two_types(hip_lib):
    """Of an 8-bit cache with a scale for each head either 16-bit type is read and written."""
    scale = torch.full((2,), 0.02, device=dev())
    layer, normal, _ = _layer(cache_dtype=FP8, k_scale=scale, v_scale=scale)
    q, k, v = normal(3, 4, 64).half(), normal(3, 2, 64), normal(3, 2, 64)
    out = layer.attend(q, k, v)
    want = aref.attention(q, layer.k_cache, layer.v_cache, layer.table, layer.lens_dev, torch.tensor([0, 1, 2, 3]),
                          scale=64 ** -0.5, sinks=layer.sinks.cpu(), k_scale=scale.cpu(), v_scale=scale.cpu())
    assert out.dtype is torch.float16
    ref.assert_attention(out, None, want, torch.float16)


def test_the_command_runs(hip_lib):
    for kw in (dict(rotary=True), dict(window=64, window_first=4, scale_blocks=1), dict(rotary=True, scale_blocks=16, window=100)):
        seconds, layer = _example("c0", 4, 150, 3, None, 8, 2, 64, **kw)
        assert seconds > 0 and max(layer.lens) == 153
