"""The cache, its attention and its eviction together, as a decode loop uses them, next to the MoE layer:
every step's attention against the definition on what the cache should hold, and every eviction
against the weights that the positions were given."""
from __future__ import annotations

import pytest
import torch

import kv_reference as ref
from vkernels_amd import synth
from vkernels_amd import vllm_experts as ve
from vkernels_amd.decode_layer import DecodeLayer, _example

pytestmark = pytest.mark.gpu


class Watched(DecodeLayer):
    """Keeps what the cache should hold, one list of rows for each sequence and head, and compares."""

    def __init__(self, *args, **kw):
        super().__init__(*args, **kw)
        B, self.evictions, self.steps = len(self.lens), 0, 0
        self.rows = [[[] for _ in range(self.kv_heads)] for _ in range(B)]       # (key, value, weight so far)

    def _store(self, b, k, v):
        for g in range(self.kv_heads):
            self.rows[b][g].append([k[g], v[g], 0.0])

    def prefill(self, k, v, lengths):
        super().prefill(k, v, lengths)
        at = 0
        for b, n in enumerate(lengths):
            for t in range(at, at + n):
                self._store(b, k[t].cpu(), v[t].cpu())
            at += n

    def attend(self, q, k, v):
        out = super().attend(q, k, v)
        self.steps += 1
        longest = max(self.lens)
        for b in range(len(self.lens)):
            self._store(b, k[b].cpu(), v[b].cpu())
            n = len(self.rows[b][0])
            assert n == self.lens[b] == int(self.lens_dev[b])
            kc, vc = (torch.stack([torch.stack([row[i] for row in head]) for head in self.rows[b]])[None] for i in (0, 1))
            want = ref.attention(q[b:b + 1], kc, vc, torch.zeros((1, 1), dtype=torch.int32),
                                 torch.tensor([n], dtype=torch.int32), scale=self.head_dim ** -0.5,
                                 sinks=None if self.sinks is None else self.sinks.cpu())
            ref.assert_attention(out[b:b + 1], None, want, q.dtype, f"step {self.steps} sequence {b} of {longest}")
            for g in range(self.kv_heads):
                for j, row in enumerate(self.rows[b][g]):
                    row[2] += float(want[2][0, g, j])
        return out

    def evict(self):
        before = list(self.lens)
        sums = None if self.sums is None else ref.host(self.sums)
        kept = super().evict()
        if kept is None:
            return None
        self.evictions += 1
        kept = kept.cpu()
        for b, n in enumerate(before):
            for g in range(self.kv_heads):
                rows = self.rows[b][g]
                # 2^-24 of each addition so far, and the weights' own error, far below 1e-4 of a row
                assert all(abs(float(sums[b, g, j]) - row[2]) <= 1e-4 * (1 + row[2]) for j, row in enumerate(rows))
                at = [int(j) for j in kept[b, g] if j >= 0]
                assert len(at) == min(n, self.budget) and at == sorted(set(at))
                if n > self.budget:
                    assert at[:self.keep_first] == list(range(self.keep_first))
                    assert at[-self.keep_last:] == list(range(n - self.keep_last, n))
                    gone = set(range(n)) - set(at)
                    middle = [j for j in at if self.keep_first <= j < n - self.keep_last]
                    assert min(sums[b, g, j] for j in middle) >= max(sums[b, g, j] for j in gone)
                self.rows[b][g] = [rows[j] for j in at]
        return kept


def _layer(budget, sinks):
    cfg = synth.CONFIGS["c0"]
    dev = torch.device("cuda", 0)
    w = synth.make_weights(cfg.E, cfg.H, cfg.I, 3, device=dev)
    experts = ve.FusedExperts(w.w13, w.w13_scale, w.w2, w.w2_scale)
    g = torch.Generator(device=dev).manual_seed(4)

    def normal(*shape, std=1.0):
        return (torch.randn(shape, device=dev, generator=g) * std).to(torch.bfloat16)

    layer = Watched(experts, normal(cfg.H, 8 * 64, std=0.15), normal(4 * 64, cfg.H, std=0.1), normal(cfg.H, cfg.E, std=0.06),
                    kv_heads=2, head_dim=64, top_k=cfg.top_k, sequences=3, pages=24, page_size=16, max_positions=128,
                    budget=budget, slack=16, keep_first=2, keep_last=8,
                    sinks=torch.randn(4, device=dev, generator=g) if sinks else None)
    return layer, normal, cfg


@pytest.mark.parametrize("budget,sinks", [(None, False), (40, False), (40, True)])
def test_decode_steps(hip_lib, budget, sinks):
    layer, normal, cfg = _layer(budget, sinks)
    layer.prefill(normal(60, 2, 64), normal(60, 2, 64), [30, 0, 30])
    hidden = normal(3, cfg.H)
    for _ in range(60):
        hidden = layer.step(hidden)
        hidden = (hidden.float() / hidden.float().std(-1, keepdim=True)).to(torch.bfloat16)
        assert bool(torch.isfinite(hidden).all())
    assert layer.steps == 60 and layer.evictions == (0 if budget is None else 3)
    assert len(layer.free) + sum(map(len, layer.owned)) == 24
    if budget is not None:
        assert max(layer.lens) <= budget + 16


def test_the_cache_runs_out_of_pages(hip_lib):
    layer, normal, cfg = _layer(None, False)
    with pytest.raises(RuntimeError, match="no page left"):
        layer.prefill(normal(600, 2, 64), normal(600, 2, 64), [200, 200, 200])


def test_example(hip_lib):
    seconds, layer = _example("c0", 5, 100, 40, 64, 8, 2, 64)
    assert seconds > 0 and max(layer.lens) < 64 + 32
