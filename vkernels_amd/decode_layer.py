"""One decoder layer's decode step on this library: projections, the new token into the paged cache,
attention over it, eviction when the cache is over its budget, and the MoE layer.

    python -m vkernels_amd.decode_layer [--sequences 64] [--context 2048] [--steps 64] [--budget 1024]

runs it on synthetic weights of one of the benchmark configurations' widths.  What a serving program
keeps is kept here as well: the pages and their free list, the block table, the lengths (on the host,
so that no step reads them back) and what every position has been given so far.  The lengths and new
pages go to the device by small copies from ordinary host memory, for which the host waits in every step: a
step cannot be captured in a graph (the operators by themselves can).
"""
from __future__ import annotations

import contextlib

import torch

from .kv_cache import kv_cache_append, kv_cache_evict, paged_attention

__all__ = ["DecodeLayer"]


def _norm(x):
    """Root-mean-square norm without a weight."""
    return (x.float() * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + 1e-6)).to(x.dtype)


class DecodeLayer:
    """A layer's weights and the key-value cache of a batch of sequences.

    ``experts`` is a FusedExperts; ``w_qkv`` [hidden, (Hq + 2 Hkv) D], ``w_out`` [Hq D, hidden] and
    ``w_router`` [hidden, experts] are bf16.  With a ``budget`` a sequence whose cache has grown to
    ``budget + slack`` positions is cut back to ``budget``: its first ``keep_first``, its latest
    ``keep_last`` and those that have been given the most weight (position encodings, where a model
    has them, go into the keys before they are stored).  ``pages`` bounds the cache; pages that an
    eviction empties serve other sequences.
    """

    def __init__(self, experts, w_qkv, w_out, w_router, *, kv_heads, head_dim, top_k, sequences, pages, page_size=16,
                 max_positions, cache_dtype=torch.bfloat16, k_scale=None, v_scale=None, sinks=None, budget=None,
                 slack=256, keep_first=4, keep_last=None):
        dev = w_qkv.device
        self.experts, self.w_qkv, self.w_out, self.w_router = experts, w_qkv, w_out, w_router
        self.kv_heads, self.head_dim, self.top_k, self.page_size = kv_heads, head_dim, top_k, page_size
        self.heads = w_out.shape[0] // head_dim
        if w_qkv.shape[1] != (self.heads + 2 * kv_heads) * head_dim or self.heads % kv_heads:
            raise ValueError("w_qkv must be [hidden, (Hq + 2 Hkv) D] with Hq a multiple of Hkv")
        if budget is not None and budget + slack > max_positions:
            raise ValueError("budget + slack must be within max_positions")
        self.sinks, self.scales = sinks, dict(k_scale=k_scale, v_scale=v_scale)
        self.budget, self.slack, self.keep_first = budget, slack, keep_first
        self.keep_last = keep_last if keep_last is not None else (budget or 0) // 8
        width = -(-max_positions // page_size)
        self.k_cache, self.v_cache = (torch.zeros((pages, kv_heads, page_size, head_dim), dtype=cache_dtype, device=dev)
                                      for _ in range(2))
        self.free = list(range(pages))
        self.owned = [[] for _ in range(sequences)]          # pages of every sequence, in order
        self.lens = [0] * sequences
        self.table = torch.full((sequences, width), -1, dtype=torch.int32, device=dev)
        self.lens_dev = torch.zeros(sequences, dtype=torch.int32, device=dev)
        # only a cache that is evicted from needs to know what its positions were given
        self.sums = None if budget is None else torch.zeros((sequences, kv_heads, width * page_size), device=dev)

    def _grow(self, by):
        """Room for `by` more positions in every sequence (host lists, one small copy to the device).  Where
        there is none, nothing has been taken when the call is refused."""
        lens, grow, left = [], [], len(self.free)
        for b, n in enumerate(self.lens):
            n += by[b]
            lens.append(n)
            have = len(self.owned[b])
            if n > have * self.page_size:
                more = -(-n // self.page_size) - have
                left -= more
                if left < 0 or have + more > self.table.shape[1]:
                    raise RuntimeError("the cache has no page left for sequence %d" % b)
                grow.append((b, more))
        rows, columns, pages = [], [], []
        for b, more in grow:
            for _ in range(more):
                rows.append(b)
                columns.append(len(self.owned[b]))
                pages.append(self.free.pop())
                self.owned[b].append(pages[-1])
        if pages:
            at = torch.tensor([rows, columns, pages], device=self.table.device)
            self.table[at[0], at[1]] = at[2].to(torch.int32)
        self._set_lens(lens)

    @contextlib.contextmanager
    def _grown(self, by):
        """The sequences longer by `by` for calls that fill the new positions; where one of them is refused the
        lengths are what they were (the pages taken stay with their sequences)."""
        before = list(self.lens)
        self._grow(by)
        try:
            yield
        except Exception:
            self._set_lens(before)
            raise

    def _set_lens(self, lens):
        self.lens[:] = lens
        self.lens_dev.copy_(torch.tensor(lens, dtype=torch.int32))

    def prefill(self, k, v, lengths):
        """Keys and values [tokens, Hkv, D] of the sequences' prompts, one behind the other."""
        starts = torch.tensor([0, *lengths]).cumsum(0).to(torch.int32).to(k.device)
        with self._grown(lengths):
            kv_cache_append(k, v, self.k_cache, self.v_cache, self.table, self.lens_dev, query_start=starts, **self.scales)

    def attend(self, q, k, v):
        """Attention of one new token of every sequence: q [B, Hq, D], its k and v [B, Hkv, D]."""
        with self._grown([1] * len(self.lens)):
            kv_cache_append(k, v, self.k_cache, self.v_cache, self.table, self.lens_dev, **self.scales)
            return paged_attention(q, self.k_cache, self.v_cache, self.table, self.lens_dev, max_len=max(self.lens),
                                   sinks=self.sinks, weight_sums=self.sums, **self.scales)

    def evict(self):
        """Cuts the sequences back to the budget when one has outgrown it; the old positions that were
        kept [B, Hkv, budget], or None when there was nothing to do."""
        if self.budget is None or max(self.lens) < self.budget + self.slack:
            return None
        _, kept = kv_cache_evict(self.k_cache, self.v_cache, self.table, self.lens_dev, self.sums, self.budget,
                                 keep_first=self.keep_first, keep_last=self.keep_last, max_len=max(self.lens))
        need = -(-self.budget // self.page_size)
        for b, n in enumerate(self.lens):
            self.lens[b] = min(n, self.budget)
            self.free += self.owned[b][need:]
            del self.owned[b][need:]
        self.table[:, need:] = -1
        self.lens_dev.clamp_(max=self.budget)
        return kept

    def step(self, hidden):
        """One token of every sequence, hidden [B, H] bf16, through the layer."""
        B, D = hidden.shape[0], self.head_dim
        qkv = (_norm(hidden) @ self.w_qkv).view(B, self.heads + 2 * self.kv_heads, D)
        q, k, v = qkv.split([self.heads, self.kv_heads, self.kv_heads], 1)
        hidden = hidden + self.attend(q, k, v).view(B, -1) @ self.w_out
        self.evict()
        x = _norm(hidden)
        out, _, _ = self.experts.forward(x, (x @ self.w_router).float(), self.top_k)
        return hidden + out.to(hidden.dtype)


def _example(config, sequences, context, steps, budget, heads, kv_heads, head_dim, seed=0):
    """(seconds a step, layer) of `steps` steps behind prompts of `context` positions."""
    from . import synth
    from .vllm_experts import FusedExperts
    cfg = synth.CONFIGS[config]
    dev = torch.device("cuda", torch.cuda.current_device())
    w = synth.make_weights(cfg.E, cfg.H, cfg.I, seed, device=dev)
    experts = FusedExperts(w.w13, w.w13_scale, w.w2, w.w2_scale, prepack=True, keep_raw=False)
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, std=1.0):
        return (torch.randn(shape, device=dev, generator=gen) * std).to(torch.bfloat16)

    longest = context + steps + 1
    pages = sequences * -(-longest // 16)
    layer = DecodeLayer(experts, normal(cfg.H, (heads + 2 * kv_heads) * head_dim, std=cfg.H ** -0.5),
                        normal(heads * head_dim, cfg.H, std=0.02), normal(cfg.H, cfg.E, std=cfg.H ** -0.5),
                        kv_heads=kv_heads, head_dim=head_dim, top_k=cfg.top_k, sequences=sequences, pages=pages,
                        max_positions=max(longest, (budget or 0) + 256), budget=budget, slack=32)
    tokens = sequences * context
    layer.prefill(normal(tokens, kv_heads, head_dim), normal(tokens, kv_heads, head_dim), [context] * sequences)
    hidden = normal(sequences, cfg.H)
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    for i in range(steps):
        if i == min(8, steps - 1):
            start.record()
        hidden = _norm(layer.step(hidden))
    end.record()
    torch.cuda.synchronize()
    return start.elapsed_time(end) * 1e-3 / max(1, steps - min(8, steps - 1)), layer


if __name__ == "__main__":
    import argparse
    ap = argparse.ArgumentParser(description="decode steps of one layer: cache, attention, eviction, experts")
    ap.add_argument("--config", default="c1", help="widths and experts: one of synth.CONFIGS")
    ap.add_argument("--sequences", type=int, default=64)
    ap.add_argument("--context", type=int, default=2048, help="positions of the prompts")
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--budget", type=int, default=None, help="positions a sequence may keep")
    ap.add_argument("--heads", type=int, default=64)
    ap.add_argument("--kv-heads", type=int, default=8)
    ap.add_argument("--head-dim", type=int, default=64)
    a = ap.parse_args()
    seconds, layer = _example(a.config, a.sequences, a.context, a.steps, a.budget, a.heads, a.kv_heads, a.head_dim)
    print(f"{a.sequences} sequences, {seconds * 1e6:.0f} us a step of the layer, "
          f"{max(layer.lens)} positions in the longest cache")
