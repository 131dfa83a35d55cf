"""One decoder layer's decode step on this library: projections, norm and rotation of queries and keys, the new
token into the paged cache, attention over it, eviction when the cache is over its budget, and the MoE layer; and the
attention of prompts.

    python -m vkernels_amd.decode_layer [--sequences 64] [--context 2048] [--steps 64] [--budget 1024]
                                        [--rotary] [--window 128 --window-first 4] [--scale-blocks 1]

runs it on synthetic weights of one of the benchmark configurations' widths.  What a serving program
keeps is kept here as well: the pages and their free list, the block table, the lengths (on the host,
so that no step reads them back) and what every position has been given so far.  The lengths and new
pages go to the device by small copies from ordinary host memory, for which the host waits in every step: a
step cannot be captured in a graph (the operators by themselves can).
"""
from __future__ import annotations

import contextlib

import torch

from .kv_cache import kv_cache_append, kv_cache_evict, kv_cache_read, paged_attention
from .rotary import qk_norm_rope

__all__ = ["DecodeLayer"]


def _norm(x):
    """Root-mean-square norm without a weight."""
    return (x.float() * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + 1e-6)).to(x.dtype)


class DecodeLayer:
    """A layer's weights and the key-value cache of a batch of sequences.

    ``experts`` is a FusedExperts; ``w_qkv`` [hidden, (Hq + 2 Hkv) D], ``w_out`` [Hq D, hidden] and
    ``w_router`` [hidden, experts] are bf16.  With a ``budget`` a sequence whose cache has grown to
    ``budget + slack`` positions is cut back to ``budget``: its first ``keep_first``, its latest
    ``keep_last`` and those that have been given the most weight (position encodings go into the keys
    before they are stored).  Decode steps alone count weight: an eviction ranks a prompt's positions by what the
    steps behind it have given them, and not by what the prompt's own tokens have.  ``pages`` bounds the cache; pages
    that an eviction empties serve other sequences.

    ``rotary`` are the arguments of qk_norm_rope besides queries, keys and positions (``inv_freq`` and what else a
    model has): every token is turned by the number of its sequence's tokens in front of it, on all axes alike.
    ``window`` and ``window_first`` are paged_attention's ``window`` and ``keep_first``.  With ``scale_blocks`` a
    float8_e4m3fn cache has that many scales a page for each head, found as the rows are written.  A budget goes
    with neither (evicted rows leave their blocks, and the positions that a window counts).
    """

    def __init__(self, experts, w_qkv, w_out, w_router, *, kv_heads, head_dim, top_k, sequences, pages, page_size=16,
                 max_positions, cache_dtype=torch.bfloat16, k_scale=None, v_scale=None, sinks=None, budget=None,
                 slack=256, keep_first=4, keep_last=None, rotary=None, window=0, window_first=0, scale_blocks=None):
        dev = w_qkv.device
        if budget is not None and (window or scale_blocks):
            raise ValueError("a budget goes neither with a window nor with scale_blocks")
        if scale_blocks is not None:
            if cache_dtype is not torch.float8_e4m3fn or scale_blocks < 1 or page_size % scale_blocks:
                raise ValueError("scale_blocks are equal parts of a float8_e4m3fn cache's pages")
            if k_scale is not None or v_scale is not None:
                raise ValueError("with scale_blocks the cache has its own scales")
            k_scale, v_scale = (torch.zeros((pages, kv_heads, scale_blocks), device=dev) for _ in range(2))
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
        self.rotary, self.scale_blocks, self.sees = rotary, scale_blocks, dict(window=window, keep_first=window_first)
        self.positions = torch.zeros(sequences, dtype=torch.int32, device=dev)      # of the next tokens
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

    def _turned(self, q, k, positions):
        """Queries and keys as the attention and the cache take them.  What the attention would refuse of them where
        blocks have scales, which grow with what is written, is refused ahead of the cache."""
        if q.shape != (k.shape[0], self.heads, self.head_dim):
            raise ValueError("q must be [tokens, Hq, D]")
        if self.scale_blocks and q.dtype is not k.dtype:
            raise ValueError("with scale_blocks q must be of k's type")
        if self.rotary is None:
            return q, k
        sections = self.rotary.get("sections")
        return qk_norm_rope(q, k, positions if sections is None else positions.expand(len(sections), -1), **self.rotary)

    def prefill(self, k, v, lengths, q=None):
        """Keys and values [tokens, Hkv, D] of pieces of the sequences' prompts, one behind the other, `lengths` of
        them each; with their queries [tokens, Hq, D] also the attention of these tokens."""
        if q is None and self.rotary is not None:
            raise ValueError("with rotary positions the keys come with their queries")
        count = torch.tensor(lengths, dtype=torch.int32)
        starts = torch.cat([torch.zeros(1, dtype=torch.int32), count.cumsum(0).to(torch.int32)]).to(k.device)
        count = count.to(k.device)
        if q is not None:
            if sum(lengths) != k.shape[0] or min(lengths, default=0) < 0:
                raise ValueError("lengths must add up to the tokens")
            positions = None
            if self.rotary is not None:
                # of a token: its sequence's next position and how many of the call's tokens are in front of it
                first = (self.positions - starts[:-1]).repeat_interleave(count.long(), output_size=k.shape[0])
                positions = first + torch.arange(k.shape[0], dtype=torch.int32, device=k.device)
            q, k = self._turned(q, k, positions)
        out = None
        with self._grown(lengths):
            kv_cache_append(k, v, self.k_cache, self.v_cache, self.table, self.lens_dev, query_start=starts, **self.scales)
            if q is not None:
                out = paged_attention(q, self.k_cache, self.v_cache, self.table, self.lens_dev, query_start=starts,
                                      max_len=max(self.lens), sinks=self.sinks, **self.sees, **self.scales)
        self.positions += count
        return out

    def attend(self, q, k, v):
        """Attention of one new token of every sequence: q [B, Hq, D], its k and v [B, Hkv, D]."""
        q, k = self._turned(q, k, self.positions)
        with self._grown([1] * len(self.lens)):
            kv_cache_append(k, v, self.k_cache, self.v_cache, self.table, self.lens_dev, **self.scales)
            out = paged_attention(q, self.k_cache, self.v_cache, self.table, self.lens_dev, max_len=max(self.lens),
                                  sinks=self.sinks, weight_sums=self.sums, **self.sees, **self.scales)
        self.positions += 1
        return out

    def read(self, dtype=None):
        """Every sequence's cached keys and values, one behind the other: (k, v) [positions, Hkv, D]."""
        starts = torch.tensor([0, *self.lens]).cumsum(0).to(torch.int32).to(self.table.device)
        return kv_cache_read(self.k_cache, self.v_cache, self.table, self.lens_dev, query_start=starts, tokens=sum(self.lens),
                             dtype=dtype, **self.scales)

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


def _example(config, sequences, context, steps, budget, heads, kv_heads, head_dim, seed=0, rotary=False, window=0,
             window_first=0, scale_blocks=None):
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
                        max_positions=max(longest, (budget or 0) + 256), budget=budget, slack=32, window=window,
                        window_first=window_first, scale_blocks=scale_blocks,
                        cache_dtype=torch.float8_e4m3fn if scale_blocks else torch.bfloat16,
                        rotary=dict(inv_freq=1e4 ** -(torch.arange(0, head_dim, 2, device=dev) / head_dim)) if rotary else None)
    tokens = sequences * context
    layer.prefill(normal(tokens, kv_heads, head_dim), normal(tokens, kv_heads, head_dim), [context] * sequences,
                  q=normal(tokens, heads, head_dim) if rotary else None)
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
    ap.add_argument("--rotary", action="store_true", help="norm and rotation of queries and keys, and the prompts' attention")
    ap.add_argument("--window", type=int, default=0, help="positions a token sees (0: all)")
    ap.add_argument("--window-first", type=int, default=0, help="first positions that stay visible beside the window")
    ap.add_argument("--scale-blocks", type=int, default=None, help="an 8-bit cache with so many scales a page")
    a = ap.parse_args()
    seconds, layer = _example(a.config, a.sequences, a.context, a.steps, a.budget, a.heads, a.kv_heads, a.head_dim,
                              rotary=a.rotary, window=a.window, window_first=a.window_first, scale_blocks=a.scale_blocks)
    print(f"{a.sequences} sequences, {seconds * 1e6:.0f} us a step of the layer, "
          f"{max(layer.lens)} positions in the longest cache")
