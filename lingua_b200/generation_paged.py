"""Generation with a paged KV cache.

Same contract as ``generation.PackedCausalTransformerGenerator`` (apps/main/generate.py:140-400), selected by
``page_size > 0``. Sequences take pages as they grow, so that

* a prompt may be prefilled in chunks (``prefill_chunk`` tokens per forward pass) over what earlier chunks left in the cache,
* several samples of one prompt (``samples_per_prompt``) share its pages and are prefilled once,
* with ``attention_window`` a sequence holds only the pages of its window and of the first ``attention_sinks`` tokens,
  however long it gets.

A layer of a step is two launches besides the products: rotary embedding with the write to the cache, and attention over it.
"""
from __future__ import annotations

from typing import List

import torch
import torch.nn as nn

from .generation import (PackedCausalTransformerGenerator, PackedCausalTransformerGeneratorArgs, lengths_to_start_ids)
from .models.transformer import Attention
from .ops.paged import HEAD_DIMS, paged_append, paged_attention
from .paged_cache import PagedCache


class PagedPlan:
    """What the current forward pass does with the cache; shared by all layers."""

    def __init__(self, window: int = 0, sinks: int = 0):
        self.window, self.sinks = window, sinks
        self.table = None  # [n, cols] int32
        self.kv_len = None  # [n] int32, the tokens of this pass included
        self.cu_q = None  # [n + 1] int32, None: one token per sequence
        self.max_q = 1


class PagedKVCache(nn.Module):
    """One layer's view of the cache, in the place of ``generation.KVCache``."""

    rotates = True  # the native path hands over unrotated projections

    def __init__(self, cache: PagedCache, layer: int, plan: PagedPlan):
        super().__init__()
        self.cache, self.layer, self.plan = cache, layer, plan

    def native_attention(self, q, k, v, cs=None):
        pl = self.plan
        kp, vp = self.cache.layer(self.layer)
        q = paged_append(q, k, v, kp, vp, pl.table, pl.kv_len, pl.cu_q, cs)
        o = paged_attention(q, kp, vp, pl.table, pl.kv_len, pl.cu_q, pl.max_q, window=pl.window, sinks=pl.sinks)
        return o.view(q.shape[0], -1)

    def attend(self, q, k, v, tok_idx=None):
        """Reference path: q / k / v are [1, T, heads, Dh], rotated already."""
        return self.native_attention(q[0], k[0], v[0]).view(q.shape)


class PagedCausalTransformerGenerator(PackedCausalTransformerGenerator):
    def __init__(self, cfg: PackedCausalTransformerGeneratorArgs, model: nn.Module, tokenizer):
        super().__init__(cfg, model, tokenizer, paged=True)
        if cfg.samples_per_prompt < 1 or cfg.attention_sinks < 0 or (cfg.attention_window or 0) < 0:
            raise ValueError("samples_per_prompt must be positive, attention_window and attention_sinks not negative")
        if cfg.prefill_chunk is not None and cfg.prefill_chunk < 1:
            raise ValueError("prefill_chunk must be positive")
        self.page_size, self.prefill_chunk, self.samples = cfg.page_size, cfg.prefill_chunk, cfg.samples_per_prompt
        window = cfg.attention_window
        if window is None:
            window = getattr(model, "sliding_window", None)
        self.plan = PagedPlan(window or 0, cfg.attention_sinks)
        self._layers = [m for m in model.modules() if isinstance(m, Attention)]
        p = next(model.parameters())
        if p.is_cuda and (p.dtype != torch.bfloat16 or self._layers[0].head_dim not in HEAD_DIMS):
            raise ValueError(f"on a GPU the paged cache takes bf16 models with head dims {HEAD_DIMS}")
        self.cache = None
        self._seqs: List[int] = []

    # ---- cache
    def cache_need(self, prompt_len: int) -> int:
        """Cache slots a prompt and its samples can come to hold."""
        P = self.page_size
        shared = prompt_len // P  # pages of the prompt that are never written again
        own = (prompt_len + self.max_gen_len + P - 1) // P - shared
        return (shared + self.samples * own) * P

    def prompt_room(self) -> int:
        """Longest prompt such that it and all shorter ones fit (rounding to pages makes some shorter ones need more)."""
        slots, n = max(1, self.max_tokens // self.page_size) * self.page_size, 0
        while n < self.max_tokens and self.cache_need(n + 1) <= slots:
            n += 1
        if n == 0:
            raise ValueError(f"max_tokens={self.max_tokens} has no room for a prompt and {self.samples} x {self.max_gen_len} new tokens")
        return n

    def clear_cache(self):
        if self.cache is None:
            at, p = self._layers[0], next(self.model.parameters())
            n_pages = max(1, self.max_tokens // self.page_size)
            self.cache = PagedCache(len(self._layers), n_pages, self.page_size, at.n_kv_heads, at.head_dim, p.dtype, p.device)
        self._drop_sequences()
        for i, m in enumerate(self._layers):
            m.kv_cache = PagedKVCache(self.cache, i, self.plan)

    def _drop_sequences(self):
        for s in self._seqs:
            self.cache.free(s)
        self._seqs = []

    def release_cache(self):
        self._drop_sequences()
        for m in self._layers:
            m.kv_cache = None
        self.cache = self._graph = self._g_out = None

    # ---- prompts
    def prefill(self, tokens: torch.Tensor, lengths: torch.Tensor):
        """tokens [1, T], the prompts one after the other. Returns their logits [1, T, vocab]."""
        self.clear_cache()
        lens = lengths.tolist()
        self._seqs = [self.cache.add() for _ in lens]
        starts = lengths_to_start_ids(lengths).tolist()
        out = None
        for part in self._passes(lens):
            ids = [self._seqs[i] for i, _, _ in part]
            self.cache.reserve(ids, [n for _, _, n in part])
            rows = torch.cat([torch.arange(starts[i] + at, starts[i] + at + n) for i, at, n in part]).to(tokens.device)
            pos = torch.cat([torch.arange(at, at + n) for _, at, n in part]).to(tokens.device)
            self._aim(ids, [n for _, _, n in part])
            logits = self.model(tokens[:, rows], tok_idx=pos.view(1, -1))
            if out is None and rows.numel() == tokens.shape[1]:
                out = logits
            else:
                if out is None:
                    out = logits.new_empty(1, tokens.shape[1], logits.shape[2])
                out[:, rows] = logits
            if self.plan.window:
                for s in ids:
                    self.cache.release_behind(s, self.plan.window, self.plan.sinks)
        self.setup_generation(lengths)
        return out

    def _passes(self, lens):
        """Lists of (prompt, first token, number of tokens), each list one forward pass of at most ``prefill_chunk`` tokens."""
        if self.prefill_chunk is None:
            return [[(i, 0, n) for i, n in enumerate(lens)]]
        passes, part, room = [], [], self.prefill_chunk
        for i, n in enumerate(lens):
            at = 0
            while at < n:
                take = min(n - at, room)
                part.append((i, at, take))
                at, room = at + take, room - take
                if room == 0:
                    passes.append(part)
                    part, room = [], self.prefill_chunk
        return passes + ([part] if part else [])

    def _aim(self, ids, n_new):
        pl, dev = self.plan, next(self.model.parameters()).device
        pl.table = self.cache.table(ids).to(dev)
        pl.kv_len = torch.tensor([self.cache.length(s) for s in ids], dtype=torch.int32).to(dev)
        cu = [0]
        for n in n_new:
            cu.append(cu[-1] + n)
        pl.cu_q, pl.max_q = torch.tensor(cu, dtype=torch.int32).to(dev), max(n_new)

    # ---- decoding: the plan's tensors stay in place from here on, a captured step reads them
    def setup_generation(self, lengths: torch.Tensor):
        if self.samples > 1:
            self._seqs = [t for s in self._seqs for t in (s, *self.cache.fork(s, self.samples - 1))]
        pl, dev = self.plan, next(self.model.parameters()).device
        lens = [self.cache.length(s) for s in self._seqs]
        self._cols = (max(lens) + self.max_gen_len + self.page_size) // self.page_size
        pl.table = self.cache.table(self._seqs, self._cols).to(dev)
        pl.kv_len = torch.tensor(lens, dtype=torch.int32).to(dev)
        pl.cu_q, pl.max_q = None, 1
        self._graph, self._eager_steps = None, 0

    def _step(self, token: torch.Tensor):
        pl = self.plan
        pl.kv_len.add_(1)
        return self.model(token, tok_idx=(pl.kv_len - 1).long().view(1, -1))

    def generate_next_token(self, current_token: torch.Tensor):
        changed = False
        if self.plan.window:
            for s in self._seqs:
                changed |= self.cache.release_behind(s, self.plan.window, self.plan.sinks)
        changed |= self.cache.reserve(self._seqs, [1] * len(self._seqs))
        if changed:
            table = self.cache.table(self._seqs)
            if table.shape[1] > self._cols:  # past max_gen_len: a wider table, and a captured step is stale
                self._cols, self._graph = 2 * table.shape[1], None
                self.plan.table = torch.full((len(self._seqs), self._cols), -1, dtype=torch.int32, device=self.plan.table.device)
            self.plan.table[:, :table.shape[1]] = table.to(self.plan.table.device)
        if not (self.use_graph and current_token.is_cuda):
            return self._step(current_token)
        if self._graph is None:
            if self._eager_steps < 2:  # kernels, allocator and status word come to life outside the capture
                self._eager_steps += 1
                return self._step(current_token)
            self._g_token = current_token.clone()
            graph = torch.cuda.CUDAGraph()
            torch.cuda.synchronize()
            with torch.cuda.graph(graph):
                out = self._step(self._g_token)
            self._graph, self._g_out = graph, out
        self._g_token.copy_(current_token)
        self._graph.replay()
        return self._g_out
