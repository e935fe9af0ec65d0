"""Generation and scoring with the hierarchical byte model.

The prompt batch is prefilled with one pass over all stages (rows are sequences, padded on the right, every
stage flattened to one packed row for its key/value caches). Decoding then feeds one byte per sequence: the
byte-level encoder always runs; a sequence goes one stage deeper only when the new byte closes a unit of that
level (its level comes from the regex pooler over the sequence's recent bytes, or from the model's own level
head); on the way back a stage that did not run in this step is represented by its last output, repeated with
the distance counter that selects the up-projection. What the reference keeps as "residual", "decoder" and
"local position" caches (apps/aunet/generate.py:223-368) are the ``resid``, ``deep_out`` and ``dist`` tensors
here. Differences: sequences are rows of a batch instead of one packed row, so a decode step is a handful of
dense calls on [n_active, dim] tensors; the final norm is applied before the vocabulary head, as in training
(the reference's generator skips it); ``use_regex_for_level_mask=False`` selects the learned level head.
On a GPU, stages with heads of 128 use the native prefill and decode-attention kernels, narrower stages the
generic cached attention."""
from __future__ import annotations

from dataclasses import dataclass
from pathlib import Path
from typing import List, Optional

import torch
import torch.nn.functional as TF

from .checkpoint import CONSOLIDATE_NAME
from .config import dataclass_from_dict, load_yaml
from .data.regex_cutting import RegexArgs, RegexPool
from .generation import (CachePlan, KVCache, LogitControls, PackedCausalTransformerGeneratorArgs, batch_prompts, sample_tokens)
from .models.aunet import HierarchicalArgs, HierarchicalTransformer, make_level_plan
from .models.transformer import Attention, RotaryEmbedding
from .tokenizer import build_tokenizer


@dataclass
class PackedHierarchicalCausalTransformerGeneratorArgs(PackedCausalTransformerGeneratorArgs):
    regex_buffer_size: Optional[int] = None  # bytes of history the regex pooler sees per sequence (None = all)
    use_regex_for_level_mask: bool = True  # False: levels of generated bytes come from the model's level head


class _StageCache:
    """Key/value caches of one stage: ``cap`` slots per sequence, one plan shared by the stage's layers."""

    def __init__(self, stage, n_seqs: int, cap: int):
        self.stage, self.cap, self.plan = stage, cap, CachePlan()
        self.window = stage.sliding_window or 0
        for m in stage.modules():
            if isinstance(m, Attention):
                p = next(m.parameters())
                m.kv_cache = KVCache(n_seqs * cap, m.n_kv_heads, m.head_dim, p.dtype, p.device, self.plan)

    def prefill(self, h: torch.Tensor) -> torch.Tensor:
        """h [n, L, dim]: rows are written to their own slot ranges and attend within the row only."""
        n, L, D = h.shape
        dev = h.device
        row = torch.arange(n, device=dev).repeat_interleave(L)
        pos = torch.arange(L, device=dev).repeat(n)
        pl = self.plan
        pl.mode, pl.window = "prefill", self.window
        pl.slots = row * self.cap + pos
        pl.doc_start = (row * L).int().view(1, -1).contiguous()
        return self.stage(h.reshape(1, n * L, D), tok_idx=pos.view(1, -1)).view(n, L, D)

    def step(self, x: torch.Tensor, seqs: torch.Tensor, count: torch.Tensor) -> torch.Tensor:
        """x [m, dim]: one new position for each sequence in ``seqs``, which has ``count`` cached positions."""
        pl = self.plan
        pl.mode = "decode"
        seen = count + 1
        if self.window:
            seen = seen.clamp(max=self.window)
        pl.start = (seqs * self.cap + count + 1 - seen).int().contiguous()
        pl.len = seen.int().contiguous()
        return self.stage(x.unsqueeze(0), tok_idx=count.view(1, -1)).squeeze(0)

    def release(self):
        for m in self.stage.modules():
            if isinstance(m, Attention):
                m.kv_cache = None


class PackedHierarchicalCausalTransformerGenerator:
    """Same contract as the flat generator: ``generate(prompts) -> (texts, log-likelihoods, greedy matches)``."""

    def __init__(self, cfg: PackedHierarchicalCausalTransformerGeneratorArgs, model: HierarchicalTransformer, tokenizer,
                 regex_pool: RegexPool):
        if LogitControls(cfg) or cfg.page_size or cfg.prefill_chunk or cfg.samples_per_prompt != 1 or cfg.attention_window \
                or cfg.attention_sinks:
            raise ValueError("the byte model's generator has neither logit controls nor a paged cache")
        self.model, self.tokenizer, self.regex_pool = model, tokenizer, regex_pool
        self.temperature, self.top_p, self.top_k = cfg.temperature, cfg.top_p, cfg.top_k
        self.max_gen_len, self.max_tokens, self.max_prompt_len = cfg.max_gen_len, cfg.max_tokens, cfg.max_prompt_len
        self.until = cfg.until
        self.regex_buffer_size, self.use_regex = cfg.regex_buffer_size, cfg.use_regex_for_level_mask
        self.device = cfg.device if (cfg.device != "cuda" or torch.cuda.is_available()) else "cpu"
        self.show_progress = cfg.show_progress
        self.n_levels = len(model.encoders)
        self.caches: List[_StageCache] = []

    # ------------------------------------------------------------------ prefill
    def prefill(self, tokens: torch.Tensor, levels: torch.Tensor, lengths: torch.Tensor):
        """tokens / levels [n, L] right-padded (padding has level 0). Returns logits [n, L, vocab]."""
        m, n_lv = self.model, self.n_levels
        n, L = tokens.shape
        dev = tokens.device
        valid = torch.arange(L, device=dev).unsqueeze(0) < lengths.unsqueeze(1)
        masks, _, _ = m.get_pool_mask(levels * valid, None, return_idcs=False, force_first=True)
        counts = [lengths] + [mk.sum(1) for mk in masks]  # real positions of every sequence at every level
        widths = [L] + [max(1, int(c.max())) for c in counts[1:]]
        stages = [*m.encoders, m.trunk]
        room = self.max_gen_len + 1
        enc_c = [_StageCache(s, n, min(w + room, max(s.max_seqlen, w + 1))) for s, w in zip(stages, widths)]
        dec_c = [_StageCache(s, n, c.cap) for s, c in zip(m.decoders, enc_c)]
        self.caches, self.enc_c, self.dec_c = enc_c + dec_c, enc_c, dec_c
        plans = [make_level_plan(masks[k], widths[k], widths[k + 1], m.transitions[k].repeat,
                                 m.transitions[k].indexed_matmul) for k in range(n_lv)]
        rows = torch.arange(n, device=dev)
        last = [(c - 1).clamp(min=0) for c in counts]
        self.count = [c.clone() for c in counts]
        self.resid, self.deep_out, self.dist = [None] * n_lv, [None] * (n_lv + 1), [None] * n_lv
        x = m.tok_embeddings(tokens)
        skips = []
        for k in range(n_lv):
            x = enc_c[k].prefill(x)
            skips.append(x)
            self.resid[k] = x[rows, last[k]].clone()
            self.dist[k] = (plans[k].position[rows, last[k]] + 1) % m.transitions[k].max_pos \
                if plans[k].position is not None else torch.zeros(n, dtype=torch.long, device=dev)
            x = m.transitions[k].down(x, plans[k])
        x = enc_c[n_lv].prefill(x)
        self.deep_out[n_lv] = x[rows, last[n_lv]].clone()
        for k in reversed(range(n_lv)):
            x = m.transitions[k].up(x, skips[k], plans[k])
            if m.adding_residuals[k]:
                x = skips[k] + x
            x = dec_c[k].prefill(x)
            self.deep_out[k] = x[rows, last[k]].clone()
        self.features = self.deep_out[0]
        return m.vocab(m.vocab_norm(x))

    # ------------------------------------------------------------------ one byte per sequence
    def generate_next_token(self, tokens: torch.Tensor, levels: torch.Tensor) -> torch.Tensor:
        """tokens / levels [n]: the byte just chosen for every sequence and its pooling level. Logits [n, vocab]."""
        m, n_lv = self.model, self.n_levels
        n = tokens.shape[0]
        seqs = torch.arange(n, device=tokens.device)
        x = m.tok_embeddings(tokens)
        active = [seqs]  # sequences for which this byte is a position of level k
        for k in range(n_lv):
            a = active[k]
            x = self.enc_c[k].step(x, a, self.count[k][a])
            self.resid[k][a] = x
            deeper = levels[a] > k
            self.dist[k][a[deeper]] = 0  # a new unit starts: the distance counter restarts
            active.append(a[deeper])
            if active[-1].numel() == 0:
                break
            x = m.transitions[k]._down_map(x[deeper])
        if len(active) == n_lv + 1 and active[n_lv].numel() > 0:
            a = active[n_lv]
            self.deep_out[n_lv][a] = self.enc_c[n_lv].step(x, a, self.count[n_lv][a])
            self.count[n_lv][a] += 1
        for k in reversed(range(len(active) - 1)):
            a, t = active[k], m.transitions[k]
            if a.numel() == 0:
                continue
            u = self._up_one(t, self.deep_out[k + 1][a], self.dist[k][a], levels[a] > k)
            x = self.resid[k][a] + u if m.adding_residuals[k] else u
            self.deep_out[k][a] = self.dec_c[k].step(x, a, self.count[k][a])
            self.count[k][a] += 1
            self.dist[k][a] = (self.dist[k][a] + 1) % t.max_pos
        self.features = self.deep_out[0]
        return m.vocab(m.vocab_norm(self.deep_out[0]))

    @staticmethod
    def _up_one(t, deep: torch.Tensor, dist: torch.Tensor, is_boundary: torch.Tensor) -> torch.Tensor:
        x = t.up_norm(deep) if hasattr(t, "up_norm") else deep
        if t.repeat:
            if t.indexed_matmul:
                xi = t.indexed_norm(x) if hasattr(t, "indexed_norm") else x
                return t._up_map(x) + t.indexed_linear(xi.unsqueeze(0), dist.unsqueeze(0)).squeeze(0)
            return t._up_map(x + t.pos_encoding(dist).to(x.dtype))
        return t._up_map(x) * is_boundary.to(x.dtype).unsqueeze(-1)  # scatter pooling: boundaries only

    def release_cache(self):
        for c in self.caches:
            c.release()
        self.caches = []

    def _levels_of(self, current: torch.Tensor) -> torch.Tensor:
        if self.model.lambda_level > 0 and not self.use_regex:
            return self.model._level_mask_logits(self.features, current).argmax(dim=-1)
        lv = self.regex_pool.get_levels_mask_gen(current.tolist())
        return torch.tensor(lv, dtype=torch.long, device=current.device)

    @torch.inference_mode()
    def generate(self, prompts: List[str]):
        prompts = [self.tokenizer.encode(p, add_bos=True, add_eos=False) for p in prompts]
        limit = self.model.encoders[0].max_seqlen if self.n_levels else self.model.trunk.max_seqlen
        max_prompt_len = self.max_prompt_len or min(limit - self.max_gen_len, self.max_tokens - self.max_gen_len)
        prompts = [p[-max_prompt_len:] for p in prompts]
        padded_lengths = [len(p) + self.max_gen_len for p in prompts]
        generation, loglikelihood, greedy = [], [], []
        max_until = max((len(e) for e in self.until), default=1)
        batches = batch_prompts(prompts, self.max_tokens, lengths=padded_lengths)
        if self.show_progress:
            from tqdm import tqdm

            batches = tqdm(batches)
        for batch in batches:
            n, L = len(batch), max(len(p) for p in batch)
            lengths = torch.tensor([len(p) for p in batch], device=self.device)
            flat = self.regex_pool.get_levels_mask_prefill(batch, size=self.regex_buffer_size, force_first=True)
            tokens = torch.zeros(n, L, dtype=torch.long)
            levels = torch.zeros(n, L, dtype=torch.long)
            o = 0
            for i, p in enumerate(batch):
                tokens[i, :len(p)] = torch.tensor(p)
                levels[i, :len(p)] = torch.tensor(flat[o:o + len(p)])
                o += len(p)
            prompt_logits = self.prefill(tokens.to(self.device), levels.to(self.device), lengths)
            rows = torch.arange(n, device=self.device)
            current = sample_tokens(prompt_logits[rows, lengths - 1].unsqueeze(0), self.temperature, self.top_p,
                                    self.top_k).squeeze(0)
            generated = [[t] for t in current.tolist()]
            is_done = [False] * n
            for _ in range(1, self.max_gen_len):
                logits = self.generate_next_token(current, self._levels_of(current))
                nxt = sample_tokens(logits.unsqueeze(0).clone(), self.temperature, self.top_p, self.top_k).squeeze(0)
                for i, tok in enumerate(nxt.tolist()):
                    if not is_done[i]:
                        generated[i].append(tok)
                        is_done[i] = tok == self.tokenizer.eos_id
                        if self.until and not is_done[i]:
                            tail = self.tokenizer.decode(generated[i][-max_until:])
                            is_done[i] = any(e in tail for e in self.until)
                if all(is_done):
                    break
                current = nxt
            generation.extend(self.tokenizer.decode(g) for g in generated)
            for i, p in enumerate(batch):
                x = prompt_logits[i, :len(p) - 1].float()
                y = torch.tensor(p[1:], device=x.device)
                loglikelihood.append(-TF.cross_entropy(x, y, reduction="none").cpu())
                greedy.append((x.argmax(dim=-1) == y).cpu())
            self.release_cache()
        return generation, loglikelihood, greedy


def load_consolidated_model_and_tokenizer(consolidated_path, model_cls=HierarchicalTransformer,
                                          model_args_cls=HierarchicalArgs):
    """(model, tokenizer, regex pooler, training config) from ``consolidated.pth`` + ``params.json``
    (apps/aunet/generate.py:42-69 of the reference)."""
    ckpt = Path(consolidated_path)
    config = load_yaml(str(ckpt / "params.json"))
    dtype = dict(fp32=torch.float32, fp16=torch.float16, bf16=torch.bfloat16)[config["distributed"]["model_dtype"]]
    margs = dataclass_from_dict(model_args_cls, config["model"], strict=False)
    tok = config["data"]["tokenizer"]
    tokenizer = build_tokenizer(tok["name"], tok.get("path"))
    model = model_cls(margs)
    model.load_state_dict(torch.load(ckpt / CONSOLIDATE_NAME, weights_only=True)["model"])
    if torch.cuda.is_available():
        model = model.cuda().to(dtype)
    model = model.eval()
    for mod in model.modules():
        if isinstance(mod, RotaryEmbedding):
            mod.reset_parameters()  # non-persistent tables: not in the checkpoint
    regex = (config["data"].get("regex") or {}).get("strategy") or {}
    return model, tokenizer, RegexPool(RegexArgs(strategy=dict(regex))), config


class _Bound(PackedHierarchicalCausalTransformerGenerator):
    """Adapter to the (cfg, model, tokenizer) constructor that the shared evaluation driver calls."""
    regex_pool_for_eval: Optional[RegexPool] = None

    def __init__(self, cfg, model, tokenizer):
        super().__init__(cfg, model, tokenizer, type(self).regex_pool_for_eval)


def launch_eval(cfg):
    """Harness tasks and validation perplexity for a hierarchical checkpoint (apps/aunet/eval.py of the
    reference): the shared driver with this module's loader and generator."""
    from . import evaluation

    def loader(path):
        model, tokenizer, pool, config = load_consolidated_model_and_tokenizer(path)
        _Bound.regex_pool_for_eval = pool
        return model, tokenizer, config

    return evaluation.launch_eval(cfg, generator_cls=_Bound, loader=loader)


def main(argv=None):
    """``python -m apps.aunet.generate ckpt=<consolidated dir> max_gen_len=64 ...``: prompts from stdin."""
    import time

    from .config import from_cli

    cfg = from_cli(argv)
    gen_cfg = dataclass_from_dict(PackedHierarchicalCausalTransformerGeneratorArgs, cfg, strict=False)
    model, tokenizer, pool, _ = load_consolidated_model_and_tokenizer(cfg["ckpt"])
    generator = PackedHierarchicalCausalTransformerGenerator(gen_cfg, model, tokenizer, pool)
    prompts = []
    while True:
        prompt = input("Enter a prompt (or press enter to finish): ")
        if not prompt:
            break
        prompts.append(prompt)
    t0 = time.time()
    generation, _, _ = generator.generate(prompts)
    dt = time.time() - t0
    total = sum(len(tokenizer.encode(g, False, False)) for g in generation)
    for i, g in enumerate(generation):
        print(f"\nPrompt {i + 1}: {prompts[i]}")
        print(f"Generated Text: {g}")
    print(f"\nTokens per second: {total / dt:.2f}")
