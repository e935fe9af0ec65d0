"""Penalties, bias and grammar mask on the logits of a sampling step (``csrc/logits.cu``).

Runs between the model and ``generation.sample_tokens`` (the step of apps/main/generate.py:49-63 that the reference takes
on unmodified logits)."""
from __future__ import annotations

from typing import Optional, Union

import torch

from . import _lib
from .paged import _on, _refuse, _tracked

Knob = Optional[Union[float, torch.Tensor]]


def _knob(value: Knob, name: str, N: int, neutral: float, dev: int):
    """(per-row tensor or None, scalar) of a penalty given as a number, an fp32 [N] tensor or None."""
    if value is None:
        return None, neutral
    if isinstance(value, torch.Tensor):
        if value.shape != (N,) or value.dtype is not torch.float32 or not value.is_contiguous() or value.get_device() != dev:
            raise ValueError(f"{name} must be a number or a contiguous fp32 [N] tensor on the logits' device")
        return value, neutral
    return None, float(value)


def _rows(t: Optional[torch.Tensor], dtype: torch.dtype, shape, dev: int) -> bool:
    """An operand that is absent, or as the kernel reads it: rows of ``shape`` without gaps inside them."""
    return t is None or (t.dtype is dtype and t.shape == shape and t.get_device() == dev
                         and (t.is_contiguous() or shape[-1] <= 1 or t.stride(-1) == 1))


def _torn(out: torch.Tensor, logits: torch.Tensor) -> bool:
    """Whether ``out`` overlaps the logits without being them: a block would read what another one has written."""
    a, b = out.data_ptr(), logits.data_ptr()
    if out.numel() == 0 or (a == b and (out.shape[0] <= 1 or out.stride(0) == logits.stride(0))):
        return False
    es, V = out.element_size(), out.shape[1]
    end = [t.data_ptr() + ((t.shape[0] - 1) * t.stride(0) + V) * es for t in (out, logits)]
    if a >= end[1] or b >= end[0]:
        return False
    if out.shape[0] <= 1 or out.stride(0) != logits.stride(0):
        return True
    row = out.stride(0) * es  # rows of one spacing may lie side by side
    return not V * es <= (a - b) % row <= row - V * es


def penalize_logits_ref(logits, history, history_len, prompt_len=None, repetition=None, presence=None, frequency=None,
                        bias=None, allowed=None):
    N, V = logits.shape
    x = logits.double() if logits.dtype == torch.float64 else logits.float()
    at = torch.arange(history.shape[1], device=x.device).view(1, -1)
    live = (at < history_len.view(N, 1)) & (history >= 0) & (history < V)
    new = live if prompt_len is None else live & (at >= prompt_len.view(N, 1))
    ids = history.clamp(0, V - 1)
    seen = torch.zeros_like(x).scatter_add_(1, ids, live.to(x.dtype))
    made = torch.zeros_like(x).scatter_add_(1, ids, new.to(x.dtype))
    rep, pres, freq = (k.view(N, 1).to(x.dtype) if isinstance(k, torch.Tensor) else (neutral if k is None else float(k))
                       for k, neutral in ((repetition, 1.0), (presence, 0.0), (frequency, 0.0)))
    z = torch.where(seen > 0, torch.where(x > 0, x / rep, x * rep), x)
    z = torch.where(made > 0, z - (pres + freq * made), z)
    if bias is not None:
        z = z + bias.to(x.dtype)
    if allowed is not None:
        tok = torch.arange(V, device=x.device)
        z = z.masked_fill(((allowed[:, tok // 32] >> (tok % 32).int()) & 1) == 0, float("-inf"))
    return z.to(logits.dtype)


def penalize_logits(logits: torch.Tensor, history: torch.Tensor, history_len: torch.Tensor,
                    prompt_len: Optional[torch.Tensor] = None, repetition: Knob = None, presence: Knob = None,
                    frequency: Knob = None, bias: Optional[torch.Tensor] = None, allowed: Optional[torch.Tensor] = None,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Logits [N, V] (bf16 or fp32) after the penalties of each row's history, in their own dtype.

    history       int64 [N, L] token ids, of which the first ``history_len[n]`` (int32) count; ids outside the vocabulary
                  are ignored
    prompt_len    int32 [N]: entries from here on were generated (None: all of them)
    repetition    > 0; a token of the history has its logit divided by this if positive, else multiplied by it
    presence      subtracted once from every generated token's logit
    frequency     subtracted once per occurrence among the generated tokens
    bias          fp32 [V] or [N, V], added
    allowed       int32 [N, ceil(V / 32)]: bit (t % 32) of word t / 32 clear means token t becomes -inf, whatever its logit
    out           destination: ``logits`` itself or memory apart from them; a new tensor by default

    The penalties are numbers or fp32 [N] tensors. A row whose mask allows nothing comes out as -inf everywhere."""
    _refuse(logits.dim() != 2, "logits must be [N, V]")
    N, V = logits.shape
    dev, dt = logits.get_device(), logits.dtype
    rep_t, rep = _knob(repetition, "repetition", N, 1.0, dev)
    _refuse(rep_t is None and not rep > 0.0, "repetition must be positive")
    pres_t, pres = _knob(presence, "presence", N, 0.0, dev)
    freq_t, freq = _knob(frequency, "frequency", N, 0.0, dev)
    i32 = torch.int32
    if not (dev >= 0 and (dt is torch.bfloat16 or dt is torch.float32) and N <= 65535 and history.dim() == 2
            and _rows(logits, dt, (N, V), dev) and _rows(history, torch.int64, (N, history.shape[1]), dev)
            and _rows(history_len, i32, (N,), dev) and _rows(prompt_len, i32, (N,), dev)
            and (bias is None or _rows(bias, torch.float32, (V,) if bias.dim() == 1 else (N, V), dev))
            and _rows(allowed, i32, (N, (V + 31) // 32), dev)
            and (out is None or (_rows(out, dt, (N, V), dev) and (N <= 1 or out.stride(0) >= V) and not _torn(out, logits)))
            and not _tracked(logits)):
        # something is unusual: the reference path, or words for what is wrong
        _refuse(history.dim() != 2 or history.shape[0] != N or history.dtype != torch.int64, "history must be int64 [N, L]")
        for t, name in ((history_len, "history_len"), (prompt_len, "prompt_len")):
            _refuse(t is not None and (t.shape != (N,) or t.dtype != i32), f"{name} must be int32 [N]")
        _refuse(bias is not None and (bias.dtype != torch.float32 or bias.shape not in ((V,), (N, V))),
                "bias must be fp32 [V] or [N, V]")
        _refuse(allowed is not None and (allowed.dtype != i32 or allowed.shape != (N, (V + 31) // 32)),
                "allowed must be int32 [N, ceil(V / 32)]")
        for t in (history, history_len, prompt_len, bias, allowed, out):
            _refuse(t is not None and t.device != logits.device, "all tensors must be on one device")
        if out is not None:
            _refuse(out.shape != logits.shape or out.dtype != dt, "out must have the logits' shape and dtype")
            _refuse(N > 1 and out.stride(0) < V, "rows of out must not overlap")
            _refuse(_torn(out, logits), "out must be the logits themselves or not overlap them")
        _refuse(_tracked(logits), "penalize_logits has no gradient")
        if not logits.is_cuda:
            z = penalize_logits_ref(logits, history, history_len, prompt_len, repetition, presence, frequency, bias, allowed)
            return z if out is None else out.copy_(z)
        _refuse(dt not in (torch.bfloat16, torch.float32), "the kernel takes bf16 and fp32 logits")
        _refuse(N > 65535, "too many rows")
        raise ValueError("rows must be contiguous")
    if out is None:
        out = torch.empty_like(logits, memory_format=torch.contiguous_format)
    if N == 0 or V == 0:
        return out
    args = _lib.PENALIZE_ARGS.pack(
        logits.data_ptr(), out.data_ptr(), history.data_ptr(), history_len.data_ptr(),
        *[0 if t is None else t.data_ptr() for t in (prompt_len, rep_t, pres_t, freq_t, bias, allowed)], N, V,
        history.shape[1], _lib.LB_BF16 if dt is torch.bfloat16 else _lib.LB_F32, rep, pres, freq,
        logits.stride(0), out.stride(0), history.stride(0), 0 if bias is None or bias.dim() == 1 else bias.stride(0),
        0 if allowed is None else allowed.stride(0))
    with _on(dev):
        rc = _lib.load().lb_penalize_logits(args, _lib.stream_ptr())
    _lib.check(rc, "lb_penalize_logits")
    return out
