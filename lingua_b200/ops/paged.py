"""Operators of a paged KV cache: append, attention, page copies (``csrc/paged_cache.cu``, ``csrc/paged_attention.cu``).

A cache layer is a pair of pools ``k_pages`` / ``v_pages`` [n_pages, page, Hkv, D]. Row ``s`` of ``block_table`` (int32
[n_seqs, cols]) names the page that holds positions ``[c * page, (c + 1) * page)`` of sequence ``s``; entries that no visible
position needs may hold anything. ``kv_len`` (int32 [n_seqs]) counts a sequence's keys including the new tokens of the call,
which are its last positions. New tokens are packed rows: ``cu_q`` (int32 [n_seqs + 1]) holds the first row of every sequence;
``cu_q=None`` means one token per sequence. Rows that belong to no sequence (behind ``cu_q[-1]``, or with a position below
zero, as for a sequence with ``kv_len`` 0) are padding: they come out as zeros and leave the cache alone.

What a page holds where no row of its sequence may look is never seen, NaN included. A NaN or infinity among the values that
one of the call's rows sees may reach the sequence's other rows too, as in a product with a masked matrix of probabilities.

The tables live on the device and may change between replays of a captured graph. A page id outside the pool, or a position
past the table (or past the rotary table), is skipped and recorded in the status word that ``_lib.check_status`` raises on;
what the call returns for such a sequence is finite and otherwise unspecified. These are inference operators: no gradients.

The paged cache plays the part of the fixed cache of apps/main/generate.py:104-137 and of the dense decode mask of
apps/main/generate.py:299-320.
"""
from __future__ import annotations

import math
from contextlib import nullcontext
from typing import Optional

import torch

from . import _lib

PAGE_SIZES = (16, 32, 64, 128, 256)
HEAD_DIMS = (64, 128)
MAX_POSITIONS = 1 << 30


def _refuse(cond: bool, msg: str) -> None:
    if cond:
        raise ValueError(msg)


def _strided(t: torch.Tensor, name: str) -> None:
    """Rows of channels that 16-byte accesses can read: unit channel stride, other strides positive multiples of 8."""
    st = t.stride()
    ok = st[-1] == 1 and t.data_ptr() % 16 == 0
    for n, s in zip(t.shape[:-1], st[:-1]):
        ok = ok and (n <= 1 or (s > 0 and s % 8 == 0))
    _refuse(not ok, f"{name} needs contiguous channels, 16-byte aligned rows and positive strides, got {tuple(st)}")


def _tracked(*ts: torch.Tensor) -> bool:
    if torch.is_grad_enabled():
        for t in ts:
            if t.requires_grad:
                return True
    return False


def _aligned(t: torch.Tensor) -> bool:
    """What ``_strided`` asks for, without the explanation."""
    if t.data_ptr() % 16 or t.stride(-1) != 1:
        return False
    if t.is_contiguous():
        return t.shape[-1] % 8 == 0
    return all(n <= 1 or (s > 0 and s % 8 == 0) for n, s in zip(t.shape[:-1], t.stride()[:-1]))


def _plain(*strides: int) -> bool:
    """Strides that need no look at the sizes (that of a dimension of size one may be anything)."""
    bits = 0
    for s in strides:
        bits |= s
    return not bits & 7 and min(strides) > 0


def _check_cache(q, k_pages, v_pages, block_table, kv_len, cu_q):
    """One pass over the conditions; ``_refuse_cache`` finds the words when one fails. Returns the sizes and strides that the
    kernels' argument blocks are made of, read once: (device, T, H, D, n_pages, page, Hkv, n_seqs, cols, stride of a table
    row, (strides of q), (of k_pages), (of v_pages)), the strides without that of the channels."""
    dev, dt, i32 = q.get_device(), q.dtype, torch.int32
    qs, ks, bs = q.shape, k_pages.shape, block_table.shape
    if len(qs) == 3 and len(ks) == 4 and len(bs) == 2 and dev >= 0 and dt is torch.bfloat16:
        (T, H, D), (n_pages, P, Hkv, Dk), (n, cols) = qs, ks, bs
        if (ks == v_pages.shape and Dk == D and D in HEAD_DIMS and P in PAGE_SIZES and n_pages > 0 and Hkv > 0
                and H > 0 and H % Hkv == 0 and k_pages.dtype is dt and v_pages.dtype is dt
                and block_table.dtype is i32 and kv_len.dtype is i32 and kv_len.shape == (n,)
                and dev == k_pages.get_device() == v_pages.get_device() == block_table.get_device() == kv_len.get_device()
                and kv_len.is_contiguous()
                and (T == n if cu_q is None else cu_q.dtype is i32 and cu_q.shape == (n + 1,)
                     and cu_q.get_device() == dev and cu_q.is_contiguous())
                and cols * P <= MAX_POSITIONS and not _tracked(q, k_pages, v_pages)):
            row, col = block_table.stride()
            (*q_st, q_c), (*k_st, k_c), (*v_st, v_c) = q.stride(), k_pages.stride(), v_pages.stride()
            if ((col == 1 or cols <= 1) and q_c == k_c == v_c == 1
                    and not (q.data_ptr() | k_pages.data_ptr() | v_pages.data_ptr()) & 15
                    and (_plain(*q_st, *k_st, *v_st) or _aligned(q) and _aligned(k_pages) and _aligned(v_pages))):
                return dev, T, H, D, n_pages, P, Hkv, n, cols, row, q_st, k_st, v_st
    _refuse_cache(q, k_pages, v_pages, block_table, kv_len, cu_q)
    return (dev, *qs, *ks[:3], *bs, block_table.stride(0), q.stride()[:2], k_pages.stride()[:3], v_pages.stride()[:3])


def _refuse_cache(q, k_pages, v_pages, block_table, kv_len, cu_q):
    _refuse(q.dim() != 3, "new tokens are packed rows [T, heads, D]")
    _refuse(k_pages.dim() != 4 or k_pages.shape != v_pages.shape, "k_pages and v_pages must both be [n_pages, page, Hkv, D]")
    H, D, Hkv = q.shape[1], q.shape[2], k_pages.shape[2]
    _refuse(k_pages.shape[3] != D, f"head dim of the cache ({k_pages.shape[3]}) is not that of the tokens ({D})")
    _refuse(Hkv < 1 or H < 1 or H % Hkv != 0, f"{H} query heads do not share {Hkv} key heads evenly")
    _refuse(block_table.dim() != 2 or block_table.dtype != torch.int32, "block_table must be int32 [n_seqs, cols]")
    n = block_table.shape[0]
    _refuse(kv_len.shape != (n,) or kv_len.dtype != torch.int32, "kv_len must be int32 [n_seqs]")
    if cu_q is None:
        _refuse(q.shape[0] != n, "without cu_q there is one token per sequence")
    else:
        _refuse(cu_q.shape != (n + 1,) or cu_q.dtype != torch.int32, "cu_q must be int32 [n_seqs + 1]")
    dev = q.device
    for t in (k_pages, v_pages, block_table, kv_len, cu_q):
        _refuse(t is not None and t.device != dev, "all tensors must be on one device")
    dt = q.dtype
    _refuse(k_pages.dtype != dt or v_pages.dtype != dt, "tokens and cache must have one dtype")
    _refuse(_tracked(q, k_pages, v_pages), "paged-cache operators have no gradient")
    _refuse(block_table.shape[1] * k_pages.shape[1] > MAX_POSITIONS, f"a sequence has at most {MAX_POSITIONS} positions")
    if not q.is_cuda:
        return
    _refuse(dt != torch.bfloat16, "the kernels take bf16")
    _refuse(D not in HEAD_DIMS, f"head dim must be one of {HEAD_DIMS}, got {D}")
    _refuse(k_pages.shape[1] not in PAGE_SIZES, f"page size must be one of {PAGE_SIZES}, got {k_pages.shape[1]}")
    _refuse(k_pages.shape[0] < 1, "the pool has no pages")
    _refuse(not kv_len.is_contiguous() or (cu_q is not None and not cu_q.is_contiguous())
            or (block_table.shape[1] > 1 and block_table.stride(1) != 1), "kv_len, cu_q and table rows must be contiguous")
    _strided(q, "q")
    _strided(k_pages, "k_pages")
    _strided(v_pages, "v_pages")


_HERE = nullcontext()


def _on(index: int):
    """Work on the operands' device, on that device's current stream, whichever device is current."""
    return _HERE if index == torch._C._cuda_getDevice() else torch.cuda.device(index)


def _status(index: int) -> int:
    t = _lib._status.get(index)
    if t is None:
        # made here it would live in the graph's private memory and die with the graph
        _refuse(torch.cuda.is_current_stream_capturing(), "call a paged-cache operator once before capturing it into a graph")
        t = _lib.status_word(torch.device("cuda", index))
    return t.data_ptr()


# ----------------------------------------------------------------------------- where the new tokens stand
def token_coordinates(T: int, kv_len: torch.Tensor, cu_q: Optional[torch.Tensor]):
    """(sequence, position) of every packed row; padding rows have position -1 (reference path)."""
    n = kv_len.numel()
    row = torch.arange(T, device=kv_len.device)
    if cu_q is None:
        return row, (kv_len.long() - 1).clamp(min=-1)
    cu = cu_q.long()
    if n == 0:
        return torch.zeros_like(row), torch.full_like(row, -1)
    seq = (torch.searchsorted(cu, row, right=True) - 1).clamp(0, n - 1)
    new = cu[seq + 1] - cu[seq]
    at = row - cu[seq]
    pos = kv_len.long()[seq] - new + at
    return seq, torch.where((at >= 0) & (at < new) & (pos >= 0), pos, torch.full_like(pos, -1))


# ----------------------------------------------------------------------------- append
def paged_append_ref(q, k, v, k_pages, v_pages, block_table, kv_len, cu_q=None, cs=None):
    from .functional import rope_ref

    T, P = q.shape[0], k_pages.shape[1]
    seq, pos = token_coordinates(T, kv_len, cu_q)
    live = pos >= 0
    seq, pos = seq[live], pos[live]
    _refuse(bool((pos >= block_table.shape[1] * P).any()), "position past the block table")
    page = block_table[seq, pos // P].long()
    _refuse(bool(((page < 0) | (page >= k_pages.shape[0])).any()), "page id outside the pool")
    _refuse(cs is not None and bool((pos >= cs.shape[0]).any()), "position past the rotary table")
    qo, kk = q[live], k[live]
    if cs is not None and pos.numel():
        qo, kk = (rope_ref(t.unsqueeze(0), cs, pos).squeeze(0) for t in (qo, kk))
    k_pages[page, pos % P] = kk
    v_pages[page, pos % P] = v[live]
    out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    out[live] = qo
    return out


def paged_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 block_table: torch.Tensor, kv_len: torch.Tensor, cu_q: Optional[torch.Tensor] = None,
                 cs: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Writes the keys and values of the new tokens to their pages and returns the queries [T, H, D].

    With ``cs`` (rotary table [positions, D / 2, 2], fp32) queries and keys are rotated by their position on the way, as
    ``functional.rope_`` does; k itself is not changed. Two tokens must not share a position of a page."""
    dev, T, H, D, n_pages, P, Hkv, n, cols, row, q_st, kp_st, vp_st = _check_cache(q, k_pages, v_pages, block_table, kv_len, cu_q)
    dt, shape = q.dtype, (T, Hkv, D)
    if not (dev >= 0 and k.shape == shape and v.shape == shape and k.dtype is dt and v.dtype is dt and k.get_device() == dev
            and v.get_device() == dev and _aligned(k) and _aligned(v) and not _tracked(k, v)
            and (cs is None or (cs.dtype is torch.float32 and cs.dim() == 3 and cs.shape[1] == D // 2 and cs.shape[2] == 2
                                and cs.is_contiguous() and cs.get_device() == dev and cs.data_ptr() % 16 == 0))):
        _refuse(k.shape != shape or v.shape != shape, "k and v must be [T, Hkv, D]")
        _refuse(k.dtype != dt or v.dtype != dt or k.device != q.device or v.device != q.device,
                "q, k and v must share dtype and device")
        _refuse(_tracked(k, v), "paged-cache operators have no gradient")
        if cs is not None:
            _refuse(cs.dtype != torch.float32 or cs.dim() != 3 or cs.shape[1:] != (D // 2, 2) or not cs.is_contiguous()
                    or cs.device != q.device, "cs must be a contiguous fp32 [positions, D / 2, 2] table")
        if not q.is_cuda:
            return paged_append_ref(q, k, v, k_pages, v_pages, block_table, kv_len, cu_q, cs)
        _refuse(cs is not None and cs.data_ptr() % 16 != 0, "cs must be 16-byte aligned")
        _strided(k, "k")
        _strided(v, "v")
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if T == 0:
        return out
    args = _lib.PAGED_APPEND_ARGS.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
        block_table.data_ptr(), kv_len.data_ptr(), 0 if cu_q is None else cu_q.data_ptr(),
        0 if cs is None else cs.data_ptr(), _status(dev),
        T, n, H, Hkv, D, P, n_pages, cols, 0 if cs is None else cs.shape[0],
        row, *q_st, *k.stride()[:2], *v.stride()[:2], *kp_st, *vp_st)
    with _on(dev):
        rc = _lib.load().lb_paged_append(args, _lib.stream_ptr())
    _lib.check(rc, "lb_paged_append")
    return out


# ----------------------------------------------------------------------------- attention
def paged_attention_ref(q, k_pages, v_pages, block_table, kv_len, cu_q=None, scale=None, window=0, sinks=0):
    """Masked softmax attention in fp32 (fp64 for fp64 inputs), one sequence at a time."""
    T, H, D = q.shape
    n_pages, P, Hkv, _ = k_pages.shape
    scale = scale if scale is not None else 1.0 / math.sqrt(D)
    ct = torch.float64 if q.dtype == torch.float64 else torch.float32
    seq, pos = token_coordinates(T, kv_len, cu_q)
    out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    for s in range(block_table.shape[0]):
        rows = torch.nonzero((seq == s) & (pos >= 0)).view(-1)
        if rows.numel() == 0:
            continue
        p = pos[rows].view(-1, 1)
        n = int(p.max()) + 1
        _refuse(n > block_table.shape[1] * P, "position past the block table")
        key = torch.arange(n, device=q.device)
        see = key.view(1, -1) <= p
        if window > 0:
            see = see & ((key.view(1, -1) > p - window) | (key.view(1, -1) < sinks))
        used = torch.nonzero(see.any(0)).view(-1)  # what no row sees is not read: it may hold anything
        page = block_table[s, used // P].long()
        _refuse(bool(((page < 0) | (page >= n_pages)).any()), "page id outside the pool")
        kk, vv = (t[page, used % P].to(ct).repeat_interleave(H // Hkv, dim=1) for t in (k_pages, v_pages))
        sc = torch.einsum("thd,shd->hts", q[rows].to(ct), kk) * scale
        sc = sc.masked_fill(~see[:, used], float("-inf"))
        out[rows] = torch.einsum("hts,shd->thd", torch.softmax(sc, dim=-1), vv).to(q.dtype)
    return out


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                    kv_len: torch.Tensor, cu_q: Optional[torch.Tensor] = None, max_q: int = 1,
                    scale: Optional[float] = None, window: int = 0, sinks: int = 0) -> torch.Tensor:
    """Attention of the new tokens over their sequences' cached keys (the new tokens' own included). Returns [T, H, D].

    A token at position p sees the keys j <= p; with ``window`` > 0 of those only j > p - window and the first ``sinks``
    positions. Pages that hold no visible position are not read. ``max_q``: most new tokens of a sequence, used to choose
    the kernel (a wrong value costs speed, not correctness)."""
    dev, T, H, D, n_pages, P, Hkv, n, cols, row, q_st, kp_st, vp_st = _check_cache(q, k_pages, v_pages, block_table, kv_len, cu_q)
    _refuse(window < 0 or sinks < 0, "window and sinks must not be negative")
    window, sinks = window if window < MAX_POSITIONS else 0, min(sinks, MAX_POSITIONS)  # no position is further away
    scale = float(scale) if scale is not None else 1.0 / math.sqrt(D)
    _refuse(not scale >= 0.0, "scale must not be negative")
    if not q.is_cuda:
        return paged_attention_ref(q, k_pages, v_pages, block_table, kv_len, cu_q, scale, window, sinks)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if T == 0:
        return out
    args = _lib.PAGED_ATTN_ARGS.pack(
        q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), out.data_ptr(), block_table.data_ptr(), kv_len.data_ptr(),
        0 if cu_q is None else cu_q.data_ptr(), _status(dev),
        T, n, H, Hkv, D, P, n_pages, cols, window, sinks, min(max_q, MAX_POSITIONS), scale, row, *q_st, *kp_st, *vp_st)
    lib = _lib.load()
    with _on(dev):
        need = lib.lb_paged_attention_workspace(args)
        # a buffer of this call alone, from the allocator of the current stream (or graph)
        ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
        rc = lib.lb_paged_attention(args, None if ws is None else ws.data_ptr(), _lib.stream_ptr())
    _lib.check(rc, "lb_paged_attention")
    return out


# ----------------------------------------------------------------------------- page copies
def copy_pages(pool: torch.Tensor, src: torch.Tensor, dst: torch.Tensor) -> torch.Tensor:
    """``pool[:, dst[i]] = pool[:, src[i]]`` for every i, in place, one launch for all rows of ``pool``
    [rows, n_pages, ...] (the layers of a cache, keys and values). ``src`` / ``dst``: int32 page ids.

    A source may repeat; a destination must not, and must not be a source either: the copies run in no order. Lists in
    host memory are checked for that and uploaded; ids that are on the device already are taken as they are."""
    _refuse(pool.dim() < 2, "pool must be [rows, n_pages, ...]")
    _refuse(src.dim() != 1 or src.shape != dst.shape, "src and dst must be two lists of the same length")
    _refuse(src.dtype != torch.int32 or dst.dtype != torch.int32, "page ids must be int32")
    _refuse(_tracked(pool), "copy_pages has no gradient")
    _refuse(src.device != dst.device, "src and dst must be on one device")
    rows, n_pages = pool.shape[:2]
    n = src.numel()
    if not src.is_cuda:
        s, d = src.tolist(), dst.tolist()
        _refuse(any(not 0 <= i < n_pages for i in s + d), "page id outside the pool")
        _refuse(len(set(d)) != n or bool(set(d) & set(s)), "a destination repeats or is a source as well")
    if n == 0 or pool.numel() == 0:
        return pool
    if not pool.is_cuda:
        _refuse(src.is_cuda, "page ids of a host pool must be in host memory")
        pool[:, dst.long()] = pool[:, src.long()]
        return pool
    es = pool.element_size()
    page_bytes = pool[0, 0].numel() * es
    _refuse(not pool[0, 0].is_contiguous() or page_bytes % 16 or pool.data_ptr() % 16
            or any(k > 1 and (s * es % 16 or s <= 0) for k, s in zip((rows, n_pages), pool.stride()[:2])),
            "a page must be contiguous, a multiple of 16 bytes and 16-byte aligned")
    if not src.is_cuda:
        src, dst = src.to(pool.device), dst.to(pool.device)
    _refuse(src.device != pool.device, "page ids must be on the pool's device or in host memory")
    src, dst = src.contiguous(), dst.contiguous()
    with _on(pool.get_device()):
        rc = _lib.load().lb_copy_pages(pool.data_ptr(), pool.stride(0) * es, pool.stride(1) * es, page_bytes, rows, n_pages,
                                       src.data_ptr(), dst.data_ptr(), n, _status(pool.get_device()), _lib.stream_ptr())
    _lib.check(rc, "lb_copy_pages")
    return pool
