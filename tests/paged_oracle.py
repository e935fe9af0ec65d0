"""Plain 64-bit forms of the paged-cache and logits operators and the inputs their tests share."""
import math

import torch


def make_batch(q_lens, kv_lens, H, Hkv, D, page, device, seed=0, order="pool", extra_cols=1, poison=True, pad_rows=0,
               dtype=torch.bfloat16, release=None):
    """Packed new tokens, pools with their pages in random order, table, lengths. ``order``: memory order of the pools
    ("pool" [n, page, Hkv, D] contiguous, "heads" [n, Hkv, page, D], "wide" rows with gaps). ``poison``: whatever no position
    of a sequence owns holds NaN and infinities, unused table entries are out of range. ``release`` (window, sinks): pages
    that no query sees any more have been given back."""
    g = torch.Generator().manual_seed(seed)
    need = [(n + page - 1) // page for n in kv_lens]
    n_pages = sum(need) + 2
    ids = torch.randperm(n_pages, generator=g)
    cols = max(need + [1]) + extra_cols
    table = torch.full((len(need), cols), -7 if poison else 0, dtype=torch.int32)
    kv = torch.randn(2, n_pages, page, Hkv, D, generator=g)
    kv[0, ..., 3] *= 4
    kv = kv.to(dtype)
    at = 0
    used = torch.zeros(n_pages, page, dtype=torch.bool)
    for i, n in enumerate(need):
        table[i, :n] = ids[at:at + n].int()
        for c in range(n):
            if release and page * (c + 1) <= kv_lens[i] - q_lens[i] + 1 - release[0] and page * c >= release[1]:
                table[i, c] = -7
            else:
                used[ids[at + c], : min(page, kv_lens[i] - c * page)] = True
        at += n
    if poison:
        kv[:, ~used] = float("nan")
        kv[0].view(n_pages, page, -1)[~used.view(n_pages, page), ::3] = float("inf")
    pools = []
    for t in kv:
        if order == "heads":
            t = t.permute(0, 2, 1, 3).contiguous().to(device).permute(0, 2, 1, 3)
        elif order == "wide":
            w = torch.zeros(n_pages, page, Hkv, D + 8, dtype=dtype)
            w[..., :D] = t
            t = w.to(device)[..., :D]
        else:
            t = t.contiguous().to(device)
        pools.append(t)
    T = sum(q_lens) + pad_rows
    qkv = torch.randn(T, H + 2 * Hkv, D, generator=g).to(dtype).to(device)
    cu = [0]
    for n in q_lens:
        cu.append(cu[-1] + n)
    return dict(q=qkv[:, :H], k=qkv[:, H:H + Hkv], v=qkv[:, H + Hkv:], k_pages=pools[0], v_pages=pools[1],
                table=table.to(device), kv_len=torch.tensor(kv_lens, dtype=torch.int32, device=device),
                cu_q=torch.tensor(cu, dtype=torch.int32, device=device), q_lens=list(q_lens), kv_lens=list(kv_lens))


def attention64(b, window=0, sinks=0, scale=None):
    """(o, sum_j p_j |v_j|) in float64: the second says how far roundings of p can move o."""
    q, kp, vp, table = (b[n] for n in ("q", "k_pages", "v_pages", "table"))
    dev = q.device
    H, D = q.shape[1:]
    page, Hkv = kp.shape[1:3]
    G = H // Hkv
    scale = scale if scale is not None else 1.0 / math.sqrt(D)
    o = torch.zeros(q.shape, dtype=torch.float64, device=dev)
    mag = torch.zeros_like(o)
    row = 0
    for s, (nq, nk) in enumerate(zip(b["q_lens"], b["kv_lens"])):
        if nk > 0:
            pos = torch.arange(nk, device=dev)
            slot = table[s].long()[pos // page].clamp(min=0) * page + pos % page
            k = kp.reshape(-1, Hkv, D)[slot].double()
            v = vp.reshape(-1, Hkv, D)[slot].double()
            k, v = torch.nan_to_num(k, 0.0, 0.0, 0.0), torch.nan_to_num(v, 0.0, 0.0, 0.0)  # only hidden places hold any
        p = torch.arange(nk - nq, nk, device=dev).view(-1, 1)
        j = torch.arange(nk, device=dev).view(1, -1)
        see = (j <= p) & ((j > p - window) | (j < sinks)) if window else j <= p
        for h in range(H if nk > 0 else 0):
            w = (q[row:row + nq, h].double() @ k[:, h // G].t() * scale).masked_fill(~see, -math.inf)
            w = torch.exp(w - w.amax(dim=1, keepdim=True).clamp(min=-1e300))
            w = w / w.sum(dim=1, keepdim=True).clamp(min=1e-300)
            o[row:row + nq, h] = w @ v[:, h // G]
            mag[row:row + nq, h] = w @ v[:, h // G].abs()
        row += nq
    return o, mag


def attention_tolerance(o, mag):
    """bf16 result: half a step of the value itself (2^-8), half a step of every probability that the tensor cores take
    in bf16 (2^-8 of sum p |v|), and 2e-4 of that sum for fp32 scores and the exponential's 1e-4."""
    return o.abs() * 2 ** -8 + mag * (2 ** -8 + 2e-4) + 1e-6


def append64(b, cs):
    """(rotated q, {(page, row): (rotated k, v)}) in float64."""
    q, k, v, table = (b[n].cpu() for n in ("q", "k", "v", "table"))
    page = b["k_pages"].shape[1]
    cs = None if cs is None else cs.cpu().double()

    def turn(x, p):
        if cs is None:
            return x.double()
        z = torch.view_as_complex(x.double().reshape(x.shape[0], -1, 2).contiguous())
        return torch.view_as_real(z * torch.view_as_complex(cs[p].contiguous())).reshape(x.shape)

    out = torch.zeros(q.shape, dtype=torch.float64)
    writes = {}
    row = 0
    for s, (nq, nk) in enumerate(zip(b["q_lens"], b["kv_lens"])):
        for i in range(nq):
            p = nk - nq + i
            if p >= 0:
                out[row] = turn(q[row], p)
                writes[int(table[s, p // page]), p % page] = (turn(k[row], p), v[row].double())
            row += 1
    return out, writes


def rotary(n, D, device="cpu"):
    ang = torch.arange(n, dtype=torch.float64).view(-1, 1) * 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    return torch.stack((ang.cos(), ang.sin()), dim=-1).float().to(device)


def penalize64(x, history, history_len, prompt_len, rep, pres, freq, bias, allowed):
    """Row by row, token by token; rep / pres / freq are lists of floats."""
    z = x.double().cpu().clone()
    V = z.shape[1]
    for n in range(z.shape[0]):
        ids = [int(t) for t in history[n].tolist()[: max(0, int(history_len[n]))]]
        made = ids[max(0, int(prompt_len[n])):] if prompt_len is not None else ids
        for t in set(ids):
            if 0 <= t < V:
                z[n, t] = z[n, t] / rep[n] if z[n, t] > 0 else z[n, t] * rep[n]
        for t in set(made):
            if 0 <= t < V:
                z[n, t] -= pres[n] + freq[n] * made.count(t)
        if bias is not None:
            z[n] += (bias if bias.dim() == 1 else bias[n]).double().cpu()
        if allowed is not None:
            words = allowed[n].tolist()
            for t in range(V):
                if not (words[t // 32] >> (t % 32)) & 1:
                    z[n, t] = -math.inf
    return z
