"""Measured cases of the paged-cache generation operators.

Four operators run in every step of paged generation: ``append`` (rotary embedding of the new tokens' queries and keys, keys
and values written to their pages), ``attend`` (attention of the new tokens over the paged cache, one token or a chunk per
sequence, optionally with a sliding window and visible first tokens), ``pages`` (copies of pages for forks and compaction, all
layers at once) and ``logits`` (penalties, bias and grammar mask before sampling). ``run`` computes them in plain torch
operations, or, with ``own`` true, through ``lingua_b200.ops``.
"""
import math

import torch

own = False

BF16 = torch.bfloat16


# ----------------------------------------------------------------------------- cases
def listed():
    return [
        # one sequence decoding with the 1B model's heads: launch latency is all of it
        dict(name="append_one_token", op="append", heads=16, kv_heads=16, dim=128, page=16, seqs=1, q_max=1, kv_max=700,
             ragged=False),
        # packed prompts of odd lengths entering the cache, grouped heads
        dict(name="append_prompts", op="append", heads=32, kv_heads=8, dim=128, page=64, seqs=24, q_max=700, kv_max=1500,
             ragged=True),
        # 64 samples forked from their prompts: the partly filled last page of each is copied, all layers of the 1B model
        dict(name="pages_fork", op="pages", rows=50, n_pages=400, page=16, kv_heads=16, dim=128, copies=64),
        # compaction after many sequences ended: the pages at the end of the pool move into the holes
        dict(name="pages_compact", op="pages", rows=50, n_pages=160, page=64, kv_heads=16, dim=128, copies=61),
        # the smallest attention call: one sequence, one token, a short cache
        dict(name="attend_one_short", op="attend", heads=16, kv_heads=16, dim=128, page=16, seqs=1, q_max=1, kv_max=511,
             ragged=False, window=0, sinks=0),
        # a decoding batch of very different lengths, grouped heads
        dict(name="attend_batch", op="attend", heads=32, kv_heads=8, dim=128, page=64, seqs=64, q_max=1, kv_max=8192,
             ragged=True, window=0, sinks=0),
        # one sequence with a long context: few rows, a long key axis
        dict(name="attend_one_long", op="attend", heads=32, kv_heads=8, dim=128, page=64, seqs=1, q_max=1, kv_max=131072,
             ragged=False, window=0, sinks=0),
        # streaming generation: a sliding window and four first tokens, one head of keys per query head (7B model's heads)
        dict(name="attend_batch_window", op="attend", heads=32, kv_heads=32, dim=128, page=32, seqs=48, q_max=1, kv_max=20000,
             ragged=True, window=1024, sinks=4),
        # a mixed batch: some sequences bring one token, others the rest of their prompt; odd lengths, pages of 16
        dict(name="attend_mixed", op="attend", heads=32, kv_heads=8, dim=128, page=16, seqs=17, q_max=301, kv_max=2777,
             ragged=True, window=0, sinks=0),
        # a chunk of a long prompt over what earlier chunks left in the cache
        dict(name="attend_chunk_long", op="attend", heads=32, kv_heads=8, dim=128, page=64, seqs=1, q_max=2048, kv_max=32768,
             ragged=False, window=0, sinks=0),
        # one sequence of the byte model: 258 entries, a short history
        dict(name="logits_bytes", op="logits", rows=1, vocab=258, history=200, half=True, bias=False, mask=False),
        # a sampling batch over a large vocabulary with everything switched on
        dict(name="logits_batch", op="logits", rows=64, vocab=128256, history=2000, half=False, bias=True, mask=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "pages", "attend", "attend", "attend", "logits"])
    if op == "logits":
        rows = _log(rng, 1, 64)
        return dict(op=op, rows=rows, vocab=_log(rng, 200, 128256), history=_log(rng, 1, 2000), half=rng.random() < 0.5,
                    bias=rng.random() < 0.5, mask=rng.random() < 0.5)
    page = rng.choice([16, 32, 64, 128, 256])
    dim = rng.choice([64, 128, 128])
    kv_heads = rng.choice([1, 2, 4, 8, 16])
    if op == "pages":
        copies = _log(rng, 1, 64)
        rows = 2 * rng.randint(1, 25)
        # as many copies as stay within the largest listed case
        per = rows * page * kv_heads * dim
        copies = max(1, min(copies, 50 * 64 * 16 * 128 * 61 // per))
        return dict(op=op, rows=rows, n_pages=2 * copies + rng.randint(0, 40), page=page, kv_heads=kv_heads, dim=dim,
                    copies=copies)
    heads = kv_heads * rng.choice([1, 2, 3, 4, 8]) if kv_heads <= 8 else kv_heads * rng.choice([1, 2])
    if op == "append":
        q_max = rng.choice([1, _log(rng, 2, 700)])
        return dict(op=op, heads=heads, kv_heads=kv_heads, dim=dim, page=page, seqs=_log(rng, 1, 24), q_max=q_max,
                    kv_max=q_max + _log(rng, 1, 800), ragged=rng.random() < 0.7)
    window, sinks = (0, 0) if rng.random() < 0.6 else (_log(rng, 16, 4096), rng.choice([0, 1, 4, 37]))
    if rng.random() < 0.5:  # one token a sequence
        seqs = _log(rng, 1, 128)
        q_max, kv_max = 1, _log(rng, 1, min(131072, 64 * 8192 * 8 // (2 * seqs * kv_heads)))
    else:
        seqs = _log(rng, 1, 20)
        q_max = _log(rng, 2, 2048)
        kv_max = q_max + _log(rng, 1, 16384)
        while seqs > 1 and seqs * q_max * kv_max * heads > 2048 * 16384 * 32:
            seqs -= 1
        while q_max > 2 and seqs * q_max * kv_max * heads > 2048 * 16384 * 32:
            q_max //= 2
    return dict(op="attend", heads=heads, kv_heads=kv_heads, dim=dim, page=page, seqs=seqs, q_max=q_max, kv_max=kv_max,
                ragged=rng.random() < 0.7, window=window, sinks=sinks)


def _lengths(case):
    """Host lists (new tokens, keys in the cache after them) of every sequence: part of the case, not of the seed."""
    n, q_max, kv_max = case["seqs"], case["q_max"], case["kv_max"]
    q, kv = [], []
    for i in range(n):
        if not case["ragged"] or i == 0:
            q.append(q_max)
            kv.append(kv_max)
        else:
            f = ((i * 2654435761) % 1009) / 1008.0  # spread over (0, 1], the same for every run of the case
            g = ((i * 40503 + 77) % 997) / 996.0
            qi = 1 if (q_max > 1 and i % 3 == 1) else max(1, int(round(q_max ** g)))
            q.append(qi)
            kv.append(max(qi, int(round(kv_max * (0.05 + 0.95 * f)))))
    return q, kv


# ----------------------------------------------------------------------------- inputs
def _paged(case, gen, fill):
    """A pool of pages in random order and the table that maps every sequence's positions to them."""
    dev = "cuda"
    q_len, kv_len = _lengths(case)
    P = case["page"]
    need = [(n + P - 1) // P for n in kv_len]
    n_pages = sum(need) + 3
    order = torch.randperm(n_pages, generator=gen, device=dev)[: sum(need)].int()
    cols = max(need)
    table = torch.full((len(need), cols), -1, dtype=torch.int32, device=dev)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    shape = (n_pages, P, case["kv_heads"], case["dim"])
    if fill:
        k = torch.randn(shape, generator=gen, device=dev, dtype=torch.float32).to(BF16)
        v = torch.randn(shape, generator=gen, device=dev, dtype=torch.float32).to(BF16)
        # keys of trained models have a few channels that are much larger than the others
        k[..., 5] *= 4
        k[..., case["dim"] // 2 + 1] *= 3
    else:
        k = torch.zeros(shape, device=dev, dtype=BF16)
        v = torch.zeros(shape, device=dev, dtype=BF16)
    cu = [0]
    for n in q_len:
        cu.append(cu[-1] + n)
    return dict(k_pages=k, v_pages=v, table=table, kv_len=torch.tensor(kv_len, dtype=torch.int32, device=dev),
                cu_q=torch.tensor(cu, dtype=torch.int32, device=dev), q_lens=q_len, kv_lens=kv_len)


def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    st = dict(case=dict(case))
    if case["op"] == "pages":
        shape = (case["rows"], case["n_pages"], case["page"], case["kv_heads"], case["dim"])
        pool = torch.empty(shape, dtype=BF16, device=dev)
        for r in range(case["rows"]):
            pool[r] = torch.randn(shape[1:], generator=gen, device=dev)
        ids = torch.randperm(case["n_pages"], generator=gen, device=dev)[: 2 * case["copies"]].int()
        st.update(pool=pool, src=ids[: case["copies"]].clone(), dst=ids[case["copies"]:].clone())
        return st
    if case["op"] == "logits":
        N, V, L = case["rows"], case["vocab"], case["history"]
        x = torch.randn(N, V, generator=gen, device=dev) * 3
        # tokens repeat as words do: a few ids make up most of a history
        u = torch.rand(N, L, generator=gen, device=dev)
        hist = (V ** u).long().clamp(max=V) - 1
        hist_len = torch.randint((L + 1) // 2, L + 1, (N,), generator=gen, device=dev).int()
        prompt = (hist_len.float() * torch.rand(N, generator=gen, device=dev)).int()
        st.update(logits=x.to(BF16) if case["half"] else x, history=hist, history_len=hist_len, prompt_len=prompt,
                  repetition=1.0 + 0.5 * torch.rand(N, generator=gen, device=dev),
                  presence=torch.rand(N, generator=gen, device=dev), frequency=0.3 * torch.rand(N, generator=gen, device=dev),
                  bias=torch.randn(V, generator=gen, device=dev) if case["bias"] else None,
                  allowed=torch.randint(-2 ** 31, 2 ** 31, (N, (V + 31) // 32), generator=gen, device=dev).int()
                  if case["mask"] else None)
        return st
    st.update(_paged(case, gen, case["op"] == "attend"))
    T = sum(st["q_lens"])
    H, Hkv, D = case["heads"], case["kv_heads"], case["dim"]
    # the layout of the fused projection: queries, keys and values of a token side by side
    qkv = torch.randn(T, H + 2 * Hkv, D, generator=gen, device=dev).to(BF16)
    st.update(q=qkv[:, :H], k=qkv[:, H:H + Hkv], v=qkv[:, H + Hkv:], max_q=case["q_max"])
    if case["op"] == "append":
        inv = 10000.0 ** (-torch.arange(0, D, 2, device=dev, dtype=torch.float64) / D)
        ang = torch.arange(case["kv_max"], device=dev, dtype=torch.float64).view(-1, 1) * inv
        st["cs"] = torch.stack((ang.cos(), ang.sin()), dim=-1).float()
    return st


# ----------------------------------------------------------------------------- plain forms
def _rotate(x, cs):
    a, b = x.float()[..., 0::2], x.float()[..., 1::2]
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    return torch.stack((a * c - b * s, a * s + b * c), dim=-1).flatten(-2).to(x.dtype)


def _plain_append(st):
    P = st["k_pages"].shape[1]
    cu = st["cu_q"].long()
    n = cu[1:] - cu[:-1]
    T = st["q"].shape[0]
    seq = torch.repeat_interleave(torch.arange(n.numel(), device=cu.device), n, output_size=T)
    pos = st["kv_len"].long()[seq] - n[seq] + torch.arange(T, device=cu.device) - cu[seq]
    page = st["table"][seq, pos // P].long()
    cs = st["cs"][pos]
    st["k_pages"][page, pos % P] = _rotate(st["k"], cs)
    st["v_pages"][page, pos % P] = st["v"]
    return [_rotate(st["q"], cs), st["k_pages"], st["v_pages"]]


def _plain_attend(st):
    case = st["case"]
    P, H, Hkv, D = case["page"], case["heads"], case["kv_heads"], case["dim"]
    G, W, sinks = H // Hkv, case["window"], case["sinks"]
    q = st["q"]
    out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    at = 0
    for i, (nq, nk) in enumerate(zip(st["q_lens"], st["kv_lens"])):
        pages = st["table"][i, : (nk + P - 1) // P].long()
        k = st["k_pages"][pages].reshape(-1, Hkv, D)[:nk]
        v = st["v_pages"][pages].reshape(-1, Hkv, D)[:nk]
        pos = torch.arange(nk - nq, nk, device=q.device).view(nq, 1)
        key = torch.arange(nk, device=q.device).view(1, nk)
        hide = key > pos
        if W:
            hide = hide | ((key <= pos - W) & (key >= sinks))
        if nk == 0:
            continue
        qi = q[at:at + nq].float().reshape(nq, Hkv, G, D)
        step = Hkv if nq * nk * H <= 1 << 24 else 1  # heads at once: the scores of a long chunk do not fit together
        for h in range(0, Hkv, step):
            hs = slice(h, h + step)
            kt = k[:, hs].float().permute(1, 2, 0)
            vt = v[:, hs].float().permute(1, 0, 2)
            s = torch.matmul(qi[:, hs].permute(1, 2, 0, 3).reshape(-1, G * nq, D), kt).reshape(-1, G, nq, nk) / math.sqrt(D)
            s.masked_fill_(hide, float("-inf"))
            s = torch.exp(s - s.amax(dim=-1, keepdim=True))
            den = s.sum(dim=-1, keepdim=True)
            o = torch.matmul(s.reshape(-1, G * nq, nk), vt).reshape(-1, G, nq, D) / den
            out[at:at + nq].view(nq, Hkv, G, D)[:, hs] = o.permute(2, 0, 1, 3).to(q.dtype)
        at += nq
    return out


def _plain_logits(st):
    x = st["logits"].float()
    N, V = x.shape
    L = st["history"].shape[1]
    at = torch.arange(L, device=x.device).view(1, L)
    live = at < st["history_len"].view(N, 1)
    new = live & (at >= st["prompt_len"].view(N, 1))
    seen = torch.zeros(N, V, device=x.device).scatter_add_(1, st["history"], live.float())
    made = torch.zeros(N, V, device=x.device).scatter_add_(1, st["history"], new.float())
    r = st["repetition"].view(N, 1)
    z = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x)
    z = z - st["frequency"].view(N, 1) * made - st["presence"].view(N, 1) * (made > 0)
    if st["bias"] is not None:
        z = z + st["bias"]
    if st["allowed"] is not None:
        tok = torch.arange(V, device=x.device)
        ok = (st["allowed"][:, tok // 32] >> (tok % 32)) & 1
        z = z.masked_fill(ok == 0, float("-inf"))
    return z.to(st["logits"].dtype)


def run(state):
    st = state
    op = st["case"]["op"]
    if not own:
        if op == "append":
            return _plain_append(st)
        if op == "attend":
            return _plain_attend(st)
        if op == "pages":
            st["pool"][:, st["dst"].long()] = st["pool"][:, st["src"].long()]
            return st["pool"]
        return _plain_logits(st)
    from lingua_b200.ops.logits import penalize_logits
    from lingua_b200.ops.paged import copy_pages, paged_append, paged_attention

    one = st["case"].get("q_max") == 1  # one token a sequence: token i belongs to sequence i
    if op == "append":
        q = paged_append(st["q"], st["k"], st["v"], st["k_pages"], st["v_pages"], st["table"], st["kv_len"],
                         cu_q=None if one else st["cu_q"], cs=st["cs"])
        return [q, st["k_pages"], st["v_pages"]]
    if op == "attend":
        return paged_attention(st["q"], st["k_pages"], st["v_pages"], st["table"], st["kv_len"],
                               cu_q=None if one else st["cu_q"], max_q=st["max_q"], window=st["case"]["window"],
                               sinks=st["case"]["sinks"])
    if op == "pages":
        return copy_pages(st["pool"], st["src"], st["dst"])
    return penalize_logits(st["logits"], st["history"], st["history_len"], prompt_len=st["prompt_len"],
                           repetition=st["repetition"], presence=st["presence"], frequency=st["frequency"],
                           bias=st["bias"], allowed=st["allowed"])


# ----------------------------------------------------------------------------- definitions in 64 bits
def exact(case, seed):
    if case["op"] == "pages":
        return None  # copies, nothing is computed
    st = prepare(case, seed)
    dev = st["logits"].device if case["op"] == "logits" else st["q"].device
    if case["op"] == "logits":
        z = st["logits"].double()
        N, V = z.shape
        hist, total, prompt = st["history"].cpu(), st["history_len"].tolist(), st["prompt_len"].tolist()
        for n in range(N):
            row = hist[n, : total[n]]
            seen = torch.unique(row).to(dev)
            ids, times = (t.to(dev) for t in torch.unique(row[prompt[n]:], return_counts=True))
            r = st["repetition"][n].double()
            old = z[n, seen]
            z[n, seen] = torch.where(old > 0, old / r, old * r)
            z[n, ids] -= st["frequency"][n].double() * times.double() + st["presence"][n].double()
        if st["bias"] is not None:
            z += st["bias"].double()
        if st["allowed"] is not None:
            bits = (st["allowed"].unsqueeze(-1) >> torch.arange(32, device=dev)) & 1
            z[bits.reshape(N, -1)[:, :V] == 0] = -math.inf
        return z
    P, D = case["page"], case["dim"]
    H, Hkv = case["heads"], case["kv_heads"]
    if case["op"] == "append":
        q = st["q"].double()
        kp, vp = st["k_pages"].double(), st["v_pages"].double()
        out = torch.empty_like(q)
        t = 0
        for i, (nq, nk) in enumerate(zip(st["q_lens"], st["kv_lens"])):
            pos = torch.arange(nk - nq, nk, device=dev)
            z = torch.view_as_complex(st["cs"].double()[pos].contiguous()).unsqueeze(1)
            turn = [torch.view_as_real(torch.view_as_complex(x.reshape(nq, -1, D // 2, 2).contiguous()) * z).reshape(nq, -1, D)
                    for x in (q[t:t + nq], st["k"][t:t + nq].double())]
            slot = st["table"][i].long()[torch.div(pos, P, rounding_mode="floor")] * P + pos % P
            out[t:t + nq] = turn[0]
            kp.view(-1, Hkv, D)[slot] = turn[1]
            vp.view(-1, Hkv, D)[slot] = st["v"][t:t + nq].double()
            t += nq
        return [out, kp, vp]
    # attention: one query head at a time over the rows its sequence's table names
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=dev)
    kf, vf = st["k_pages"].view(-1, Hkv, D), st["v_pages"].view(-1, Hkv, D)
    t = 0
    for i, (nq, nk) in enumerate(zip(st["q_lens"], st["kv_lens"])):
        j = torch.arange(nk, device=dev)
        slot = st["table"][i].long()[j // P] * P + j % P
        p = (nk - nq + torch.arange(nq, device=dev)).unsqueeze(1)
        see = (j <= p) if not case["window"] else (j <= p) & ((j + case["window"] > p) | (j < case["sinks"]))
        for h in range(H):
            hk = h // (H // Hkv)
            s = (st["q"][t:t + nq, h].double() @ kf[slot, hk].double().t()) * D ** -0.5
            w = torch.softmax(torch.where(see, s, torch.full((), -math.inf, dtype=torch.float64, device=dev)), dim=-1)
            out[t:t + nq, h] = w @ vf[slot, hk].double()
        t += nq
    return out


# ----------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["op"] == "pages":
        return {"bytes": 2 * 2 * case["rows"] * case["copies"] * case["page"] * case["kv_heads"] * case["dim"], "flops": 0}
    if case["op"] == "logits":
        n = case["rows"] * case["vocab"]
        b = n * (4 if case["half"] else 8) + (n // 8 if case["mask"] else 0) + (4 * case["vocab"] if case["bias"] else 0)
        return {"bytes": b + 8 * case["rows"] * case["history"], "flops": 6 * n}
    q_len, kv_len = _lengths(case)
    H, Hkv, D = case["heads"], case["kv_heads"], case["dim"]
    T = sum(q_len)
    if case["op"] == "append":
        return {"bytes": 2 * 2 * T * (H + 2 * Hkv) * D + 4 * T * D, "flops": 3 * T * (H + Hkv) * D}
    W, sinks = case["window"], case["sinks"]
    rows = pairs = 0
    for nq, nk in zip(q_len, kv_len):
        first = max(0, nk - nq - W + 1) if W else 0  # first key inside the window of the first new token
        rows += nk - max(0, first - min(sinks, first))
        for p in range(nk - nq, nk):
            lo = max(0, p - W + 1) if W else 0
            pairs += p + 1 - lo + min(sinks, lo)
    return {"bytes": 2 * 2 * T * H * D + 2 * 2 * rows * Hkv * D, "flops": 4 * D * H * pairs}
