"""Paged-cache and logits operators on the CPU: the reference forms against 64-bit loops, and what is refused."""
import pytest
import torch

from lingua_b200.ops import logits as L
from lingua_b200.ops import paged as P
from paged_oracle import append64, attention64, make_batch, penalize64, rotary


@pytest.mark.parametrize("window,sinks", [(0, 0), (5, 0), (5, 3), (1, 0), (100, 4)])
@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1, 1], [1, 17, 33]), ([3, 0, 7, 1], [3, 9, 20, 0]), ([5], [4])])
def test_attention_reference(q_lens, kv_lens, window, sinks):
    b = make_batch(q_lens, kv_lens, 4, 2, 8, 16, "cpu", dtype=torch.float64, pad_rows=2)
    o = P.paged_attention(b["q"], b["k_pages"], b["v_pages"], b["table"], b["kv_len"], cu_q=b["cu_q"], max_q=max(q_lens),
                          window=window, sinks=sinks)
    ref, _ = attention64(b, window, sinks)
    assert torch.allclose(o, ref, atol=1e-12, rtol=0)


def test_attention_reference_one_token_per_sequence():
    b = make_batch([1, 1, 1], [9, 0, 40], 6, 2, 8, 16, "cpu", dtype=torch.float64)
    o = P.paged_attention(b["q"], b["k_pages"], b["v_pages"], b["table"], b["kv_len"])
    assert torch.allclose(o, attention64(b)[0], atol=1e-12, rtol=0)
    assert (o[1] == 0).all()


@pytest.mark.parametrize("turn", [True, False])
def test_append_reference(turn):
    b = make_batch([3, 0, 20, 1], [3, 9, 40, 0], 4, 2, 8, 16, "cpu", dtype=torch.float32, pad_rows=3)
    cs = rotary(64, 8) if turn else None
    before = b["k_pages"].clone(), b["v_pages"].clone()
    q = P.paged_append(b["q"], b["k"], b["v"], b["k_pages"], b["v_pages"], b["table"], b["kv_len"], cu_q=b["cu_q"], cs=cs)
    out, writes = append64(b, cs)
    assert torch.allclose(q.double(), out, atol=1e-5, rtol=0)
    for (page, row), (k, v) in writes.items():
        assert torch.allclose(b["k_pages"][page, row].double(), k, atol=1e-5, rtol=0)
        assert torch.equal(b["v_pages"][page, row].double(), v)
        before[0][page, row], before[1][page, row] = b["k_pages"][page, row], b["v_pages"][page, row]
    for now, then in zip((b["k_pages"], b["v_pages"]), before):  # nothing else is touched
        assert torch.equal(torch.nan_to_num(now), torch.nan_to_num(then))


def test_copy_pages_reference_and_refusals():
    pool = torch.arange(2 * 6 * 4, dtype=torch.float32).view(2, 6, 4)
    want = pool.clone()
    want[:, [0, 5, 1]] = want[:, [2, 2, 3]]
    ids = lambda *a: torch.tensor(a, dtype=torch.int32)
    assert P.copy_pages(pool, ids(2, 2, 3), ids(0, 5, 1)) is pool and torch.equal(pool, want)
    assert torch.equal(P.copy_pages(pool, ids(), ids()), want)
    for src, dst in (((0,), (6,)), ((-1,), (2,)), ((0, 1), (2, 2)), ((0, 1), (1, 2)), ((3,), (3,))):
        with pytest.raises(ValueError):
            P.copy_pages(pool, ids(*src), ids(*dst))
    for src, dst in ((ids(0).long(), ids(1).long()), (ids(0, 1), ids(2)), (ids(0).view(1, 1), ids(1).view(1, 1))):
        with pytest.raises(ValueError):
            P.copy_pages(pool, src, dst)
    assert torch.equal(pool, want)


def _call(b, **kw):
    a = dict(q=b["q"], k_pages=b["k_pages"], v_pages=b["v_pages"], block_table=b["table"], kv_len=b["kv_len"],
             cu_q=b["cu_q"])
    a.update(kw)
    return P.paged_attention(**a)


def test_attention_refusals():
    b = make_batch([1, 2], [9, 20], 4, 2, 8, 16, "cpu", dtype=torch.float32)
    bad = [dict(q=b["q"][:, :3]), dict(q=b["q"][0]), dict(v_pages=b["v_pages"][:-1]), dict(k_pages=b["k_pages"][..., :4]),
           dict(block_table=b["table"].long()), dict(block_table=b["table"][0]), dict(kv_len=b["kv_len"].long()),
           dict(kv_len=b["kv_len"][:1]), dict(cu_q=b["cu_q"].long()), dict(cu_q=b["cu_q"][:-1]), dict(cu_q=None),
           dict(window=-1), dict(sinks=-1), dict(q=b["q"].double()), dict(q=b["q"].clone().requires_grad_(True)),
           dict(kv_len=torch.tensor([9, 60], dtype=torch.int32)), dict(block_table=b["table"] + 50)]
    for kw in bad:
        with pytest.raises(ValueError):
            _call(b, **kw)
    assert _call(b).shape == b["q"].shape


def test_append_refusals():
    b = make_batch([1, 2], [9, 20], 4, 2, 8, 16, "cpu", dtype=torch.float32)
    base = dict(q=b["q"], k=b["k"], v=b["v"], k_pages=b["k_pages"], v_pages=b["v_pages"], block_table=b["table"],
                kv_len=b["kv_len"], cu_q=b["cu_q"], cs=rotary(64, 8))
    bad = [dict(k=b["k"][:, :1]), dict(v=b["v"][:2]), dict(k=b["k"].double()), dict(cs=rotary(64, 8).double()),
           dict(cs=rotary(64, 16)), dict(cs=rotary(10, 8)), dict(block_table=b["table"][:, :1]),
           dict(block_table=torch.full_like(b["table"], -1))]
    for kw in bad:
        with pytest.raises(ValueError):
            P.paged_append(**{**base, **kw})
    P.paged_append(**base)


def _logits_inputs(N, V, Lh, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(N, V, generator=g) * 3
    hist = torch.randint(0, max(1, V // 3), (N, Lh), generator=g)
    if Lh > 2:
        hist[:, 1] = hist[:, 0]  # the same token twice
        hist[0, 2] = V + 5  # not in the vocabulary
        hist[-1, 0] = -1
    hl = torch.randint(0, Lh + 1, (N,), generator=g).int()
    pl = (hl.float() * torch.rand(N, generator=g)).int()
    return x, hist, hl, pl, g


@pytest.mark.parametrize("N,V,Lh", [(1, 1, 1), (3, 33, 7), (2, 258, 40), (4, 64, 0)])
def test_penalize_reference(N, V, Lh):
    x, hist, hl, pl, g = _logits_inputs(N, V, Lh)
    rep, pres, freq = 1 + torch.rand(N, generator=g), torch.rand(N, generator=g), torch.rand(N, generator=g)
    bias = torch.randn(N, V, generator=g)
    allowed = torch.randint(-2 ** 31, 2 ** 31, (N, (V + 31) // 32), generator=g).int()
    allowed[0] = 0  # nothing is allowed
    x[-1, 0] = float("nan") if N > 1 else 0.0
    if N > 1:
        allowed[-1, 0] &= ~1  # the NaN is masked
    z = L.penalize_logits(x, hist, hl, pl, rep, pres, freq, bias, allowed)
    ref = penalize64(x, hist, hl, pl, rep.tolist(), pres.tolist(), freq.tolist(), bias, allowed)
    assert torch.allclose(z.double(), ref, atol=1e-5, rtol=0)
    assert torch.isinf(z[0]).all()
    # one neutral call changes nothing
    y = torch.randn(N, V)
    assert torch.equal(L.penalize_logits(y, hist, hl, repetition=1.0, presence=0.0), y)


def test_penalize_refusals():
    x, hist, hl, pl, _ = _logits_inputs(2, 40, 6)
    for kw in (dict(logits=x[0]), dict(history=hist.int()), dict(history=hist[:1]), dict(history_len=hl.long()),
               dict(history_len=hl[:1]), dict(prompt_len=pl.long()), dict(repetition=0.0), dict(repetition=-1.0),
               dict(repetition=float("nan")), dict(repetition=torch.ones(3)), dict(presence=torch.ones(2).double()),
               dict(bias=torch.zeros(39)), dict(bias=torch.zeros(40).double()), dict(allowed=torch.zeros(2, 1).int()),
               dict(allowed=torch.zeros(2, 2).long()), dict(out=x.double()), dict(out=x[:1]),
               dict(logits=x.clone().requires_grad_(True))):
        with pytest.raises(ValueError):
            L.penalize_logits(**{**dict(logits=x, history=hist, history_len=hl), **kw})
    out = torch.empty_like(x)
    assert L.penalize_logits(x, hist, hl, out=out) is out


def test_penalize_destinations():
    x, hist, hl, pl, _ = _logits_inputs(3, 40, 6)
    kw = dict(history=hist, history_len=hl, repetition=1.5, presence=0.5)
    want = L.penalize_logits(x, **kw)
    both = torch.zeros(3, 90)
    both[:, :40] = x
    left, right = both[:, :40], both[:, 50:]
    assert torch.equal(L.penalize_logits(left, **kw, out=right), want) and torch.equal(left, x)
    for bad in (both[:, 1:41], both[:, 39:79], both.view(-1)[90:210].view(3, 40), both.view(-1)[20:140].view(3, 40)):
        with pytest.raises(ValueError):
            L.penalize_logits(left, **kw, out=bad)
    assert torch.equal(L.penalize_logits(left, **kw, out=left), want) and torch.equal(left, want)
    one = torch.zeros(1, 50)
    with pytest.raises(ValueError):
        L.penalize_logits(one[:, :40], hist[:1], hl[:1], out=one[:, 8:48])
    flat = torch.zeros(60)
    with pytest.raises(ValueError):
        L.penalize_logits(flat[:40].expand(1, 40), hist[:1], hl[:1], out=flat[8:48].expand(1, 40))
    L.penalize_logits(flat[:20].expand(1, 20), hist[:1], hl[:1], out=flat[20:40].expand(1, 20))
