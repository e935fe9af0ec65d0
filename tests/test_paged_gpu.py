"""Paged-cache kernels against 64-bit forms (tests/paged_oracle.py says where the tolerances come from)."""
import pytest
import torch

from lingua_b200.ops import _lib
from lingua_b200.ops import paged as P
from paged_oracle import append64, attention64, attention_tolerance, make_batch, rotary

pytestmark = pytest.mark.gpu
DEV = "cuda"


def attend(b, one=False, **kw):
    return P.paged_attention(b["q"], b["k_pages"], b["v_pages"], b["table"], b["kv_len"],
                             cu_q=None if one else b["cu_q"], max_q=max(b["q_lens"] + [1]), **kw)


def check(o, b, window=0, sinks=0, scale=None):
    ref, mag = attention64(b, window, sinks, scale)
    err = (o.double() - ref).abs()
    assert torch.isfinite(o.float()).all()
    bad = err > attention_tolerance(ref, mag)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, largest {err[bad].max():.3g} at {bad.nonzero()[0].tolist()}"


MASKS = [(0, 0), (1, 0), (40, 0), (40, 5), (200, 33), (1000, 2)]


@pytest.mark.parametrize("window,sinks", MASKS)
@pytest.mark.parametrize("H,Hkv,D,page", [(1, 1, 128, 16), (8, 2, 128, 32), (6, 2, 64, 16), (16, 1, 128, 64), (4, 4, 64, 256),
                                          (14, 2, 128, 128), (40, 2, 128, 16)])
def test_one_token_per_sequence(H, Hkv, D, page, window, sinks):
    kv = [1, 2, 0, 15, 16, 17, 63, 64, 65, 129, 300, 777]
    b = make_batch([1] * len(kv), kv, H, Hkv, D, page, DEV, seed=H + page, release=(window, sinks) if window else None)
    check(attend(b, one=True, window=window, sinks=sinks), b, window, sinks)
    check(attend(b, window=window, sinks=sinks), b, window, sinks)  # the same through cu_q


@pytest.mark.parametrize("window,sinks", MASKS)
@pytest.mark.parametrize("H,Hkv,D,page", [(2, 2, 128, 16), (8, 2, 128, 64), (6, 2, 64, 32), (16, 1, 128, 128), (3, 1, 128, 256),
                                          (7, 7, 64, 16), (48, 2, 128, 16)])
def test_chunks(H, Hkv, D, page, window, sinks):
    q = [1, 5, 0, 33, 130, 257, 1, 7]
    kv = [1, 5, 40, 200, 130, 700, 321, 3]  # the last has more new tokens than keys: rows that see nothing
    b = make_batch(q, kv, H, Hkv, D, page, DEV, seed=H + page, pad_rows=3, release=(window, sinks) if window else None)
    o = attend(b, window=window, sinks=sinks)
    check(o, b, window, sinks)
    assert (o[-3:] == 0).all() and (o[sum(q) - 7:sum(q) - 4] == 0).all()


@pytest.mark.parametrize("order", ["heads", "wide"])
@pytest.mark.parametrize("q,kv", [([1, 1, 1], [40, 333, 65]), ([20, 150, 1], [40, 333, 65])])
def test_memory_orders(order, q, kv):
    b = make_batch(q, kv, 8, 2, 128, 32, DEV, order=order)
    check(attend(b), b)


@pytest.mark.parametrize("q,kv", [([1], [20001]), ([1, 1], [33000, 5]), ([300], [9000]), ([17, 1], [5000, 30])])
def test_long_keys(q, kv):
    b = make_batch(q, kv, 4, 1, 128, 64, DEV)
    check(attend(b), b)


def test_many_sequences():
    kv = [(i * 37) % 150 for i in range(700)]
    b = make_batch([1] * 700, kv, 2, 1, 128, 16, DEV)
    check(attend(b, one=True), b)


@pytest.mark.parametrize("scale", [0.0, 0.02, 1.0])
def test_scale(scale):
    for q, kv in (([1, 1], [100, 37]), ([140, 3], [300, 50])):
        b = make_batch(q, kv, 8, 2, 128, 16, DEV, seed=3)
        check(attend(b, scale=scale), b, scale=scale)


def test_values_far_apart():
    """A running maximum that grows late, and scores whose exponentials underflow."""
    for q, kv in (([1], [700]), ([200], [700])):
        b = make_batch(q, kv, 4, 4, 128, 16, DEV, seed=4)
        k = b["k_pages"]
        page = b["table"][0, 30].long()
        k[page] = k[page] * 30
        check(attend(b, scale=0.5), b, scale=0.5)


def test_repeats_bit_for_bit_and_on_other_streams():
    b = make_batch([1] * 5 + [300], [4000, 17, 900, 64, 2500, 2000], 8, 2, 128, 16, DEV)
    first = attend(b)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = []
    for s in (s1, s2) * 4:  # calls that overlap
        with torch.cuda.stream(s):
            outs.append(attend(b))
    torch.cuda.synchronize()
    assert all(torch.equal(first, o) for o in outs)


@pytest.mark.parametrize("one", [True, False])
def test_graph_replay_with_new_lengths(one):
    q, kv = ([1, 1, 1], [500, 1, 900]) if one else ([30, 1, 200], [500, 1, 900])
    b = make_batch(q, kv, 8, 2, 128, 16, DEV, poison=False)
    cs = rotary(1000, 128, DEV)
    attend(b, one)  # status word and kernels are loaded before the capture
    P.paged_append(b["q"], b["k"], b["v"], b["k_pages"], b["v_pages"], b["table"], b["kv_len"], b["cu_q"], cs)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            qr = P.paged_append(b["q"], b["k"], b["v"], b["k_pages"], b["v_pages"], b["table"], b["kv_len"],
                                None if one else b["cu_q"], cs)
            o = attend({**b, "q": qr}, one)
        graphs.append((g, qr, o))
    for kv_new in ([300, 1, 640], [499, 0, 256]):
        b["kv_len"].copy_(torch.tensor(kv_new, dtype=torch.int32))
        streams = [torch.cuda.Stream() for _ in graphs]
        torch.cuda.synchronize()
        for (g, _, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        now = {**b, "kv_lens": kv_new}
        for _, qr, o in graphs:
            check(o, {**now, "q": qr})


@pytest.mark.parametrize("turn", [True, False])
@pytest.mark.parametrize("H,Hkv,D,page", [(1, 1, 128, 16), (8, 2, 64, 32), (32, 8, 128, 64), (5, 5, 128, 256)])
@pytest.mark.parametrize("order", ["pool", "heads", "wide"])
def test_append(H, Hkv, D, page, order, turn):
    q, kv = [3, 0, 20, 1, 1, 300, 4], [3, 9, 40, 0, 77, 301, 2]
    b = make_batch(q, kv, H, Hkv, D, page, DEV, order=order, pad_rows=2, poison=order == "pool")
    cs = rotary(400, D, DEV) if turn else None
    kb, vb = b["k_pages"].clone(), b["v_pages"].clone()
    raw = b["k"].clone()
    out = P.paged_append(b["q"], b["k"], b["v"], b["k_pages"], b["v_pages"], b["table"], b["kv_len"], b["cu_q"], cs)
    ref, writes = append64(b, cs)
    kw = kb.double()
    for (pg, row), (k, v) in writes.items():
        kw[pg, row], vb[pg, row] = k.to(DEV), v.to(DEV).bfloat16()
    # a rotated value is one rounding to bf16 of two fp32 products: half a step, plus 2^-22 of the pair's size
    pair = 8.0 * 2 ** -22 * 8
    assert ((out.double().cpu() - ref).abs() <= ref.abs() * 2 ** -8 + pair).all()
    same = torch.isnan(kw) | torch.isinf(kw) | ((b["k_pages"].double() - kw).abs() <= kw.abs() * 2 ** -8 + pair)
    assert same.all()
    assert torch.equal(torch.isnan(b["k_pages"]), torch.isnan(kw)) and torch.equal(torch.isinf(b["k_pages"]), torch.isinf(kw))
    assert torch.equal(torch.nan_to_num(b["v_pages"].float()), torch.nan_to_num(vb.float()))
    assert torch.equal(raw, b["k"])
    if not turn:
        assert torch.equal(out[:3], b["q"][:3])


def test_append_one_token_and_same_bits_as_the_unpaged_rotation():
    from lingua_b200.ops import functional as F

    b = make_batch([1] * 4, [5, 90, 0, 33], 8, 2, 128, 16, DEV, poison=False)
    cs = F.rope_table(128, 100, 10000.0, DEV)
    q1 = P.paged_append(b["q"], b["k"], b["v"], b["k_pages"], b["v_pages"], b["table"], b["kv_len"], cs=cs)
    qkv = torch.cat((b["q"], b["k"]), dim=1).reshape(4, -1).contiguous()
    F.rope_(qkv, cs, 10, 128, 4, torch.tensor([4, 89, 0, 32], dtype=torch.int32, device=DEV))
    qkv = qkv.view(4, 10, 128)
    live = [0, 1, 3]
    assert torch.equal(q1[live], qkv[live, :8]) and (q1[2] == 0).all()
    for s, p in ((0, 4), (1, 89), (3, 32)):
        assert torch.equal(b["k_pages"][b["table"][s, p // 16].long(), p % 16], qkv[s, 8:])


@pytest.mark.parametrize("dtype,page_shape", [(torch.bfloat16, (16, 2, 64)), (torch.float32, (4,)), (torch.uint8, (48,)),
                                              (torch.bfloat16, (64, 16, 128)), (torch.bfloat16, (5, 3, 8))])
@pytest.mark.parametrize("n", [1, 7, 40])
def test_copy_pages(dtype, page_shape, n):
    g = torch.Generator().manual_seed(n)
    pool = torch.randint(0, 200, (3, 100, *page_shape), generator=g).to(dtype).to(DEV)
    ids = torch.randperm(100, generator=g).int()
    src, dst = ids[:n].clone(), ids[n:2 * n].clone()
    src[-1] = src[0]  # a source may repeat
    want = pool.clone()
    want[:, dst.long().to(DEV)] = want[:, src.long().to(DEV)]
    a = pool.clone()
    assert P.copy_pages(a, src, dst) is a and torch.equal(a, want)
    a = pool.clone()
    assert torch.equal(P.copy_pages(a, src.to(DEV), dst.to(DEV)), want)
    part = pool[1:, 0:100]  # rows of a larger pool
    P.copy_pages(part, src, dst)
    assert torch.equal(pool[1:], want[1:]) and not torch.equal(pool[0], want[0])


def test_bad_pages_are_reported_not_followed():
    """Ids outside the pool, positions past the table: skipped, recorded, everybody else served."""
    b = make_batch([1, 1, 1], [40, 40, 40], 4, 2, 128, 16, DEV, poison=False)
    b["table"][1, 1] = 10 ** 6
    with pytest.raises(RuntimeError, match="status"):
        o = attend(b, one=True)
        _lib.check_status()
    good = [0, 2]
    ref, mag = attention64({**b, "table": b["table"].where(b["table"] < b["k_pages"].shape[0], 0)})
    assert ((o.double() - ref).abs() <= attention_tolerance(ref, mag))[good].all() and torch.isfinite(o.float()).all()
    b["q_lens"], many = [40, 40, 40], torch.randn(120, 4, 128, device=DEV).bfloat16()
    b["cu_q"] = torch.tensor([0, 40, 80, 120], dtype=torch.int32, device=DEV)
    b["q"] = many
    with pytest.raises(RuntimeError, match="status"):
        o = attend(b)
        _lib.check_status()
    assert torch.isfinite(o.float()).all()
    with pytest.raises(RuntimeError, match="status"):
        P.paged_append(many, many[:, :2], many[:, 2:], b["k_pages"], b["v_pages"], b["table"], b["kv_len"], b["cu_q"])
        _lib.check_status()
    with pytest.raises(RuntimeError, match="status"):
        attend({**b, "kv_len": torch.full_like(b["kv_len"], 10 ** 9)})
        _lib.check_status()
    with pytest.raises(RuntimeError, match="status"):
        P.copy_pages(b["k_pages"].unsqueeze(0), torch.tensor([0, 1], dtype=torch.int32, device=DEV),
                     torch.tensor([10 ** 6, -1], dtype=torch.int32, device=DEV))
        _lib.check_status()


def test_refusals_on_the_gpu():
    b = make_batch([1, 1], [20, 30], 4, 2, 128, 16, DEV, poison=False)
    for kw in (dict(q=b["q"].half()), dict(k_pages=b["k_pages"].float(), v_pages=b["v_pages"].float(), q=b["q"].float()),
               dict(table=b["table"].cpu()), dict(q=b["q"][..., ::2], k_pages=b["k_pages"][..., ::2], v_pages=b["v_pages"][..., ::2]),
               dict(k_pages=b["k_pages"][:, :8], v_pages=b["v_pages"][:, :8]),
               dict(q=b["q"][..., :32], k_pages=b["k_pages"][..., :32], v_pages=b["v_pages"][..., :32]),
               dict(q=torch.zeros(2 * 4 * 128 + 1, device=DEV).bfloat16()[1:].view(2, 4, 128)),
               dict(q=b["q"][:1].expand(2, 4, 128)),
               dict(kv_len=torch.stack((b["kv_len"], b["kv_len"]), 1)[:, 0])):
        with pytest.raises(ValueError):
            attend({**b, **kw}, one=True)
    for pool in (torch.zeros(1, 4, 3, device=DEV), torch.zeros(1, 4, 8, 8, device=DEV)[..., ::2],
                 torch.zeros(1, 1, 8, device=DEV).expand(1, 4, 8)):
        with pytest.raises(ValueError):
            P.copy_pages(pool, torch.tensor([0], dtype=torch.int32), torch.tensor([1], dtype=torch.int32))
    empty = make_batch([], [], 4, 2, 128, 16, DEV, poison=False)
    assert attend(empty, one=True).shape == (0, 4, 128)


def test_further_refusals_on_the_gpu():
    b = make_batch([1, 1], [20, 30], 4, 2, 128, 16, DEV, poison=False)
    app = lambda **kw: P.paged_append(**{**dict(q=b["q"], k=b["k"], v=b["v"], k_pages=b["k_pages"], v_pages=b["v_pages"],
                                                block_table=b["table"], kv_len=b["kv_len"], cs=rotary(64, 128, DEV)), **kw})
    odd = torch.zeros(64 * 128 + 1, device=DEV)[1:].view(64, 64, 2)  # a rotary table that 16-byte loads cannot read
    for kw in (dict(cs=odd), dict(k=b["k"].clone().requires_grad_(True)), dict(cs=rotary(64, 128)),
               dict(k=torch.zeros(2 * 2 * 128 + 1, device=DEV).bfloat16()[1:].view(2, 2, 128)), dict(v=b["v"].float())):
        with pytest.raises(ValueError):
            app(**kw)
    for kw in (dict(k_pages=b["k_pages"].clone().requires_grad_(True)),
               dict(table=torch.zeros(1, 1, dtype=torch.int32, device=DEV).expand(2, 2 ** 27))):
        with pytest.raises(ValueError):
            attend({**b, **kw}, one=True)
    for scale in (-0.1, float("nan")):
        with pytest.raises(ValueError):
            attend(b, one=True, scale=scale)
    assert app().shape == (2, 4, 128)


@pytest.mark.parametrize("q,kv", [([1, 1, 1], [300, 40, 7]), ([40, 1, 200], [300, 40, 200])])
def test_no_sequences_rows_before_the_first_and_wide_limits(q, kv):
    b = make_batch(q, kv, 8, 2, 128, 16, DEV, pad_rows=2, seed=5)
    ref, mag = attention64(b)
    # the largest window and as many first tokens as there can be change nothing
    for kw in (dict(window=2 ** 31 - 1), dict(window=2 ** 40, sinks=2 ** 40), dict(window=5, sinks=2 ** 31 - 1)):
        o = attend(b, **kw)
        assert ((o.double() - ref).abs() <= attention_tolerance(ref, mag)).all()
    # three rows in front that belong to nobody
    front = {**b, "q": torch.cat((b["q"][:3], b["q"])), "cu_q": b["cu_q"] + 3}
    o = attend(front)
    assert (o[:3] == 0).all() and ((o[3:].double() - ref).abs() <= attention_tolerance(ref, mag)).all()
    none = {**b, "table": b["table"][:0], "kv_len": b["kv_len"][:0], "cu_q": torch.zeros(1, dtype=torch.int32, device=DEV)}
    assert (attend(none) == 0).all()
    assert (P.paged_append(b["q"], b["k"], b["v"], b["k_pages"], b["v_pages"], none["table"], none["kv_len"], none["cu_q"]) == 0).all()


@pytest.mark.parametrize("G", [72, 128, 160])
def test_large_groups(G):
    b = make_batch([1, 3, 9], [50, 131, 9], G, 1, 128, 32, DEV, seed=G)
    check(attend(b), b)


@pytest.mark.parametrize("max_q", [0, 1, 2, 10 ** 6, 2 ** 40])
def test_a_wrong_max_q_only_costs_time(max_q):
    b = make_batch([1, 50, 3], [700, 600, 5], 8, 2, 128, 16, DEV, seed=8)
    o = P.paged_attention(b["q"], b["k_pages"], b["v_pages"], b["table"], b["kv_len"], cu_q=b["cu_q"], max_q=max_q)
    check(o, b)


def test_one_token_batches_of_every_split():
    """Whole items, clusters of 2 to 8 and equal shares, with lengths far below what the table allows."""
    for n, cols in ((1, 300), (3, 40), (9, 40), (18, 40), (40, 40), (150, 40), (7, 3)):
        kv = [(i * 61 + 1) % min(16 * cols, 700) for i in range(n)]
        b = make_batch([1] * n, kv, 16, 8, 128, 16, DEV, seed=n)
        wide = torch.full((n, cols), -5, dtype=torch.int32, device=DEV)
        w = min(cols, b["table"].shape[1])
        wide[:, :w] = b["table"][:, :w]
        check(attend({**b, "table": wide}, one=True), b)


def test_offsets_past_32_bits():
    """The last pages of a pool of more than 2^31 elements, through every operator."""
    page, Hkv, D, n_pages = 64, 8, 128, 2 ** 31 // (64 * 8 * 128) + 40
    pool = torch.empty(2, n_pages, page, Hkv, D, dtype=torch.bfloat16, device=DEV)
    last = torch.arange(n_pages - 20, n_pages, device=DEV).int()
    for q, kv in (([1, 1], [300, 129]), ([70, 200], [300, 700])):
        b = make_batch(q, kv, 16, Hkv, D, page, DEV, poison=False)
        old, used = b["table"], b["k_pages"].shape[0]
        assert used <= 20
        pool[0, last[:used].long()], pool[1, last[:used].long()] = b["k_pages"], b["v_pages"]
        big = {**b, "k_pages": pool[0], "v_pages": pool[1], "table": torch.where(old >= 0, last[old.long().clamp(min=0)], old)}
        P.paged_append(b["q"], b["k"], b["v"], b["k_pages"], b["v_pages"], old, b["kv_len"], b["cu_q"])
        P.paged_append(b["q"], b["k"], b["v"], pool[0], pool[1], big["table"], b["kv_len"], b["cu_q"])
        assert torch.equal(pool[0, last[:used].long()], b["k_pages"]) and torch.equal(pool[1, last[:used].long()], b["v_pages"])
        assert torch.equal(attend(big), attend(b))
    P.copy_pages(pool, last[:3].contiguous(), torch.tensor([0, 5, n_pages - 1], dtype=torch.int32, device=DEV))
    for s, d in zip(last[:3].tolist(), (0, 5, n_pages - 1)):
        assert torch.equal(pool[:, d], pool[:, s])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("q,kv", [([1, 1], [100, 40]), ([1], [511]), ([1, 1], [20001, 70]), ([5], [9000]), ([300, 40], [9000, 90])])
def test_what_is_not_a_number_stays_so(q, kv, D):
    """A NaN among the scores that a row sees gives NaN, whichever way the row's keys are cut up; other rows are as before."""
    b = make_batch(q, kv, 8, 2, D, 64, DEV, seed=D + kv[0])
    one = max(q) == 1
    ref, mag = attention64(b)
    tol = attention_tolerance(ref, mag)

    def expect(o, lost):
        assert torch.equal(torch.isnan(o), lost)
        assert ((o.double() - ref).abs() <= tol)[~lost].all()

    dirty = dict(b, q=b["q"].clone())
    dirty["q"][0, 3, 7] = float("nan")
    lost = torch.zeros(ref.shape, dtype=torch.bool, device=DEV)
    lost[0, 3] = True
    expect(attend(dirty, one=one), lost)
    at = kv[0] - 1 - q[0] // 2  # a key that the first sequence's later rows see
    b["k_pages"][b["table"][0, at // 64].item(), at % 64, 1, 9] = float("nan")
    lost = torch.zeros(ref.shape, dtype=torch.bool, device=DEV)
    lost[q[0] - 1 - q[0] // 2:q[0], 4:] = True
    expect(attend(b, one=one), lost)


def test_two_graphs_at_once():
    """Graphs of calls that cut sequences up, replayed on two streams at the same time: neither disturbs the other's parts."""
    cases = [([1, 1, 1], [30000, 17, 9000]), ([300, 1], [9000, 4000])]
    graphs, outs, want = [], [], []
    for q, kv in cases:
        b = make_batch(q, kv, 8, 2, 128, 64, DEV, seed=kv[0])
        one = max(q) == 1
        want.append(attend(b, one=one))
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = attend(b, one=one)
        graphs.append((g, b))  # the inputs stay where the graph reads them
        outs.append(o)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(20):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for (g, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))
    _lib.check_status()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,Hkv", [(8, 8), (24, 2)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (130, 3)])
def test_many_items_a_block(H, Hkv, D, window, sinks):
    """More items than blocks of the grid, of one to forty key blocks: an item's first keys arrive while the one before is joined."""
    g = torch.Generator().manual_seed(D + H)
    kv = torch.randint(0, 700, (160,), generator=g).tolist() + [2500, 64, 65, 0, 1, 2560]
    b = make_batch([1] * len(kv), kv, H, Hkv, D, 32, DEV, seed=H, release=(window, sinks) if window else None)
    o = attend(b, one=True, window=window, sinks=sinks)
    check(o, b, window, sinks)
    assert torch.equal(o, attend(b, one=True, window=window, sinks=sinks))
    b = make_batch([1] * 200, [40 + i % 200 for i in range(200)], H, Hkv, D, 32, DEV, seed=H)  # items that are not cut up
    check(attend(b, one=True), b)
