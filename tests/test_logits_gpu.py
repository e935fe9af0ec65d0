"""Logits kernel against the 64-bit form. One rounding to the output type, and the fp32 steps before it."""
import math

import pytest
import torch

from lingua_b200.ops.logits import penalize_logits
from paged_oracle import penalize64

pytestmark = pytest.mark.gpu
DEV = "cuda"


def inputs(N, V, L, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(N, V, generator=g) * 3).to(dtype)
    hist = (V ** torch.rand(N, L, generator=g)).long().clamp(max=V) - 1
    if L > 3:
        hist[:, 1] = hist[:, 0]
        hist[0, 2], hist[-1, 3] = V + 7, -1
    hl = torch.randint(0, L + 1, (N,), generator=g).int()
    pl = (hl.float() * torch.rand(N, generator=g)).int()
    rep, pres, freq = 0.5 + torch.rand(N, generator=g), torch.rand(N, generator=g), 0.3 * torch.rand(N, generator=g)
    bias = torch.randn(N, V, generator=g)
    allowed = torch.randint(-2 ** 31, 2 ** 31, (N, (V + 31) // 32), generator=g).int()
    return x, hist, hl, pl, rep, pres, freq, bias, allowed


def close(z, ref, dtype):
    # terms up to 2^4 in size: each fp32 operation (at most five) is off by half a step of its result, 2^-24 of it, and a
    # frequency of up to 2^9 occurrences scales the largest to 0.3 * 2^9; the result is rounded once more to its type
    z = z.double().cpu()
    assert torch.equal(torch.isneginf(z), torch.isneginf(ref))
    fin = ~torch.isinf(ref)
    tol = ref.abs() * torch.finfo(dtype).eps / 2 + 5 * 2 ** -24 * (16 + 0.3 * 2 ** 9 * 2)
    assert ((z - ref).abs()[fin] <= tol[fin]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N,V,L", [(1, 1, 1), (1, 258, 200), (3, 4097, 0), (5, 5003, 700), (2, 33000, 5000)])
def test_everything_on(N, V, L, dtype):
    x, hist, hl, pl, rep, pres, freq, bias, allowed = inputs(N, V, L, dtype)
    cu = [t.to(DEV) for t in (x, hist, hl, pl, rep, pres, freq, bias, allowed)]
    z = penalize_logits(*cu[:3], prompt_len=cu[3], repetition=cu[4], presence=cu[5], frequency=cu[6], bias=cu[7], allowed=cu[8])
    assert z.dtype == dtype
    close(z, penalize64(x, hist, hl, pl, rep.tolist(), pres.tolist(), freq.tolist(), bias, allowed), dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_each_alone_numbers_strides_and_in_place(dtype):
    N, V, L = 3, 1001, 60
    x, hist, hl, pl, rep, pres, freq, bias, allowed = inputs(N, V, L, dtype, 1)
    one, zero = [1.0] * N, [0.0] * N
    X, Hh, Hl, Pl = (t.to(DEV) for t in (x, hist, hl, pl))
    wide = torch.zeros(N, V + 3, dtype=dtype, device=DEV)
    wide[:, 1:V + 1] = X
    view = wide[:, 1:V + 1]  # rows with a pitch, unaligned
    close(penalize_logits(view, Hh, Hl, repetition=1.7), penalize64(x, hist, hl, None, [1.7] * N, zero, zero, None, None), dtype)
    close(penalize_logits(X, Hh, Hl, Pl, presence=0.4), penalize64(x, hist, hl, pl, one, [0.4] * N, zero, None, None), dtype)
    close(penalize_logits(X, Hh, Hl, Pl, frequency=0.2), penalize64(x, hist, hl, pl, one, zero, [0.2] * N, None, None), dtype)
    close(penalize_logits(X, Hh, Hl, bias=bias[1].to(DEV)), penalize64(x, hist, hl, None, one, zero, zero, bias[1], None), dtype)
    assert torch.equal(penalize_logits(X, Hh, Hl), X)
    wide_hist = torch.cat((Hh, Hh), dim=1)[:, :L]
    out = penalize_logits(view, wide_hist, Hl, Pl, repetition=1.2, allowed=allowed.to(DEV), out=view)
    assert out is view
    close(out, penalize64(x, hist, hl, pl, [1.2] * N, zero, zero, None, allowed), dtype)
    assert (wide[:, 0] == 0).all() and (wide[:, V + 1:] == 0).all()


def test_nothing_allowed_nan_and_infinities():
    x = torch.randn(3, 100)
    x[0, 5], x[1, 6], x[1, 7], x[2, 8] = math.nan, math.inf, -math.inf, math.nan
    allowed = torch.zeros(3, 4, dtype=torch.int32)
    allowed[1:] = -1
    hist = torch.tensor([[5, 6], [6, 7], [8, 8]])
    z = penalize_logits(x.to(DEV), hist.to(DEV), torch.tensor([2, 2, 2], dtype=torch.int32, device=DEV), repetition=2.0,
                        allowed=allowed.to(DEV)).cpu()
    assert torch.isneginf(z[0]).all()  # the NaN is masked away
    assert z[1, 6] == math.inf and z[1, 7] == -math.inf
    assert torch.isnan(z[2, 8]) and torch.equal(z[2, :8], x[2, :8])  # one that is allowed shows


def test_refusals_on_the_gpu():
    x, hist, hl, *_ = inputs(2, 64, 4, torch.float32)
    X, Hh, Hl = x.to(DEV), hist.to(DEV), hl.to(DEV)
    for a, kw in (((X.half(), Hh, Hl), {}), ((X.double(), Hh, Hl), {}), ((X, hist, Hl), {}), ((X[:, ::2], Hh, Hl), {}),
                  ((X, Hh, Hl), dict(repetition=torch.ones(2))), ((X, Hh[:, ::2], Hl), {})):
        with pytest.raises(ValueError):
            penalize_logits(*a, **kw)
    with pytest.raises(ValueError):
        penalize_logits(X, Hh, Hl, out=torch.empty(1, 64, device=DEV).expand(2, 64))
    assert penalize_logits(X[:0], Hh[:0], Hl[:0]).shape == (0, 64)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_destinations(dtype):
    both = torch.randn(3, 2 * 5000 + 24, device=DEV).to(dtype)
    left, right = both[:, :5000], both[:, 5008:10008]
    hist = torch.randint(0, 5000, (3, 50), device=DEV)
    kw = dict(history=hist, history_len=torch.tensor([50, 0, 7], dtype=torch.int32, device=DEV), repetition=1.5, frequency=0.25)
    want = penalize_logits(left, **kw)
    penalize_logits(left, **kw, out=right)
    assert torch.equal(right, want)
    for bad in (both[:, 8:5008], both[:, 4992:9992], both.view(-1)[8000:23000].view(3, 5000)):
        with pytest.raises(ValueError):
            penalize_logits(left, **kw, out=bad)
    penalize_logits(left, **kw, out=left)
    assert torch.equal(left, want)
