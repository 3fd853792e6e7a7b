"""The reference for gathered attention weights: its two forms agree, fp32 weights keep its bound, and weights rounded to 16
bits, which it is there to find, do not."""
import pytest
import torch

from oracle import evict_ref as E


def rows(seed, lq, lk, Hq, H, D, dtype):
    g = torch.Generator().manual_seed(seed)
    q, k = torch.randn(lq, Hq, D, generator=g).to(dtype), torch.randn(lk, H, D, generator=g).to(dtype)
    return q, k


@pytest.mark.parametrize("lq,lk,kw", [(1, 6000, {}), (40, 300, {}), (40, 300, dict(window=70)), (30, 20, {}), (9, 100, dict(causal=False)),
                                      (5, 0, {})])
def test_both_forms_agree(lq, lk, kw):
    q, k = rows(lq, lq, lk, 4, 2, 64, torch.float16)
    a, coarse = E.weights(q, k, 0.125, **kw)
    b, bound = E.gathered(q, k, 0.125, **kw)
    assert bool(((a - b).abs() <= 1e-13 + 1e-12 * a).all())
    assert lk < 6000 or bool((4 * bound <= coarse).all())


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lk", [700, 3000, 6000])
def test_bound(lk, D):
    q, k = rows(lk, 1, lk, 2, 2, D, torch.float16)
    scale = D ** -0.5
    want, bound = E.gathered(q, k, scale)
    s = torch.stack([k[:, h].float() @ q[0, h].float() for h in range(2)]) * torch.tensor(scale, dtype=torch.float32)
    assert bool(((torch.softmax(s, -1).double() - want).abs() <= bound).all())
    for rounded in (want.half().double(), want.bfloat16().double()):
        missed = ((rounded - want).abs() > bound).double().mean()
        assert missed > 0.1, float(missed)
