"""Dropping tokens from 4-bit pages on the GPU (PagedStore.evict, append(evicted=)) against plain definitions
(oracle/evict_ref.py): which tokens stay, where they go, and that nothing else changes."""
import random

import numpy as np
import pytest
import torch

from innerq_amd import ops, paged
from oracle import evict_ref as E
from oracle import serving_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def case(lens, H, D, seed, width=None, T=None, dtype=torch.float16):
    """A store of random words (any codes, scales and zeros), its table, and weights with 0 behind the ends."""
    rng, g = random.Random(seed), torch.Generator().manual_seed(seed)
    P = width or max(1, max(-(-n // 64) for n in lens))
    pool = len(lens) * P + 3
    ids = rng.sample(range(pool), len(lens) * P)
    table = i32(ids).view(len(lens), P)
    st = paged.PagedStore(pool, H, D, DEV, dtype)
    words = torch.randint(-2 ** 31, 2 ** 31 - 1, st.pages.shape, generator=g, dtype=torch.int64)
    st.pages.copy_(words.to(torch.int32))
    w = torch.rand(len(lens), H, T or P * 64, generator=g) ** 4
    for s, n in enumerate(lens):
        w[s, :, max(n, 0):] = 0
    return st, table, w.to(DEV)


def check(st, table, lens, w, keep, recent=0, sinks=0, shared=1, in_place=False):
    before, w0 = st.pages.cpu(), w.cpu().numpy().copy()
    ll = i32(lens)
    if in_place:
        out, new = st.evict(table, ll, w, keep, recent, sinks, shared, out=w, lens_out=ll)[::-1]
        assert out is w and new is ll
    else:
        new, out = st.evict(table, ll, w, keep, recent, sinks, shared)
        assert np.array_equal(w.cpu().numpy(), w0, equal_nan=True) and ll.tolist() == lens
    st.check()
    assert new.tolist() == [min(n, keep) for n in lens]
    after, tab, got = st.pages.cpu(), table.cpu().numpy(), out.cpu().numpy()
    want_pages = before.numpy().view(np.uint32).copy()
    H, D = st.H, st.D
    for s, n in enumerate(lens):
        if n <= keep:
            assert np.array_equal(got[s], w0[s], equal_nan=True), s
            continue
        was, now = E.token_words(before, tab[s], n, D), E.token_words(after, tab[s], n, D)
        for h0 in range(0, H, shared):
            total = w0[s, h0].copy()
            for h in range(h0 + 1, h0 + shared):
                total = total + w0[s, h]  # in fp32, head by head
            src = E.kept(total[:n], keep, recent, sinks)
            for h in range(h0, h0 + shared):
                assert np.array_equal(now[h, :keep], was[h, src]), (s, h)
                assert np.array_equal(now[h, keep:], was[h, keep:]), (s, h)
                assert np.array_equal(got[s, h, :keep], w0[s, h, src], equal_nan=True), (s, h)
                assert not got[s, h, keep:].any(), (s, h)
    mine = set()
    for s, n in enumerate(lens):
        if n > keep:
            mine |= set(tab[s, :-(-n // 64)].tolist())
    rest = [i for i in range(before.shape[0]) if i not in mine]
    assert torch.equal(before[rest], after[rest])
    return out


@pytest.mark.parametrize("D,H", [(128, 2), (64, 3)])
@pytest.mark.parametrize("lens", [[200, 64, 65, 1, 0, 128], [1500, 700, 300]])
@pytest.mark.parametrize("keep,recent,sinks", [(64, 0, 0), (64, 10, 0), (100, 30, 4), (1, 0, 0), (1, 1, 0), (1, 0, 1), (128, 128, 0),
                                               (65, 64, 1), (199, 150, 0), (299, 5, 3), (2000, 100, 0)])
@pytest.mark.parametrize("in_place", [False, True])
def test_what_stays_and_where(D, H, lens, keep, recent, sinks, in_place):
    st, table, w = case(lens, H, D, keep + recent + sum(lens))
    check(st, table, lens, w, keep, recent, sinks, in_place=in_place)


@pytest.mark.parametrize("H,shared", [(4, 2), (4, 4), (6, 3), (2, 2)])
def test_heads_that_keep_the_same(H, shared):
    lens = [300, 90, 40]
    st, table, w = case(lens, H, 64, H + shared)
    check(st, table, lens, w, 80, 20, 2, shared)


@pytest.mark.parametrize("keep,recent", [(4096, 512), (4095, 0), (700, 700), (9000, 3000), (8999, 8999), (5000, 1)])
def test_long_sequences(keep, recent):
    """Past one turn of the selecting workgroup, of the rows that come and of the recent ones."""
    lens = [9001, 4097, 5000]
    st, table, w = case(lens, 1, 64, keep, T=142 * 64 + 5)
    check(st, table, lens, w, keep, recent, in_place=recent % 2 == 0)


def test_longer_than_one_histogram():
    lens = [40000]
    st, table, w = case(lens, 1, 64, 9)
    check(st, table, lens, w, 2048, 64, 4)


@pytest.mark.parametrize("values", ["equal", "zero", "two", "special", "negative", "near"])
@pytest.mark.parametrize("keep,recent,sinks", [(100, 20, 0), (64, 0, 3), (1500, 10, 0)])
def test_ties_and_special_weights(values, keep, recent, sinks):
    """Equal weights (the first stay), zeros of both signs, infinities, NaN, negative ones, neighbours in the last bit."""
    lens = [2100, 130]
    st, table, w = case(lens, 2, 64, keep)
    g = torch.Generator().manual_seed(1)
    shape = w.shape
    x = {"equal": torch.full(shape, 0.25), "zero": torch.randint(0, 2, shape, generator=g) * -0.0,
         "two": torch.randint(0, 2, shape, generator=g) + 0.5,
         "special": torch.tensor([float("nan"), float("inf"), -float("inf"), 0.0, -0.0, 1e-45, 3e38, -float("nan")])[
             torch.randint(0, 8, shape, generator=g)],
         "negative": torch.randn(shape, generator=g), "near": 1 + torch.randint(0, 50, shape, generator=g) * 2.0 ** -23}[values]
    w.copy_(x.float())
    check(st, table, lens, w, keep, recent, sinks)


def test_weights_of_other_strides():
    lens = [150, 80, 300]
    st, table, w = case(lens, 2, 64, 5, T=400)
    for x in (w.transpose(0, 1).contiguous().transpose(0, 1), torch.zeros(3, 2, 801, device=DEV)[..., 1:401].copy_(w)):
        check(st, table, lens, x, 70, 7)
    both = torch.zeros(3, 4, 400, device=DEV)
    both[:, :2] = w
    want = st.evict(table, i32([0, 0, 0]), w, 70)[1]
    new, out = st.evict(table, i32([0, 0, 0]), both[:, :2], 70, out=both[:, 2:])
    assert torch.equal(out, want) and torch.equal(both[:, :2], w)
    one = w[:1, :1].expand(3, 2, 400)  # one row of weights for all
    check(st, table, lens, one, 70, 7)


def test_many_sequences():
    rng = random.Random(3)
    lens = [rng.choice([0, 5, 64, 100, 129]) for _ in range(300)]
    st, table, w = case(lens, 1, 64, 6)
    check(st, table, lens, w, 70, 12, 1, in_place=True)


def test_bad_lengths_and_pages():
    lens = [-1, 129, 100, 128, 100]
    st, table, w = case([128] * 5, 2, 64, 7)
    before, w0 = st.pages.clone(), w.clone()
    new, out = st.evict(table[:2], i32(lens[:2]), w[:2], 70)
    assert new.tolist() == lens[:2] and torch.equal(out, w0[:2]) and torch.equal(st.pages, before)
    with pytest.raises(RuntimeError, match="negative length"):
        st.check()
    # a row whose source has no page becomes NaN; one whose place has none is not written
    w[2, :, :70] = 0
    w[2, :, 70:] = 1
    w[3], w[4] = w[2], w[2]
    table[2, 1] = st.n_pages
    table[3, 0] = -1
    st.evict(table[2:4], i32([100, 100]), w[2:4], 20)
    with pytest.raises(RuntimeError, match="outside the pool"):
        st.check()
    k, v = st.read(table[2:3], i32([0]), i32([0, 20]), 20)
    assert bool(k.isnan().all()) and bool(v.isnan().all())
    same = [i for i in range(st.n_pages) if i != int(table[2, 0])]
    assert torch.equal(st.pages[same], before[same])


def test_pages_that_nobody_drops_may_be_shared():
    lens = [130, 64, 64]
    st, table, w = case(lens, 2, 64, 8)
    table[2] = table[1]
    check(st, table, lens, w, 64, 8)


def test_positions_after_dropping():
    """append(evicted=): a token's rotation row is its place and what its sequence has dropped."""
    g = torch.Generator().manual_seed(2)
    H, D, half = 2, 64, 32
    a = torch.arange(500)[:, None] * 10000.0 ** (-torch.arange(half) / half)
    cos, sin = a.cos().float(), a.sin().float()
    k, v, q = (torch.randn(7, H, D, generator=g).half() for _ in range(3))
    lens, gone, new = [10, 63, 0], [300, 0, 493], [4, 1, 2]
    table = i32([[0, 1], [2, 3], [4, 5]])
    st = paged.PagedStore(6, H, D, DEV)
    got = st.append(k.to(DEV), v.to(DEV), table, i32(lens), i32([0, 4, 5, 7]), cos.to(DEV), sin.to(DEV), q.to(DEV),
                    evicted=i32(gone))
    st.check()
    at = torch.tensor([lens[s] + gone[s] + i for s, n in enumerate(new) for i in range(n)])
    assert torch.equal(got.cpu(), R.rotate(q, cos[at], sin[at]))
    kk, _ = st.read(table, i32(lens), i32([0, 4, 5, 7]), 7)
    assert torch.equal(kk.cpu(), R.value(*R.quantize(R.rotate(k, cos[at], sin[at]))))
    # one step, its rows one per sequence; a row past the table, and a negative one
    one = st.append(k[:3].to(DEV), v[:3].to(DEV), table, i32(lens), None, cos.to(DEV), sin.to(DEV), q[:3].to(DEV),
                    evicted=i32([490, -64, 2]))
    with pytest.raises(RuntimeError, match="rotation"):
        st.check()
    assert one.isnan().all(-1).all(-1).tolist() == [True, True, False]
    assert torch.equal(one[2].cpu(), R.rotate(q[2:3], cos[2:3], sin[2:3])[0])
    for bad in (i32([1, 2]), i32([1, 2, 3]).float(), i32([[1, 2, 3]])):
        with pytest.raises((TypeError, ValueError)):
            st.append(k[:3].to(DEV), v[:3].to(DEV), table, i32(lens), None, cos.to(DEV), sin.to(DEV), evicted=bad)
    with pytest.raises(ValueError, match="rotation"):
        st.append(k[:3].to(DEV), v[:3].to(DEV), table, i32(lens), evicted=i32([1, 2, 3]))


def test_refusals():
    lens = [130, 70]
    st, table, w = case(lens, 2, 64, 10)
    ll, before = i32(lens), st.pages.clone()
    for kw in (dict(keep=0), dict(keep=-5), dict(keep=2 ** 31), dict(keep=10, recent=11), dict(keep=10, recent=-1),
               dict(keep=10, sinks=-1), dict(keep=10, recent=6, sinks=5), dict(keep=10, shared=0), dict(keep=10, shared=3)):
        with pytest.raises(ValueError):
            st.evict(table, ll, w, **kw)
    for bad in (w[:1], w[:, :1], w[..., :191], w.transpose(1, 2), w[0]):
        with pytest.raises(ValueError):
            st.evict(table, ll, bad, 10)
    for bad in (w.double(), w.cpu()):
        with pytest.raises(TypeError):
            st.evict(table, ll, bad, 10)
    big = torch.zeros(2, 2, 400, device=DEV)
    for out in (w[..., :191], w[:1].expand(2, 2, 192), big[..., :200]):
        with pytest.raises(ValueError):
            st.evict(table, ll, w, 10, out=out)
    with pytest.raises(ValueError, match="memory"):
        st.evict(table, ll, big[..., :192], 10, out=big[..., 1:193])
    ints = i32([130, 70, 5])
    for bad in (ints[1:], i32([1]), ints):
        with pytest.raises(ValueError):
            st.evict(table, ints[:2], w, 10, lens_out=bad)
    with pytest.raises(NotImplementedError):
        st.evict(table, ll, w.clone().requires_grad_(), 10)
    assert torch.equal(st.pages, before) and ll.tolist() == lens


def test_captured():
    """A captured call follows the lengths and weights of each replay."""
    st, table, w = case([300, 300], 2, 64, 11)
    ll = i32([300, 300])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        st.evict(table, ll, w, 400)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        new, out = st.evict(table, ll, w, 100, 20, 1)
    pages = st.pages.clone()
    for lens, seed in (([300, 90], 1), ([101, 250], 2), ([0, 100], 3)):
        g = torch.Generator().manual_seed(seed)
        st.pages.copy_(pages)
        ll.copy_(i32(lens))
        w.copy_(torch.rand(w.shape, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        got = new.clone(), out.clone(), st.pages.clone()
        st.pages.copy_(pages)
        want = *st.evict(table, ll, w, 100, 20, 1), st.pages
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_append_evicted_native(monkeypatch):
    """append(evicted=) through the native front and without it: one token per sequence, and ragged rows."""
    g = torch.Generator().manual_seed(40)
    H, D, lens, gone = 2, 64, [70, 3, 130], [9, 0, 400]
    table = torch.arange(12, dtype=torch.int32, device=DEV).view(3, 4)
    ang = torch.rand(700, D // 2, generator=g)
    cos, sin = ang.cos().to(DEV), ang.sin().to(DEV)
    for cu, n in ((None, 3), (i32([0, 5, 5, 11]), 11)):
        k, v, q = (torch.randn(n, h, D, generator=g).half().to(DEV) for h in (H, H, 4))
        got = []
        for native in (True, False):
            with monkeypatch.context() as m:
                if not native:
                    m.setattr(ops, "_native", lambda t: None)
                st = paged.PagedStore(12, H, D, DEV)
                st.pages.zero_()
                out = st.append(k, v, table, i32(lens), cu, cos, sin, q, evicted=i32(gone))
                got.append((out, st.pages.clone(), st.check()))
        assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1]) and got[0][2] == got[1][2]


@pytest.mark.parametrize("S,H,shared", [(70, 4, 1), (300, 2, 2), (33, 8, 1)])
@pytest.mark.parametrize("in_place", [False, True])
def test_many_sequences_and_heads(S, H, shared, in_place):
    """More (sequence, run of heads) pairs than CUs, of lengths from none to several pages."""
    rng = random.Random(41 + S)
    lens = [rng.choice([0, 1, 20, 64, 65, 100, 130, 250]) for _ in range(S)]
    st, table, w = case(lens, H, 64, 41 + S, width=4)
    check(st, table, lens, w, 64, 20, 3, shared, in_place)


@pytest.mark.parametrize("shared", [1, 2])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("lens,keep,recent", [([700], 300, 290), ([900, 40], 512, 100), ([2000, 1000], 800, 600)])
def test_few_pairs_with_many_rows(lens, keep, recent, shared, in_place):
    """Few (sequence, run of heads) pairs: with few rows to move, and with many, apart from their places and over them."""
    st, table, w = case(lens, 2, 64, 50 + keep)
    check(st, table, lens, w, keep, recent, 2, shared, in_place)


@pytest.mark.parametrize("shared", [1, 2])
def test_some_pairs_with_many_rows(shared):
    """More pairs than one, fewer than CUs, more rows than a workgroup moves by itself."""
    lens = [900, 30, 640, 641, 1200, 700, 0, 1000, 800, 950]
    for keep, recent, in_place in ((640, 64, False), (640, 500, True)):
        st, table, w = case(lens, 4, 64, 60 + recent)
        check(st, table, lens, w, keep, recent, 2, shared, in_place)


@pytest.mark.parametrize("shared", [1, 2])
def test_long_cut_to_few(shared):
    """More tokens than a workgroup holds keys of at once, of which few stay."""
    lens = [40000, 33000, 100]
    st, table, w = case(lens, 2, 64, 70)
    check(st, table, lens, w, 400, 50, 4, shared, True)
