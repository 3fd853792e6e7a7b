"""Differential attention over 4-bit pages on the GPU (PagedStore.diff_attend) against 64 bits (oracle/diff_ref.py)."""
import random

import pytest
import torch

from innerq_amd import ops, paged
from oracle import diff_ref as X
from oracle import evict_ref as E

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float16, torch.bfloat16]


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def filled(seed, lens, H, D, dtype, width=None):
    """A store whose sequences hold random tokens (NaN behind their ends), and K and V as the store holds them."""
    g, rng = torch.Generator().manual_seed(seed), random.Random(seed)
    P = width or max(1, max(-(-n // 64) for n in lens))
    pool = sum(-(-n // 64) for n in lens) + 2
    ids = rng.sample(range(pool), pool)
    table = [[-1] * P for _ in lens]
    for s, n in enumerate(lens):
        for i in range(-(-n // 64)):
            table[s][i] = ids.pop()
    table = i32(table)
    st = paged.PagedStore(pool, H, D, DEV, dtype)
    st.pages.fill_(-1)
    N, cu = sum(lens), [0]
    for n in lens:
        cu.append(cu[-1] + n)
    k, v = torch.randn(max(N, 1), H, D, generator=g), torch.randn(max(N, 1), H, D, generator=g)
    k[..., :3] *= 4
    if N:
        st.append(k.to(dtype).to(DEV), v.to(dtype).to(DEV), table, i32([0] * len(lens)), i32(cu))
        k, v = (x.cpu() for x in st.read(table, i32([0] * len(lens)), i32(cu), N))
    return st, table, cu, k, v, g


def check(st, table, cu, k, v, lens, q, lam, scale, window=None, weights=None):
    before = None if weights is None else weights.cpu().clone()
    out = st.diff_attend(q, table, i32(lens), lam, scale, window=window, weights=weights)
    st.check()
    assert out.shape == (*q.shape[:-2], q.shape[-2] // 2, 2 * st.D) and out.dtype == st.dtype
    got, qc, lam = out.cpu().double(), q.cpu(), lam.cpu()
    if q.dim() == 3:
        got, qc = got[:, None], qc[:, None]
    for s, n in enumerate(lens):
        kk, vv = k[cu[s]:cu[s + 1]], v[cu[s]:cu[s + 1]]
        want, bound = X.attention(qc[s], kk, vv.reshape(n, st.H // 2, 2 * st.D), lam, scale, window=window or 0)
        worst = ((got[s] - want).abs() - bound).max()
        assert worst <= 0, (s, n, float(worst))
        if weights is None:
            continue
        now = weights.cpu()[s]
        assert torch.equal(now[:, n:], before[s, :, n:])
        for i in (0, 1) if n else ():
            w, b = E.weights(qc[s][:, i::2], kk[:, i::2], scale, window=window or 0)
            add = before[s, i::2, :n].double()
            assert bool(((now[i::2, :n].double() - add - w).abs() <= b + 2.0 ** -24 * (add + w)).all()), (s, i)
    return out


def lams(g, Hq):
    return (torch.rand(Hq // 2, generator=g) * 0.8 + 0.1).to(DEV)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,H,Hq", [(128, 2, 8), (64, 4, 4), (128, 2, 2), (64, 2, 16), (64, 2, 18), (128, 2, 40), (64, 6, 12)])
@pytest.mark.parametrize("lens", [[1], [2, 63, 64, 65], [0, 5, 0, 300], [1000, 17, 128, 511]])
def test_lengths(dtype, D, H, Hq, lens):
    st, table, cu, k, v, g = filled(sum(lens) + H, lens, H, D, dtype)
    q = torch.randn(len(lens), Hq, D, generator=g).to(dtype).to(DEV)
    w = torch.rand(len(lens), H, table.shape[1] * 64, generator=g).to(DEV)
    out = check(st, table, cu, k, v, lens, q, lams(g, Hq), D ** -0.5, weights=w)
    assert out.isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("m,Hq", [(2, 8), (3, 16), (5, 4), (16, 4), (16, 8), (7, 12)])
@pytest.mark.parametrize("window", [None, 1, 50, 64, 200])
def test_drafts_and_windows(dtype, D, m, Hq, window):
    lens = [m, 3, 0, 64 + m - 1, 333, 1, 600]
    st, table, cu, k, v, g = filled(m, lens, 2, D, dtype, width=11)
    q = torch.randn(len(lens), m, Hq, D, generator=g).to(dtype).to(DEV)
    check(st, table, cu, k, v, lens, q, lams(g, Hq), D ** -0.5, window)


@pytest.mark.parametrize("window", [1, 64, 700, 2 ** 31 - 1])
def test_one_token_windows(window):
    lens = [1, 64, 65, 1500, 0, 129]
    st, table, cu, k, v, g = filled(3, lens, 2, 128, torch.float16)
    q = torch.randn(6, 4, 128, generator=g).half().to(DEV)
    w = torch.rand(6, 2, table.shape[1] * 64, generator=g).to(DEV)
    check(st, table, cu, k, v, lens, q, lams(g, 4), 0.1, window, w)


@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0])
@pytest.mark.parametrize("dtype", DTYPES)
def test_scales_and_factors(scale, dtype):
    lens = [300, 1, 64]
    st, table, cu, k, v, g = filled(4, lens, 4, 64, dtype)
    q = torch.randn(3, 8, 64, generator=g).to(dtype).to(DEV)
    lam = lams(g, 8)
    for x in (lam, -lam, lam * 0, lam * 20, lam[:1].expand(4), torch.stack([lam, lam], 1)[:, 1]):
        check(st, table, cu, k, v, lens, q, x, scale)


@pytest.mark.parametrize("S,H,width", [(2, 2, 8), (2, 2, 9), (16, 8, 16), (16, 8, 17), (64, 8, 32), (64, 8, 33), (300, 2, 40)])
@pytest.mark.parametrize("rep", [1, 9])
def test_table_widths(S, H, width, rep):
    """Both sides of the widths up to which a workgroup takes a whole sequence and pair, both tilings of the maps."""
    rng = random.Random(S)
    lens = [rng.choice([0, 1, 64, 130]) for _ in range(S)]
    lens[0], lens[S - 1] = width * 64, 200
    st, table, cu, k, v, g = filled(width, lens, H, 64, torch.float16, width)
    q = torch.randn(S, rep * H, 64, generator=g).half().to(DEV)
    check(st, table, cu, k, v, lens, q, lams(g, rep * H), 0.125)


def test_long_over_many_workgroups():
    """One sequence that all workgroups share, so that many partials are merged (in runs, for few rows)."""
    lens = [9000]
    for D, Hq in ((64, 2), (128, 8), (64, 24)):
        st, table, cu, k, v, g = filled(5, lens, 2, D, torch.float16)
        q = torch.randn(1, Hq, D, generator=g).half().to(DEV)
        w = torch.zeros(1, 2, table.shape[1] * 64, device=DEV)
        check(st, table, cu, k, v, lens, q, lams(g, Hq), D ** -0.5, weights=w)


@pytest.mark.parametrize("width,Hq", [(8, 4), (40, 4), (8, 40), (40, 40)])
def test_special_values(width, Hq):
    """Infinite and NaN queries, keys and pages: one map's do not reach other rows, heads, sequences, or the other map."""
    lens = [200, 100, 130, 64]
    st, table, cu, k, v, g = filled(6, lens, 4, 64, torch.float16, width)
    ll = i32(lens)
    q = torch.randn(4, Hq, 64, generator=g).half().to(DEV)
    lam = lams(g, Hq)
    want = st.diff_attend(q, table, ll, lam, 0.1)
    bad = q.clone()
    bad[0, 1, 3] = float("nan")  # second map of output head 0
    out = st.diff_attend(bad, table, ll, lam, 0.1)
    assert bool(out[0, 0].isnan().all()) and torch.equal(out[0, 1:], want[0, 1:]) and torch.equal(out[1:], want[1:])
    bad_table = table.clone()
    bad_table[1, 0] = -7
    out = st.diff_attend(q, bad_table, i32([200, 100, width * 64 + 1, 64]), lam, 0.1)
    with pytest.raises(RuntimeError, match="outside the pool and a token past"):
        st.check()
    assert bool(out[1:3].isnan().all()) and torch.equal(out[0], want[0]) and torch.equal(out[3], want[3])
    out = st.diff_attend(q, table, i32([200, -3, 130, 64]), lam, 0.1)
    with pytest.raises(RuntimeError, match="negative length"):
        st.check()
    assert bool((out[1] == 0).all()) and torch.equal(out[0], want[0]) and torch.equal(out[2:], want[2:])
    # token 7 of sequence 2: minus infinity among the first map's keys of pair 0 for queries of one sign, so that it gets no
    # weight there; the second map sees the same token as it was
    pages = st.pages.clone()
    half = st.pages.view(torch.int16)
    page = int(table[2, 0])
    half[page, 0, 2 * (64 * 8 + 7 * 2) + 1] = -1024  # K zero point of head 0, token 7, group 0
    x = q.abs()
    ref = paged.PagedStore.over(st.pages, 64)
    out = ref.diff_attend(x, table, ll, lam, 0.1)
    kk, vv = (t.cpu() for t in st.read(table[2:3], i32([0]), i32([0, 130]), 130))
    assert bool((kk[7, 0, :32] == float("-inf")).all())
    first = kk.clone()
    first[7, 0, :32] = -60000.0  # a weight of 0 in 64 bits too
    w, b = X.attention(x[2:3].cpu(), first, vv.reshape(130, 2, 128), lam.cpu(), 0.1)
    _, b = X.attention(x[2:3].cpu(), kk.nan_to_num(neginf=-8.0), vv.reshape(130, 2, 128), lam.cpu(), 0.1)
    assert bool(((out[2:3].cpu().double() - w).abs() <= b).all())
    st.pages.copy_(pages)


def test_an_infinite_value_reaches_what_sees_it():
    lens = [150]
    st, table, cu, k, v, g = filled(7, lens, 2, 64, torch.float16)
    q = torch.randn(1, 3, 4, 64, generator=g).half().to(DEV)
    lam = lams(g, 4)
    want = st.diff_attend(q, table, i32(lens), lam, 0.1)
    # V head 1 (dims 64 .. 127 of the pair's), token 148, group 0: seen by the last two of three new tokens
    row = 148 % 64
    b, p = row // 32 * 4 + row % 16 // 4, row % 4 + row // 16 % 2 * 4
    half = st.pages.view(torch.int16)
    vm = 64 * 8 + 64 * 2 + 64 * 8
    half[int(table[0, 2]), 1, 2 * vm + (b * 2) * 16 + 8 + p] = 31744  # +inf
    out = st.diff_attend(q, table, i32(lens), lam, 0.1)
    hit = torch.zeros_like(out, dtype=torch.bool)
    hit[0, 1:, :, 64:96] = True
    # (in such a page the token is added by itself: other sums may round otherwise)
    near = (out.float() - want.float()).abs() <= 2 * torch.finfo(torch.float16).eps * want.float().abs().clamp(min=2.0 ** -4)
    assert not bool(out[hit].isfinite().any()) and bool(near[~hit].all())


def test_queries_strides_streams_and_graphs():
    lens = [700, 30, 400]
    st, table, cu, k, v, g = filled(8, lens, 4, 128, torch.bfloat16, 40)
    ll = i32(lens)
    q = torch.randn(3, 8, 128, generator=g).bfloat16().to(DEV)
    lam = lams(g, 8)
    want = st.diff_attend(q, table, ll, lam, 0.1)
    wide = torch.zeros(3, 17, 128, dtype=q.dtype, device=DEV)
    wide[:, 5:13] = q
    odd = torch.zeros(3, 8, 132, dtype=q.dtype, device=DEV)[..., 2:130]
    odd.copy_(q)
    o = torch.full((3, 2, 4, 256), 5.0, dtype=q.dtype, device=DEV)
    assert torch.equal(st.diff_attend(wide[:, 5:13], table, ll, lam, 0.1, out=o[:, 1]), want) and bool((o[:, 0] == 5).all())
    assert torch.equal(st.diff_attend(odd, table, ll, lam, 0.1), want)
    assert torch.equal(st.diff_attend(q[:, None], table, ll, lam, 0.1)[:, 0], want)
    w = torch.zeros(3, 4, 2560, device=DEV)
    assert torch.equal(st.diff_attend(q, table, ll, lam, 0.1, weights=w), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        st.diff_attend(q, table, ll, lam, 0.1, weights=w)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    table.clamp_(min=0)
    with torch.cuda.graph(graph, stream=side):
        o = st.diff_attend(q, table, ll, lam, 0.1, weights=w)
    for n, f in (([700, 30, 400], 0.5), ([5, 64, 0], -1.0), ([640, 1, 65], 0.0)):
        ll.copy_(i32(n))
        lam.fill_(f)
        w.zero_()
        graph.replay()
        torch.cuda.synchronize()
        x = torch.zeros_like(w)
        y = st.diff_attend(q, table, ll, lam, 0.1, weights=x)
        assert torch.equal(o.nan_to_num(7.0), y.nan_to_num(7.0)) and torch.equal(w.nan_to_num(7.0), x.nan_to_num(7.0))


@pytest.mark.parametrize("D,dtype", [(64, torch.float16), (128, torch.bfloat16)])
def test_prompt_weights_of_both_maps(D, dtype):
    g = torch.Generator().manual_seed(9)
    lens, H, Hq = [200, 70], 4, 8
    q, k, v = (torch.randn(270, h, d, generator=g).to(dtype).to(DEV) for h, d in ((Hq, D), (H, D), (H // 2, 2 * D)))
    cu, lam = i32([0, 200, 270]), lams(g, Hq)
    w = torch.rand(2, H, 200, generator=g).to(DEV)
    before = w.cpu().double()
    want = ops.diff_prompt_attention(q, k, v, cu, lam, 0.1, window=90)
    assert torch.equal(ops.diff_prompt_attention(q, k, v, cu, lam, 0.1, window=90, weights=w), want)
    for s, (a, n) in enumerate(((0, 200), (200, 70))):
        for i in (0, 1):
            x, b = E.weights(q[a:a + n, i::2].cpu(), k[a:a + n, i::2].cpu(), 0.1, window=90)
            old = before[s, i::2, :n]
            assert bool(((w[s, i::2, :n].cpu().double() - old - x).abs() <= b + 2.0 ** -24 * (old + x)).all()), (s, i)
    assert torch.equal(w[1, :, 70:].cpu().double(), before[1, :, 70:])


def test_refusals():
    lens = [100, 30]
    st, table, cu, k, v, g = filled(10, lens, 4, 64, torch.float16)
    ll = i32(lens)
    q, lam = torch.randn(2, 8, 64, generator=g).half().to(DEV), lams(g, 8)
    w = torch.zeros(2, 4, 128, device=DEV)
    three = paged.PagedStore(4, 3, 64, DEV)
    for a in ((q[:, :6], table, ll, lam[:3]), (q[:1], table, ll, lam), (q[..., :32], table, ll, lam), (q, table, ll, lam[:3]),
              (q, table, ll, lam[None]), (q, table, ll[:1], lam), (q[:, None].expand(2, 17, 8, 64), table, ll, lam),
              (q[:, :0], table, ll, lam[:0])):
        with pytest.raises(ValueError):
            st.diff_attend(*a, 0.1)
    with pytest.raises(ValueError, match="even"):
        three.diff_attend(q[:, :6], table, ll, lam[:3], 0.1)
    for a in ((q.float(), table, ll, lam), (q, table, ll, lam.half()), (q, table, ll, 0.3), (q, table, ll, lam.cpu()),
              (q.cpu(), table, ll, lam)):
        with pytest.raises(TypeError):
            st.diff_attend(*a, 0.1)
    for kw in (dict(window=0), dict(window=-1), dict(out=q), dict(out=torch.empty(2, 4, 64, dtype=q.dtype, device=DEV)),
               dict(out=torch.empty(1, 4, 128, dtype=q.dtype, device=DEV).expand(2, 4, 128)), dict(weights=w[:, :2]),
               dict(weights=w[..., :127])):
        with pytest.raises(ValueError):
            st.diff_attend(q, table, ll, lam, 0.1, **kw)
    with pytest.raises(ValueError, match="one new token"):
        st.diff_attend(q[:, None].expand(2, 2, 8, 64), table, ll, lam, 0.1, weights=w)
    for x in (q, lam):
        y = x.clone().requires_grad_()
        with pytest.raises(NotImplementedError):
            st.diff_attend(y if x is q else q, table, ll, y if x is lam else lam, 0.1)
