"""Edges of the calls for many sequences (4-bit pages, packed prompts) on the GPU: what they refuse, and what they give
for tokens that they leave out."""
import random

import pytest
import torch

from innerq_amd import ops, paged
from oracle import serving_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float16, torch.bfloat16]


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def randn(g, *shape, dtype=torch.float16):
    return torch.randn(*shape, generator=g).to(dtype).to(DEV)


@pytest.fixture(params=["native", "general"])
def front(request, monkeypatch):
    """The same calls through csrc/iq_pyfast.cpp and through the Python path alone."""
    if request.param == "general":
        monkeypatch.setattr(ops, "_native", lambda t: None)


@pytest.mark.parametrize("shape", [(0, 32), (10, 0), (0, 0)])
def test_empty_rotation_tables_are_refused(front, shape):
    """They are no "no rotation": nothing is appended."""
    g = torch.Generator().manual_seed(0)
    st = paged.PagedStore(2, 2, 64, DEV)
    st.pages.fill_(0x11111111)
    before = st.pages.clone()
    k, q = randn(g, 2, 2, 64), randn(g, 2, 4, 64)
    empty = torch.zeros(*shape, device=DEV)
    with pytest.raises(ValueError, match="rotation"):
        st.append(k, k, i32([[0], [1]]), i32([3, 4]), cos=empty, sin=empty, q=q)
    assert torch.equal(st.pages, before)


def angles(n, half):
    a = torch.arange(n)[:, None] * 10000.0 ** (-torch.arange(half) / half)
    return a.cos().float().to(DEV), a.sin().float().to(DEV)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,H,Hq,each", [(64, 2, 4, 5), (128, 1, 3, 70), (128, 8, 32, 500)])
@pytest.mark.parametrize("in_place", [False, True])
def test_tokens_that_append_refuses_are_nan(front, dtype, D, H, Hq, each, in_place):
    """Sequence 0 fits; 1 runs past the rotation's rows, 2 past the table too, 3 needs a page outside the pool, 4 has a
    negative length: their tokens' queries are NaN, and so is what read and attend give for the rows that have pages."""
    g = torch.Generator().manual_seed(D + each)
    S, P, n_pos = 5, -(-(each + 40) // 64) + 1, each + 30
    held = [2, n_pos - each // 3, P * 64 - 2, 0, -2]
    cos, sin = angles(P * 64, D // 2)
    N = S * each
    k, v, q = randn(g, N, H, D, dtype=dtype), randn(g, N, H, D, dtype=dtype), randn(g, N, Hq, D, dtype=dtype)
    cu = i32([each * s for s in range(S + 1)])
    table = torch.arange(S * P, dtype=torch.int32, device=DEV).view(S, P).clone()
    st, want = (paged.PagedStore(S * P, H, D, DEV, dtype) for _ in range(2))
    for x in (st, want):
        x.pages.fill_(0x3C003C00)  # finite values: a row that is left as it was would pass for a token
    turned = want.append(k, v, table, i32([2, held[1], 0, 0, 0]), cu, cos, sin, q)
    table[3] = S * P
    fine = torch.zeros(N, dtype=torch.bool)
    for s in (0, 1, 2):
        most = [n_pos, n_pos, P * 64][s]
        fine[s * each:(s + 1) * each] = torch.arange(each) + held[s] < min(most, n_pos, P * 64)
    assert bool(fine[:each].all()) and 0 < int(fine[each:2 * each].sum()) < each and not bool(fine[2 * each:].any())
    q_out = q.clone() if in_place else None
    got = st.append(k, v, table, i32(held), cu, cos[:n_pos], sin[:n_pos], q_out if in_place else q, q_out)
    assert int(st.status) == 3
    assert torch.equal(got[fine], turned[fine]) and bool(got[~fine].isnan().all())
    # the pages: sequence 0's as they should be, sequence 1's with NaN from the first refused token on
    kk, vv = st.read(table[:2], i32(held[:2]), cu[:3], 2 * each)
    wk, wv = want.read(table[:2], i32(held[:2]), cu[:3], 2 * each)
    for a, b in ((kk, wk), (vv, wv)):
        assert torch.equal(a[fine[:2 * each]], b[fine[:2 * each]]) and bool(a[~fine[:2 * each]].isnan().all())
    # nothing else is touched: rows of sequence 1 outside its tokens, and the pages of 3 and 4
    rest = (torch.arange(P * 64, device=DEV) < held[1]) | (torch.arange(P * 64, device=DEV) >= held[1] + each)
    whole = torch.arange(2, dtype=torch.int32, device=DEV) * P * 64
    a, b = st.read(table[1:2], i32([0]), whole, P * 64), want.read(table[1:2], i32([0]), whole, P * 64)
    assert torch.equal(a[0][rest], b[0][rest]) and torch.equal(a[1][rest], b[1][rest])
    assert bool((st.pages[3 * P:] == 0x3C003C00).all())
    st.status.zero_()
    x = randn(g, 2, Hq, D, dtype=dtype)
    out = st.attend(x, table[:2], i32([held[0] + each, held[1] + each]), 0.1)
    assert torch.equal(out[0], want.attend(x, table[:2], i32([held[0] + each, held[1] + each]), 0.1)[0])
    assert bool(out[1].isnan().all())
    assert bool(st.attend(x, table[:2], i32([held[0] + each, n_pos]), 0.1).isfinite().all())


def off_grid(x):
    """The values of x [n, h, d] in memory that the kernels cannot read as it is, two ways: rows of an odd width, and a
    contiguous block that starts between 16-byte boundaries."""
    n, h, d = x.shape
    wide = torch.empty(n, h * d + 4, dtype=x.dtype, device=DEV)[:, :h * d].view(n, h, d)
    flat = torch.empty(4 + n * h * d, dtype=x.dtype, device=DEV)[4:].view(n, h, d)
    return [wide.copy_(x), flat.copy_(x)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N", [1, 2, 5])
def test_inputs_off_the_16_byte_grid(front, dtype, N):
    """Copied, as documented, for one row as for many."""
    g = torch.Generator().manual_seed(N)
    H, Hq, D = 2, 4, 64
    k, v, q = randn(g, N, H, D, dtype=dtype), randn(g, N, H, D, dtype=dtype), randn(g, N, Hq, D, dtype=dtype)
    table, lens, cu = torch.arange(N, dtype=torch.int32, device=DEV)[:, None], i32([3] * N), i32([0, N])
    cos, sin = angles(10, D // 2)
    stores = [paged.PagedStore(N, H, D, DEV, dtype) for _ in range(3)]
    for st in stores:
        st.pages.zero_()
    want = stores[0].append(k, v, table, lens, None, cos, sin, q)
    out = stores[0].attend(want, table, lens + 1, 0.1)
    prompt = ops.prompt_attention(q, k, v, cu, 0.1)
    for st, kk, vv, qq, ww in zip(stores[1:], off_grid(k), off_grid(v), off_grid(q), off_grid(want)):
        assert torch.equal(st.append(kk, vv, table, lens, None, cos, sin, qq), want)
        assert torch.equal(st.pages, stores[0].pages)
        assert torch.equal(st.attend(ww, table, lens + 1, 0.1), out)
        for a in ((qq, k, v), (q, kk, v), (q, k, vv), (qq, kk, vv)):
            assert torch.equal(ops.prompt_attention(*a, cu, 0.1), prompt)


def test_outputs_whose_rows_share_memory_are_refused(front):
    g = torch.Generator().manual_seed(2)
    S, H, Hq, D = 4, 2, 8, 64
    k, q = randn(g, S, H, D), randn(g, S, Hq, D)
    st = paged.PagedStore(S, H, D, DEV)
    table, lens, cu = i32([[0], [1], [2], [3]]), i32([1] * S), i32([0, S])
    st.append(k, k, table, i32([0] * S))
    memory = torch.full((4 * S * Hq * D,), 5.0, dtype=torch.float16, device=DEV)
    for size, stride in (((S, Hq, D), (8, D, 1)), ((S, Hq, D), (Hq * D - 8, D, 1)), ((S, Hq, D), (Hq * D, D - 8, 1)),
                         ((S, Hq, D), (0, D, 1))):
        out = memory.as_strided(size, stride)
        for call in (lambda: st.attend(q, table, lens, 0.1, out=out),
                     lambda: st.attend(q[:, None].expand(S, 2, Hq, D), table, lens, 0.1, out=out[:, None].expand(S, 2, Hq, D)),
                     lambda: st.append(k, k, table, lens, q=q, q_out=out),
                     lambda: ops.prompt_attention(q, k, k, cu, 0.1, out=out)):
            with pytest.raises(ValueError, match="rows"):
                call()
    for stride in ((8, D, 1), (H * D - 8, D, 1), (H * D, D - 8, 1), (H * D, 0, 1)):
        out = memory.as_strided((S, H, D), stride)
        for kw in (dict(k_out=out), dict(v_out=out)):
            with pytest.raises(ValueError, match="rows"):
                st.read(table, i32([0] * S), None, S, **kw)
    assert bool((memory == 5).all())
    out = memory.as_strided((S, Hq, D), (D, S * D, 1))  # heads outermost: rows of their own
    assert torch.equal(st.attend(q, table, lens, 0.1, out=out), st.attend(q, table, lens, 0.1))


def test_read_into_one_memory_is_refused():
    g = torch.Generator().manual_seed(3)
    st = paged.PagedStore(2, 2, 64, DEV)
    k, v = randn(g, 20, 2, 64), randn(g, 20, 2, 64)
    table, cu = i32([[0], [1]]), i32([0, 8, 20])
    st.append(k, v, table, i32([0, 0]), cu)
    wide = torch.full((20, 5, 64), 5.0, dtype=torch.float16, device=DEV)
    for a, b in ((wide[:, :2], wide[:, :2]), (wide[:, :2], wide[:, 1:3]), (wide[:, 1:3], wide[:, :2])):
        with pytest.raises(ValueError, match="share memory"):
            st.read(table, i32([0, 0]), cu, 20, k_out=a, v_out=b)
    assert bool((wide == 5).all())
    want = st.read(table, i32([0, 0]), cu, 20)
    got = st.read(table, i32([0, 0]), cu, 20, k_out=wide[:, 3:], v_out=wide[:, :2])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and bool((wide[:, 2] == 5).all())


def test_outputs_that_autograd_follows_are_refused(front):
    """A leaf, what was computed from one, a dual tensor; under no_grad the first two are memory as any other."""
    g = torch.Generator().manual_seed(4)
    S, H, Hq, D = 3, 2, 4, 64
    k, q = randn(g, S, H, D), randn(g, S, Hq, D)
    st = paged.PagedStore(S, H, D, DEV)
    table, lens, cu = i32([[0], [1], [2]]), i32([1] * S), i32([0, S])
    st.append(k, k, table, i32([0] * S))
    want, turned = st.attend(q, table, lens, 0.1), ops.prompt_attention(q, k, k, cu, 0.1)
    leaf = torch.full((S, Hq, D), 5.0, dtype=torch.float16, device=DEV, requires_grad=True)

    def calls(out):
        return [lambda: st.attend(q, table, lens, 0.1, out=out), lambda: ops.prompt_attention(q, k, k, cu, 0.1, out=out),
                lambda: st.append(k, k, table, lens, q=q, q_out=out), lambda: st.read(table, i32([0] * S), None, S, k_out=out[:, :H]),
                lambda: st.read(table, i32([0] * S), None, S, v_out=out[:, :H])]

    for out in (leaf, leaf * 1):
        for call in calls(out):
            with pytest.raises(NotImplementedError):
                call()
        assert bool((out == 5).all())
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(leaf.detach(), q)
        for call in calls(dual):
            with pytest.raises(NotImplementedError):
                call()
    assert bool((leaf == 5).all())
    with torch.no_grad():
        for out in (leaf, leaf * 1):
            assert torch.equal(calls(out)[0](), want) and torch.equal(calls(out)[1](), turned)


def test_check_keeps_what_is_told_while_it_reads(monkeypatch):
    """A call that meets a bad length after check() has taken the status word, and before check() returns, is told by the
    next check()."""
    g = torch.Generator().manual_seed(5)
    st = paged.PagedStore(2, 2, 64, DEV)
    k, table = randn(g, 2, 2, 64), i32([[0], [1]])
    st.append(k, k, i32([[9], [1]]), i32([0, 0]))
    item, other = torch.Tensor.item, torch.cuda.Stream()

    def late(t):
        word = item(t)
        monkeypatch.setattr(torch.Tensor, "item", item)
        with torch.cuda.stream(other):
            st.append(k, k, table, i32([-1, 0]))
        other.synchronize()
        return word

    monkeypatch.setattr(torch.Tensor, "item", late)
    with pytest.raises(RuntimeError, match="outside the pool$"):
        st.check()
    with pytest.raises(RuntimeError, match="met a token past"):
        st.check()
    st.check()


def test_strides_of_one_length_and_of_one_page(front):
    """A stride that is never used refuses nothing: the length of one sequence, a table of one page, taken from wider
    tensors."""
    g = torch.Generator().manual_seed(6)
    H, Hq, D = 2, 4, 64
    st = paged.PagedStore(3, H, D, DEV)
    for S in (1, 3):
        k, q = randn(g, S, H, D), randn(g, S, Hq, D)
        table, lens = i32([[0], [1], [2]])[:S], i32([2, 2, 2])[:S]
        odd_table = table.clone().as_strided((S, 1), (1, 7))
        odd_lens = i32([[2, 9]])[:, 0] if S == 1 else lens
        st.pages.zero_()
        want = st.append(k, k, table, lens, q=q), st.pages.clone(), st.attend(q, table, lens + 1, 0.1), *st.read(table, lens, None, S)
        st.pages.zero_()
        got = st.append(k, k, odd_table, odd_lens, q=q), st.pages, st.attend(q, odd_table, lens + 1, 0.1), *st.read(odd_table, odd_lens, None, S)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(ValueError, match="contiguous"):
        st.attend(q, i32([[0, 1, 2], [0, 1, 2]]).t()[:, :2], lens, 0.1)
    with pytest.raises(ValueError, match="contiguous"):
        st.attend(q, table, i32([[2, 9], [2, 9], [2, 9]])[:, 0], 0.1)


# ---- logits of minus infinity, and large finite ones -------------------------------------------------------------
def check_rows(out, q, k, v, ends, low, scale, window=0):
    """Row i of ``out`` [n, Hq, D] against attention in 64 bits over the keys below ends[i] (the last ``window`` of them)
    that are not ``low``: those have weights of exactly 0, and where all are, the row is 0."""
    got, low = out.cpu().double(), low.cpu()
    q, k, v = q.cpu(), k.cpu(), v.cpu()
    zeros = 0
    for i, end in enumerate(ends):
        keys = torch.arange(max(0, end - window) if window else 0, max(0, end))
        keys = keys[~low[keys]]
        if not len(keys):
            assert bool((got[i] == 0).all()), i
            zeros += 1
            continue
        want, bound = R.attention(q[i:i + 1], k[keys], v[keys], scale, causal=False)
        assert bool(((got[i] - want[0]).abs() <= bound[0]).all()), i
    return zeros


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window", [None, 3, 70])
def test_prompt_keys_of_minus_infinity(dtype, D, window):
    g = torch.Generator().manual_seed(D)
    n = 200
    q, k, v = randn(g, n, 2, D, dtype=dtype), randn(g, n, 1, D, dtype=dtype), randn(g, n, 1, D, dtype=dtype)
    q[..., 3] = q[..., 3].abs() + 0.5
    low = torch.zeros(n, dtype=torch.bool)
    low[:5] = low[40:50] = low[128:192] = True  # the first rows see nothing else; a whole tile of keys
    k[low.to(DEV), 0, 3] = float("-inf")
    out = ops.prompt_attention(q, k, v, i32([0, n]), 0.125, window=window)
    assert check_rows(out, q, k, v, range(1, n + 1), low, 0.125, window or 0) >= 5


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("width", [2, 30])
@pytest.mark.parametrize("window", [None, 2])
def test_attend_logits_that_overflow_to_minus_infinity(D, width, window):
    """(bf16: a page's finite keys and finite queries whose products pass fp32's range.)  Whole sequences and shares."""
    g = torch.Generator().manual_seed(D + width)
    lens, m, big = [5, 128, 70, 3], 3, 3e38
    N, starts = sum(lens), [0, 5, 133, 203]
    low = torch.zeros(N, dtype=torch.bool)
    low[:3] = low[5:15] = low[5 + 64:5 + 128] = low[203:206] = True  # (sequence 3: every key; 0: all that its first row sees)
    k, v = randn(g, N, 1, D, dtype=torch.bfloat16), randn(g, N, 1, D, dtype=torch.bfloat16)
    q = randn(g, 4, m, 2, D, dtype=torch.bfloat16)
    k[..., :32] = 0
    k[low.to(DEV), :, :32] = big
    q[..., :32] = -big
    st = paged.PagedStore(4 * width, 1, D, DEV, torch.bfloat16)
    table = torch.arange(4 * width, dtype=torch.int32, device=DEV).view(4, width)
    st.append(k, v, table, i32([0] * 4), i32(starts + [N]))
    kk, vv = st.read(table, i32([0] * 4), i32(starts + [N]), N)
    assert torch.equal(kk[..., :32], k[..., :32])
    out = st.attend(q, table, i32(lens), 0.125, window=window)
    zeros = 0
    for s, (a, n) in enumerate(zip(starts, lens)):
        zeros += check_rows(out[s], q[s], kk[a:a + n], vv[a:a + n], [n - 2, n - 1, n], low[a:a + n], 0.125, window or 0)
    assert zeros >= 4
    st.check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("width", [5, 30])
def test_attend_large_finite_logits(dtype, D, width):
    """Over pages that every row sees whole: one weight is 1, the rest 0."""
    g = torch.Generator().manual_seed(D + width)
    n, m, Hq = 300, 16, 4
    k, v = randn(g, n, 1, D, dtype=dtype) * 300, randn(g, n, 1, D, dtype=dtype)
    q = randn(g, 1, m, Hq, D, dtype=dtype) * 300
    st = paged.PagedStore(width, 1, D, DEV, dtype)
    table = torch.arange(width, dtype=torch.int32, device=DEV)[None]
    st.append(k, v, table, i32([0]), i32([0, n]))
    kk, vv = (x.cpu().double()[:, 0] for x in st.read(table, i32([0]), i32([0, n]), n))
    out = st.attend(q, table, i32([n]), 1.0).cpu()[0]
    assert bool(out.isfinite().all())
    seen = torch.arange(n)[None] < n - (m - 1) + torch.arange(m)[:, None]
    qq = q[0].cpu().double()
    s = torch.matmul(qq, kk.T).masked_fill(~seen[:, None], -1e300)
    size = torch.matmul(qq.abs(), kk.abs().T).amax(-1)
    top = s.topk(2, -1).values
    # a logit's sum of D products is off by at most (D + 8) 2^-24 of their absolute sum, on both sides; e^-100 is no weight
    sure = top[..., 0] - top[..., 1] > 100 + 2 * (D + 8) * 2.0 ** -24 * size
    assert int(sure.sum()) > 50
    assert torch.equal(out[sure].double(), vv[s.argmax(-1)[sure]])


def test_outputs_that_are_no_tensors_are_refused(front):
    st = paged.PagedStore(2, 2, 64, DEV)
    k, table, lens = torch.zeros(2, 2, 64, dtype=torch.float16, device=DEV), i32([[0], [1]]), i32([0, 0])
    for call in (lambda: st.append(k, k, table, lens, q=k, q_out=5), lambda: st.attend(k, table, lens, 1.0, out=[k]),
                 lambda: st.read(table, lens, None, 2, v_out=5), lambda: ops.prompt_attention(k, k, k, i32([0, 2]), 1.0, out=5)):
        with pytest.raises(TypeError):
            call()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_queries_of_nan_stay_in_their_rows(dtype, D, bad):
    """One head's query of one row: its output is NaN, the other rows' (of the same tiles) are right."""
    g = torch.Generator().manual_seed(D)
    Hq, n, m = 4, 150, 5
    k, v = randn(g, n, 1, D, dtype=dtype), randn(g, n, 1, D, dtype=dtype)
    q = randn(g, n, Hq, D, dtype=dtype)
    q[3, 1, 0] = q[100, 2, D - 1] = bad
    for causal, window in ((True, None), (True, 20), (False, None)):
        out = ops.prompt_attention(q, k, v, i32([0, n]), 0.1, causal=causal, window=window).cpu().double()
        want, bound = R.attention(q.cpu(), k.cpu(), v.cpu(), 0.1, causal, window or 0)
        assert torch.equal(out.isnan().all(-1).nonzero(), torch.tensor([[3, 1], [100, 2]]))
        fine = ~out.isnan()
        assert int((~fine).sum()) == 2 * D and bool(((out - want).abs() <= bound)[fine].all())
    for width in (3, 30):
        st = paged.PagedStore(width, 1, D, DEV, dtype)
        st.pages.fill_(-1)
        table = torch.arange(width, dtype=torch.int32, device=DEV)[None]
        st.append(k, v, table, i32([0]), i32([0, n]))
        kk, vv = (x.cpu() for x in st.read(table, i32([0]), i32([0, n]), n))
        out = st.attend(q[None, :m], table, i32([n]), 0.1).cpu().double()[0]
        want, bound = R.attention(q[:m].cpu(), kk, vv, 0.1)
        assert torch.equal(out.isnan().all(-1).nonzero(), torch.tensor([[3, 1]]))
        fine = ~out.isnan()
        assert int((~fine).sum()) == D and bool(((out - want).abs() <= bound)[fine].all())
