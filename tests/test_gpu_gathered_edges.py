"""Edges of gathered attention weights on the GPU: what may and may not change where rows are NaN, or only some keys
count."""
import random

import pytest
import torch

from innerq_amd import ops, paged
from oracle import evict_ref as E

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def filled(seed, lens, H, D, dtype, width):
    """A store whose sequences hold random tokens, and its table."""
    g, rng = torch.Generator().manual_seed(seed), random.Random(seed)
    pool = len(lens) * width
    table = i32(rng.sample(range(pool), pool)).view(len(lens), width)
    st = paged.PagedStore(pool, H, D, DEV, dtype)
    st.pages.zero_()
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    k, v = (torch.randn(cu[-1], H, D, generator=g).to(dtype).to(DEV) for _ in range(2))
    st.append(k, v, table, i32([0] * len(lens)), i32(cu))
    return st, table, g


@pytest.mark.parametrize("maps", [1, 2])
@pytest.mark.parametrize("D,dtype", [(64, torch.float16), (128, torch.bfloat16)])
@pytest.mark.parametrize("width", [8, 40])  # a workgroup takes a whole sequence and head; workgroups share them
@pytest.mark.parametrize("window", [1, 30, 100, 300])
def test_rows_of_nan_leave_tokens_before_the_window(maps, D, dtype, width, window):
    """A window that begins inside a page: the page's tokens before it gather nothing, from a row of NaN too."""
    lens = [200, 500, 130, 64]
    st, table, g = filled(window, lens, 2, D, dtype, width)
    q = torch.randn(4, 8, D, generator=g).to(dtype).to(DEV)
    lam = torch.full((4,), 0.5, device=DEV)
    clean = torch.randn(4, 2, width * 64 + 5, generator=g).to(DEV)

    def weights(q, table, lens):
        w = clean.clone()
        if maps == 1:
            out = st.attend(q, table, i32(lens), 0.1, window=window, weights=w)
        else:
            out = st.diff_attend(q, table, i32(lens), lam, 0.1, window=window, weights=w)
        return out, w

    def check(w, s, heads, n):
        low = max(n - window, 0)
        for h in heads:
            assert bool(w[s, h, low:n].isnan().all()), (s, h)
            assert torch.equal(w[s, h, :low], clean[s, h, :low]) and torch.equal(w[s, h, n:], clean[s, h, n:]), (s, h)

    plain = weights(q, table, lens)[1]
    st.check()
    for s, n in enumerate(lens):
        low = max(n - window, 0)
        assert torch.equal(plain[s, :, :low], clean[s, :, :low]) and torch.equal(plain[s, :, n:], clean[s, :, n:])
    bad = q.clone()
    bad[1, 0, 3] = float("nan")  # a query of KV head 0
    bad[2] = float("inf")        # logits of infinity less infinity, in every head
    out, w = weights(bad, table, lens)
    assert bool(out[1, 0].isnan().all()) and bool(out[2].isnan().all())
    check(w, 1, [0], 500)
    check(w, 2, [0, 1], 130)
    assert torch.equal(w[1, 1], plain[1, 1]) and torch.equal(w[0], plain[0]) and torch.equal(w[3], plain[3])
    # a page outside the pool, and a sequence longer than its table, whose tokens are the table's then
    bad_table = table.clone()
    bad_table[1, 499 // 64] = 10 ** 6
    out, w = weights(q, bad_table, [200, 500, width * 64 + 9, 64])
    with pytest.raises(RuntimeError, match="outside the pool and a token past"):
        st.check()
    assert bool(out[1:3].isnan().all())
    check(w, 1, [0, 1], 500)
    check(w, 2, [0, 1], width * 64)
    assert torch.equal(w[0], plain[0]) and torch.equal(w[3], plain[3])


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("D,H,Hq,dtype", [(64, 1, 2, torch.float16), (128, 2, 8, torch.bfloat16)])
def test_values_behind_logits_of_minus_infinity(value, D, H, Hq, dtype):
    """An infinity or NaN in V of a key whose logits are minus infinity (0 times it) reaches the rows that see it, whether
    or not a workgroup has only such keys: as in the call without weights."""
    g = torch.Generator().manual_seed(3)
    lens, keys = [6, 9], [4000, 3500]
    cu, cu_k = i32([0, 6, 15]), i32([0, 4000, 7500])
    q, k = torch.ones(15, Hq, D), torch.randn(7500, H, D, generator=g)
    v = torch.randn(7500, H, D, generator=g)
    q, k, v = (x.to(dtype).to(DEV) for x in (q, k, v))
    k[:3900, :, 0] = float("-inf")      # of sequence 0 the last 100 keys count, of sequence 1 all
    v[700, 0, 5] = value
    v[3990, 0, 9] = value               # a key that counts
    v[3997, 0, 11] = value              # that the first rows do not see
    want = ops.prompt_attention(q, k, v, cu, 0.1, cu_k)
    w = torch.zeros(2, H, 4000, device=DEV)
    out = ops.prompt_attention(q, k, v, cu, 0.1, cu_k, weights=w)
    assert bool(w.isfinite().all()) and bool((w[0, :, :3900] == 0).all())
    r = Hq // H
    hit = torch.zeros_like(out, dtype=torch.bool)
    hit[:6, :r, 5] = hit[:6, :r, 9] = hit[3:6, :r, 11] = True
    assert not bool(want[hit].isfinite().any()) and bool(want[~hit].isfinite().all())
    assert not bool(out[hit].isfinite().any()) and bool(out[~hit].isfinite().all())
    assert torch.equal(out.isnan(), want.isnan())


@pytest.mark.parametrize("value", [float("inf"), float("nan")])
@pytest.mark.parametrize("D,H,Hq,dtype", [(64, 2, 2, torch.float16), (128, 2, 8, torch.bfloat16)])
@pytest.mark.parametrize("past", [0, 4000])  # rows in one workgroup, and shared out
def test_rows_without_a_key_that_counts(value, D, H, Hq, dtype, past):
    """Rows that see only keys whose logits are minus infinity are 0, whatever V holds there; so is such a map of
    differential attention, with the other one as it is."""
    g = torch.Generator().manual_seed(6)
    rows, n = 90, 90 + past
    cu, cu_k = i32([0, rows]), i32([0, n])
    q, k = torch.ones(rows, Hq, D), torch.randn(n, H, D, generator=g)
    v = torch.randn(n, H, D, generator=g)
    k[:, 0, 0] = float("-inf")  # of KV head 0, the first map's
    v[n - 80, 0, 5] = v[n // 2, 0, 9] = value
    q, k, v = (x.to(dtype).to(DEV) for x in (q, k, v))
    r = Hq // H
    for kw in (dict(), dict(causal=False)):
        for w in (None, torch.zeros(1, H, n, device=DEV)):
            out = ops.prompt_attention(q, k, v, cu, 0.1, cu_k, weights=w, **kw)
            assert bool((out[:, :r] == 0).all()) and bool(out[:, r:].isfinite().all()), (kw, w is None)
            assert w is None or bool((w[0, 0] == 0).all())
    fine = v.clone()
    fine[:, 0] = 0
    lam, vv = torch.full((Hq // 2,), 0.5, device=DEV), fine.reshape(n, 1, 2 * D)
    second = -0.5 * ops.prompt_attention(q[:, 1::2], k[:, 1:], fine[:, 1:], cu, 0.1, cu_k).float()
    out = ops.diff_prompt_attention(q, k, vv, cu, lam, 0.1, cu_k)
    # each call rounds every weight (by u relatively; fp16's small ones by 2^-25) and its result once
    u, most = torch.finfo(dtype).eps / 2, float(fine.abs().max())
    near = 2 * 0.5 * (u + n * 2.0 ** -25) * most + 2 * u * second.abs() + 2.0 ** -24
    assert bool((out[..., :D] == 0).all()) and bool(((out[..., D:].float() - second).abs() <= 1.01 * near).all())
    kk = k.clone()
    kk[:, 1, 0], kk[:, 1, 1] = 0, float("-inf")  # no map has a key that counts
    out = ops.diff_prompt_attention(q, kk, v.reshape(n, 1, 2 * D), cu, lam, 0.1, cu_k)
    assert bool((out == 0).all())


@pytest.mark.parametrize("native", [True, False])
def test_strides_of_one_length(native, monkeypatch):
    """The stride of a dim of length 1 says nothing: weights of one token, one sequence or one head of any such stride."""
    if not native:
        monkeypatch.setattr(ops, "_native", lambda t: None)
    g = torch.Generator().manual_seed(4)
    q, k, v = (torch.randn(2, 2, 64, generator=g).half().to(DEV) for _ in range(3))
    cu = i32([0, 1, 2])
    a, b = torch.zeros(2, 2, 1, device=DEV), torch.zeros(2, 2, 7, device=DEV)[..., ::7]
    assert b.shape == (2, 2, 1) and b.stride(2) == 7
    assert torch.equal(ops.prompt_attention(q, k, v, cu, 0.1, weights=a), ops.prompt_attention(q, k, v, cu, 0.1, weights=b))
    assert torch.equal(a, b) and bool((a == 1).all())
    a, b = torch.zeros(2, 2, 1, device=DEV), torch.zeros(2, 2, 7, device=DEV)[..., ::7]
    lam, vv = torch.ones(1, device=DEV), v.reshape(2, 1, 128)
    ops.diff_prompt_attention(q, k, vv, cu, lam, 0.1, weights=a)
    ops.diff_prompt_attention(q, k, vv, cu, lam, 0.1, weights=b)
    assert torch.equal(a, b) and bool((a == 1).all())
    # evict in place through another view of the same memory
    for S, H in ((1, 1), (1, 2), (2, 1)):
        st, table, g = filled(5, [100] * S, H, 64, torch.float16, 2)
        w = torch.rand(S, H, 128, generator=g).to(DEV)
        want = st.evict(table, i32([100] * S), w.clone(), 60, recent=7)[1]
        for place in range(2):  # (strides of the dims of length 1 that no walk over them takes)
            x = w.clone()
            view = x.as_strided(x.shape, (x.stride(0) if S > 1 else 640, x.stride(1) if H > 1 else 1280, 1))
            st2, table2, _ = filled(5, [100] * S, H, 64, torch.float16, 2)
            new, out = st2.evict(table2, i32([100] * S), *((x, 60) if place else (view, 60)), recent=7,
                                 out=view if place else x)
            assert torch.equal(x, want) and new.tolist() == [60] * S


def gathered_check(st, table, lens, q, w, before, scale, maps, window=0):
    """w = before + what the stores' keys gather, within the bound that rounded weights would break."""
    for s, n in enumerate(lens):
        assert torch.equal(w[s, :, n:], before[s, :, n:]), s
        if not n:
            continue
        k = st.read(table[s:s + 1], i32([0]), i32([0, n]), n)[0]
        for i in range(maps):
            want, bound = E.gathered(q[s:s + 1, i::maps], k[:, i::maps], scale, window=window)
            old = before[s, i::maps, :n].double()
            worst = ((w[s, i::maps, :n].double() - old - want).abs() - bound - 2.0 ** -24 * (old + want)).amax()
            assert worst <= 0, (s, i, float(worst))


@pytest.mark.parametrize("maps", [1, 2])
@pytest.mark.parametrize("D,dtype", [(64, torch.float16), (128, torch.bfloat16), (128, torch.float16)])
@pytest.mark.parametrize("lens,Hq", [([6000, 700, 1], 2), ([6000, 700, 1], 36), ([400, 500, 0], 8), ([20000], 8)])
@pytest.mark.parametrize("window", [None, 777])
def test_a_steps_weights_are_not_rounded(maps, D, dtype, lens, Hq, window):
    st, table, g = filled(D, lens, 2, D, dtype, -(-max(lens) // 64))
    q = torch.randn(len(lens), Hq, D, generator=g).to(dtype).to(DEV)
    lam = torch.full((Hq // 2,), 0.5, device=DEV)
    w = torch.zeros(len(lens), 2, table.shape[1] * 64, device=DEV)
    for _ in range(2):  # from nothing, and on top of that
        before = w.clone()
        if maps == 1:
            st.attend(q, table, i32(lens), D ** -0.5, window=window, weights=w)
        else:
            st.diff_attend(q, table, i32(lens), lam, D ** -0.5, window=window, weights=w)
        gathered_check(st, table, lens, q, w, before, D ** -0.5, maps, window or 0)
    st.check()


@pytest.mark.parametrize("maps", [1, 2])
@pytest.mark.parametrize("width", [8, 40])
def test_captured_steps(maps, width):
    """A captured step follows its lengths and table: every replay gives what the eager call gives, all of it finite."""
    most = width * 64
    st, table, g = filled(9, [most, most, most], 2, 64, torch.float16, width)
    ll, lam = i32([most, 30, 400]), torch.full((4,), 0.5, device=DEV)
    q = torch.randn(3, 8, 64, generator=g).half().to(DEV)
    clean = torch.rand(3, 2, most, generator=g).to(DEV)
    w = clean.clone()

    def call(w):
        return st.attend(q, table, ll, 0.1, weights=w) if maps == 1 else st.diff_attend(q, table, ll, lam, 0.1, weights=w)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(w)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        o = call(w)
    for n in ([most, 30, 400], [5, most, 0], [64, 1, 65], [0, 0, 0], [400, most, 30]):
        ll.copy_(i32(n))
        table.copy_(table.flip(0))
        w.copy_(clean)
        graph.replay()
        torch.cuda.synchronize()
        x = clean.clone()
        y = call(x)
        assert bool(y.isfinite().all()) and torch.equal(o, y) and torch.equal(w, x), n
        gathered_check(st, table, n, q, w, clean, 0.1, maps)
