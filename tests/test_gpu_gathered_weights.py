"""The attention weights that keys gather (attend(weights=), prompt_attention(weights=)) on the GPU against 64 bits
(oracle/evict_ref.py); the output is that of the call without them."""
import random

import pytest
import torch

from innerq_amd import ops, paged
from oracle import evict_ref as E
from oracle import serving_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float16, torch.bfloat16]


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def filled(seed, lens, H, D, dtype, width=None):
    """A store whose sequences hold random tokens (NaN behind their ends), and K as the store holds it."""
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
    k = torch.randn(max(N, 1), H, D, generator=g)
    k[..., :3] *= 6
    v = torch.randn(max(N, 1), H, D, generator=g)
    if N:
        st.append(k.to(dtype).to(DEV), v.to(dtype).to(DEV), table, i32([0] * len(lens)), i32(cu))
        k = st.read(table, i32([0] * len(lens)), i32(cu), N)[0].cpu()
    return st, table, cu, k, g


def held(g, S, H, T):
    """What the keys have gathered before: NaN nowhere, marks behind the ends."""
    return torch.rand(S, H, T, generator=g).to(DEV)


def check(got, before, want, bound, what):
    """got = before + want, the sum rounded once."""
    b = before.double()
    worst = ((got.double() - b - want).abs() - bound - 2.0 ** -24 * (b + want).abs()).max()
    assert worst <= 0, (what, float(worst))


def check_attend(st, table, cu, k, lens, q, w, scale, window=None):
    before = w.cpu().clone()
    want_out = st.attend(q, table, i32(lens), scale, window=window)
    out = st.attend(q, table, i32(lens), scale, window=window, weights=w)
    st.check()
    assert torch.equal(out, want_out)
    got = w.cpu()
    for s, n in enumerate(lens):
        assert torch.equal(got[s, :, n:], before[s, :, n:]), s
        if n:
            want, bound = E.weights(q[s].cpu().view(1, -1, st.D), k[cu[s]:cu[s + 1]], scale, window=window or 0)
            check(got[s, :, :n], before[s, :, :n], want, bound, s)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,H,Hq", [(128, 2, 8), (64, 2, 2), (128, 1, 3), (64, 1, 32), (128, 3, 3), (64, 1, 40)])
@pytest.mark.parametrize("lens", [[1], [2, 63, 64, 65], [0, 5, 0, 300], [1000, 17, 128, 511], [700, 1, 2100]])
def test_attend_lengths(dtype, D, H, Hq, lens):
    st, table, cu, k, g = filled(sum(lens) + H, lens, H, D, dtype)
    w = held(g, len(lens), H, table.shape[1] * 64)
    q = torch.randn(len(lens), Hq, D, generator=g).to(dtype).to(DEV)
    check_attend(st, table, cu, k, lens, q, w, D ** -0.5)
    check_attend(st, table, cu, k, lens, q, w, D ** -0.5)  # on top of the first


@pytest.mark.parametrize("window", [1, 50, 64, 65, 700, 2 ** 31 - 1])
@pytest.mark.parametrize("width", [None, 60])
def test_attend_windows(window, width):
    lens = [1, 64, 65, 900, 0, 129]
    st, table, cu, k, g = filled(3, lens, 2, 128, torch.float16, width)
    w = held(g, 6, 2, table.shape[1] * 64 + 3)
    q = torch.randn(6, 4, 128, generator=g).half().to(DEV)
    check_attend(st, table, cu, k, lens, q, w, 0.1, window)


@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0])
def test_attend_scales(scale):
    lens = [300, 1, 64, 1200]
    st, table, cu, k, g = filled(4, lens, 2, 64, torch.bfloat16)
    w = held(g, 4, 2, table.shape[1] * 64)
    q = torch.randn(4, 4, 64, generator=g).bfloat16().to(DEV)
    check_attend(st, table, cu, k, lens, q, w, scale)


@pytest.mark.parametrize("S,H,width", [(2, 1, 8), (2, 1, 9), (16, 4, 17), (64, 4, 32), (64, 4, 33), (300, 1, 40)])
def test_attend_table_widths(S, H, width):
    """Both sides of the widths up to which a workgroup takes a whole sequence and head."""
    rng = random.Random(S)
    lens = [rng.choice([0, 1, 64, 130]) for _ in range(S)]
    lens[0], lens[S - 1] = width * 64, 200
    st, table, cu, k, g = filled(width, lens, H, 64, torch.float16, width)
    w = held(g, S, H, width * 64)
    q = torch.randn(S, 2 * H, 64, generator=g).half().to(DEV)
    check_attend(st, table, cu, k, lens, q, w, 0.125)


def test_attend_two_groups_of_rows():
    """More than 16 query heads per KV head, over enough pages for two groups of rows at a time."""
    lens = [40, 600, 0] + [64] * 125
    st, table, cu, k, g = filled(5, lens, 4, 64, torch.float16, 10)
    w = held(g, 128, 4, 640)
    q = torch.randn(128, 4 * 20, 64, generator=g).half().to(DEV)
    check_attend(st, table, cu, k, lens, q, w, 0.125)


@pytest.mark.parametrize("width", [8, 40])
def test_attend_special_rows(width):
    """Infinite and NaN queries, keys and pages: NaN stays with its sequence and head, and within the tokens it saw."""
    lens = [200, 100, 130, 64]
    st, table, cu, k, g = filled(6, lens, 2, 64, torch.float16, width)
    q = torch.randn(4, 4, 64, generator=g).half().to(DEV)
    clean = held(g, 4, 2, width * 64)
    want = clean.clone()
    st.attend(q, table, i32(lens), 0.1, weights=want)
    w = clean.clone()
    bad = q.clone()
    bad[0, 0, 3] = float("nan")  # of KV head 0
    st.attend(bad, table, i32(lens), 0.1, weights=w)
    assert bool(w[0, 0, :200].isnan().all()) and torch.equal(w[0, 1], want[0, 1]) and torch.equal(w[1:], want[1:])
    assert torch.equal(w[0, 0, 200:], clean[0, 0, 200:])
    # a page outside the pool, and a sequence longer than its table
    w = clean.clone()
    bad_table = table.clone()
    bad_table[1, 0] = 10 ** 6
    st.attend(q, bad_table, i32([200, 100, width * 64 + 1, 64]), 0.1, weights=w)
    with pytest.raises(RuntimeError, match="outside the pool and a token past"):
        st.check()
    assert bool(w[1, :, :100].isnan().all()) and torch.equal(w[1, :, 100:], clean[1, :, 100:])
    assert bool(w[2].isnan().all()) and torch.equal(w[0], want[0]) and torch.equal(w[3], want[3])
    # all logits minus infinity: a row of 0, and no weights
    keys = torch.full((64, 2, 64), -1.0)
    keys[..., 0] = float("-inf")
    one = paged.PagedStore(1, 2, 64, DEV)
    one.pages.zero_()
    half = one.pages.view(torch.int16)  # K: code 0 with zero point -inf in group 0
    half[:, :, 2 * 64 * 8 + 1:2 * 64 * 8 + 2 * 64 * 2:4] = torch.tensor([-1024], dtype=torch.int16, device=DEV)
    x = torch.zeros(1, 2, 64, dtype=torch.float16, device=DEV)
    x[..., :32] = 1.0
    w = clean[:1, :, :64].clone()
    out = one.attend(x, i32([[0]]), i32([50]), 1.0, weights=w)
    assert bool((out == 0).all()) and torch.equal(w, clean[:1, :, :64])


def test_attend_strides_streams_and_graphs():
    lens = [700, 30, 400]
    st, table, cu, k, g = filled(7, lens, 2, 128, torch.bfloat16, 40)
    ll = i32(lens)
    q = torch.randn(3, 4, 128, generator=g).bfloat16().to(DEV)
    clean = held(g, 3, 2, 2560)
    want = clean.clone()
    out = st.attend(q, table, ll, 0.1, weights=want)
    wide = torch.zeros(2, 3, 2601, device=DEV).transpose(0, 1)
    w = wide[..., 41:]
    w.copy_(clean)
    assert torch.equal(st.attend(q[:, None], table, ll, 0.1, weights=w)[:, 0], out) and torch.equal(w, want)
    assert not wide[..., :41].any()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    w = clean.clone()
    with torch.cuda.stream(side):
        st.attend(q, table, ll, 0.1, weights=w)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        o = st.attend(q, table, ll, 0.1, weights=w)
    for n in ([700, 30, 400], [5, 2560, 0]):
        ll.copy_(i32(n))
        table.clamp_(min=0)
        w.copy_(clean)
        graph.replay()
        torch.cuda.synchronize()
        x = clean.clone()
        y = st.attend(q, table, ll, 0.1, weights=x)
        assert torch.equal(o, y) or bool(y.isnan().any())
        assert torch.equal(w.nan_to_num(7.0), x.nan_to_num(7.0))


def test_attend_refusals():
    lens = [100, 30]
    st, table, cu, k, g = filled(8, lens, 2, 64, torch.float16)
    q = torch.randn(2, 4, 64, generator=g).half().to(DEV)
    w = held(g, 2, 2, 128)
    with pytest.raises(ValueError, match="one new token"):
        st.attend(q[:, None].expand(2, 2, 4, 64), table, i32(lens), 0.1, weights=w)
    for bad in (w[:1], w[:, :1], w[..., :127], w.transpose(1, 2), w[0], w[:1].expand(2, 2, 128), w[:, :1].expand(2, 2, 128)):
        with pytest.raises(ValueError):
            st.attend(q, table, i32(lens), 0.1, weights=bad)
    for bad in (w.half(), w.cpu()):
        with pytest.raises(TypeError):
            st.attend(q, table, i32(lens), 0.1, weights=bad)
    with pytest.raises(NotImplementedError):
        st.attend(q, table, i32(lens), 0.1, weights=w.clone().requires_grad_())


# ---- prompts ---------------------------------------------------------------------------------------------------
def prompts(seed, lens, past, H, Hq, D, dtype):
    g = torch.Generator().manual_seed(seed)
    past = past if isinstance(past, list) else [past] * len(lens)
    N, Nk = sum(lens), sum(max(a + b, 0) for a, b in zip(lens, past))
    q, k, v = torch.randn(N, Hq, D, generator=g), torch.randn(Nk, H, D, generator=g), torch.randn(Nk, H, D, generator=g)
    k[..., :3] *= 4
    cu, cu_k = [0], [0]
    for a, b in zip(lens, past):
        cu.append(cu[-1] + a)
        cu_k.append(cu_k[-1] + max(a + b, 0))
    return g, *(x.to(dtype).to(DEV) for x in (q, k, v)), cu, cu_k


def check_prompts(g, q, k, v, cu, cu_k, scale, T=None, **kw):
    S, H = len(cu) - 1, k.shape[1]
    longest = max(b - a for a, b in zip(cu_k, cu_k[1:]))
    T = longest + 3 if T is None else T
    w = held(g, S, H, T)
    before = w.cpu().clone()
    want_out = ops.prompt_attention(q, k, v, i32(cu), scale, i32(cu_k), **kw)
    out = ops.prompt_attention(q, k, v, i32(cu), scale, i32(cu_k), weights=w, **kw)
    got, qc, kc, vc = w.cpu(), q.cpu(), k.cpu(), v.cpu()
    same = torch.equal(out, want_out)  # unless few rows over many keys are shared out: other sums, each within the bound
    for s in range(S):
        if not same:
            want, bound = R.attention(qc[cu[s]:cu[s + 1]], kc[cu_k[s]:cu_k[s + 1]], vc[cu_k[s]:cu_k[s + 1]], scale,
                                      kw.get("causal", True), kw.get("window") or 0)
            assert ((out[cu[s]:cu[s + 1]].cpu().double() - want).abs() - bound).max() <= 0, s
        n = min(cu_k[s + 1] - cu_k[s], T)
        assert torch.equal(got[s, :, n:], before[s, :, n:]), s
        if n and cu[s + 1] > cu[s]:
            want, bound = E.weights(qc[cu[s]:cu[s + 1]], kc[cu_k[s]:cu_k[s + 1]], scale, kw.get("causal", True),
                                    kw.get("window") or 0)
            check(got[s, :, :n], before[s, :, :n], want[:, :n], bound[:, :n], s)
        else:
            assert torch.equal(got[s], before[s])
    return w


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,H,Hq", [(128, 2, 8), (64, 2, 2), (128, 1, 3), (64, 1, 5)])
@pytest.mark.parametrize("lens", [[1], [63, 0, 64, 65, 1], [300, 17], [128, 129, 127]])
@pytest.mark.parametrize("past", [0, 1, 200])
def test_prompt_lengths(dtype, D, H, Hq, lens, past):
    check_prompts(*prompts(sum(lens) + past, lens, past, H, Hq, D, dtype), D ** -0.5)


@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 130, 400, 2 ** 31 - 1])
@pytest.mark.parametrize("past", [0, 150])
@pytest.mark.parametrize("Hq", [2, 6])
def test_prompt_windows(window, past, Hq):
    check_prompts(*prompts(window % 1000, [200, 1, 90, 257], past, 2, Hq, 64, torch.float16), 0.125, window=window)


@pytest.mark.parametrize("past", [[0, 70, -20], [-39, 300, -89], [5, 0, 0]])
@pytest.mark.parametrize("causal", [True, False])
def test_prompt_fewer_and_more_keys(past, causal):
    """More rows than keys (the first see none), more keys than rows, and every row all keys."""
    check_prompts(*prompts(9, [40, 100, 90], past, 2, 4, 128, torch.bfloat16), 0.09, causal=causal)


@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0, 50.0])
@pytest.mark.parametrize("dtype", DTYPES)
def test_prompt_scales(scale, dtype):
    check_prompts(*prompts(10, [150, 40], 0, 2, 4, 64, dtype), scale)


@pytest.mark.parametrize("T", [0, 1, 100, 128, 129, 200])
def test_prompt_keys_past_the_weights(T):
    check_prompts(*prompts(11, [260, 40], 0, 1, 2, 64, torch.float16), 0.125, T=T)


def test_prompt_many_sequences():
    rng = random.Random(12)
    lens = [rng.choice([0, 0, 1, 3, 40]) for _ in range(400)]
    lens[7] = 300
    check_prompts(*prompts(12, lens, [rng.choice([0, 0, 5, 130]) for _ in lens], 1, 2, 64, torch.float16), 0.125)


def test_prompt_long():
    check_prompts(*prompts(13, [1500], 700, 2, 4, 128, torch.bfloat16), 0.09)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,H,Hq", [(128, 2, 8), (64, 1, 3)])
@pytest.mark.parametrize("kw", [dict(), dict(causal=False), dict(window=700), dict(window=1), dict(window=3000)])
def test_prompt_few_rows_many_keys(dtype, D, H, Hq, kw):
    """Several workgroups share a tile of rows, some without a key; their sums are merged."""
    lens, past = [5, 40, 1, 33], [2500, 1100, 0, 6000]
    g, q, k, v, cu, cu_k = prompts(17, lens, past, H, Hq, D, dtype)
    k[cu_k[1] + 3] *= 3
    w = held(g, 4, H, 6033)
    before = w.cpu().clone()
    out = ops.prompt_attention(q, k, v, i32(cu), D ** -0.5, i32(cu_k), weights=w, **kw).cpu().double()
    q, k, v, got = q.cpu(), k.cpu(), v.cpu(), w.cpu()
    for s in range(4):
        r, j, n = slice(cu[s], cu[s + 1]), slice(cu_k[s], cu_k[s + 1]), cu_k[s + 1] - cu_k[s]
        want, bound = R.attention(q[r], k[j], v[j], D ** -0.5, kw.get("causal", True), kw.get("window") or 0)
        assert ((out[r] - want).abs() - bound).max() <= 0, s
        want, bound = E.weights(q[r], k[j], D ** -0.5, kw.get("causal", True), kw.get("window") or 0)
        check(got[s, :, :n], before[s, :, :n], want, bound, s)
        assert torch.equal(got[s, :, n:], before[s, :, n:])


def test_prompt_few_rows_special():
    """Rows of NaN, and rows whose only keys that count lie in one workgroup's share, or in none."""
    g, q, k, v, cu, cu_k = prompts(18, [20, 9], [4000, 3000], 1, 2, 64, torch.float16)
    x = torch.ones_like(q)
    x[7, 1] = float("nan")
    y = torch.zeros_like(k)
    y[:, 0, 0] = float("-inf")
    y[2000, 0, 0] = y[2001, 0, 0] = 0  # of sequence 0; sequence 1 has none
    w = held(g, 2, 1, 4100)
    before = w.clone()
    out = ops.prompt_attention(x, y, v, i32(cu), 0.1, i32(cu_k), weights=w)
    assert bool(out[7, 1].isnan().all()) and bool((out[20:] == 0).all())
    mean = (v[2000].float() + v[2001].float()) / 2
    rows = [i for i in range(20) if i != 7]
    assert bool(((out[rows].float() - mean).abs() <= 2.0 ** -10 * mean.abs() + 2.0 ** -24).all())
    assert bool(w[0, 0, :4008].isnan().all()) and torch.equal(w[1], before[1])
    x[7, 1] = 1.0
    w = before.clone()
    ops.prompt_attention(x, y, v, i32(cu), 0.1, i32(cu_k), weights=w)
    add = (w - before)[0, 0]
    assert abs(float(add[2000]) - 20) < 1e-5 and abs(float(add[2001]) - 20) < 1e-5
    add[2000:2002] = 0
    assert bool((add == 0).all())


def test_prompt_special_rows():
    """NaN stays with the keys that its row and head see; rows of minus infinity give nothing."""
    g, q, k, v, cu, cu_k = prompts(14, [200, 100], 0, 2, 4, 64, torch.float16)
    clean = held(g, 2, 2, 200)
    want = clean.clone()
    ops.prompt_attention(q, k, v, i32(cu), 0.1, weights=want)
    bad = q.clone()
    bad[150, 0, 3] = float("nan")  # of KV head 0, sees keys 0 .. 150
    w = clean.clone()
    ops.prompt_attention(bad, k, v, i32(cu), 0.1, weights=w)
    assert bool(w[0, 0, :151].isnan().all()) and torch.equal(w[0, 0, 151:], want[0, 0, 151:])
    assert torch.equal(w[0, 1], want[0, 1]) and torch.equal(w[1], want[1])
    bad = k.clone()
    bad[120, 1, 3] = float("nan")  # rows from 120 on are NaN for KV head 1, and with them all keys they see
    w = clean.clone()
    ops.prompt_attention(q, bad, v, i32(cu), 0.1, weights=w)
    assert bool(w[0, 1].isnan().all()) and torch.equal(w[0, 0], want[0, 0]) and torch.equal(w[1], want[1])
    x = torch.ones_like(q)
    bad = k.clone()
    bad[:200, 0] = 0
    bad[:200, 0, 0] = float("-inf")
    bad[100, 0] = 0  # the only key that counts
    w = clean.clone()
    out = ops.prompt_attention(x, bad, v, i32(cu), 0.1, weights=w)
    got = w[0, 0] - clean[0, 0]
    assert torch.equal(out[:100, :2], torch.zeros_like(out[:100, :2])) and bool((got[:100] == 0).all())
    assert bool((got[101:] == 0).all()) and abs(float(got[100]) - 200) < 1e-3
    w = clean.clone()
    ops.prompt_attention(q * 1e4, k, v, i32(cu), 1e3, weights=w)  # logits past 65536, no infinity of their own
    assert bool(w.isfinite().all())
    assert abs(float((w - clean)[0].double().sum()) - 200 * 4) < 1.0


def test_prompt_strides_and_graphs():
    g, q, k, v, cu, cu_k = prompts(15, [300, 40, 7], 0, 2, 4, 128, torch.bfloat16)
    clean = held(g, 3, 2, 300)
    want = clean.clone()
    ops.prompt_attention(q, k, v, i32(cu), 0.1, weights=want)
    wide = torch.zeros(347 + 40, 13, 128, dtype=q.dtype, device=DEV)
    wide[:347, 1:5], wide[:347, 5:7] = q, k
    w = clean.transpose(0, 1).contiguous().transpose(0, 1)
    qt = q.transpose(0, 1).contiguous().transpose(0, 1)
    for qq in (wide[:347, 1:5], qt, torch.cat([q, q], 2)[..., 128:]):
        x = w.clone()
        ops.prompt_attention(qq, wide[:347, 5:7], v, i32(cu), 0.1, weights=x)
        assert torch.equal(x, want)
    ints, w = i32(cu), clean.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.prompt_attention(q, k, v, ints, 0.1, weights=w)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        ops.prompt_attention(q, k, v, ints, 0.1, weights=w)
    for c in (cu, [0, 0, 300, 347], [40, 41, 60, 300]):
        ints.copy_(i32(c))
        w.copy_(clean)
        graph.replay()
        torch.cuda.synchronize()
        x = clean.clone()
        ops.prompt_attention(q, k, v, ints, 0.1, weights=x)
        assert torch.equal(w, x)


def test_prompt_refusals():
    g, q, k, v, cu, cu_k = prompts(16, [60, 40], 0, 2, 4, 64, torch.float16)
    w = held(g, 2, 2, 60)
    for bad in (w[:1], w[:, :1], w.transpose(1, 2), w[0], w[:1].expand(2, 2, 60), w[:, :1].expand(2, 2, 60)):
        with pytest.raises(ValueError):
            ops.prompt_attention(q, k, v, i32(cu), 0.1, weights=bad)
    for bad in (w.half(), w.cpu(), 5):
        with pytest.raises(TypeError):
            ops.prompt_attention(q, k, v, i32(cu), 0.1, weights=bad)
    with pytest.raises(NotImplementedError):
        ops.prompt_attention(q, k, v, i32(cu), 0.1, weights=w.clone().requires_grad_())
    before = w.clone()
    none = torch.empty(0, 4, 64, dtype=torch.float16, device=DEV)
    assert ops.prompt_attention(none, k, v, i32([0, 0, 0]), 0.1, i32(cu), weights=w).shape == (0, 4, 64)
    ops.prompt_attention(q, k[:0], v[:0], i32(cu), 0.1, i32([0, 0, 0]), weights=w)
    assert torch.equal(w, before)


def test_out_over_q():
    """attend's q may become its output, with weights too; a prompt's q is read again for the weights, so it may not."""
    lens = [300, 64]
    st, table, cu, k, g = filled(16, lens, 2, 64, torch.float16)
    q = torch.randn(2, 8, 64, generator=g).half().to(DEV)
    a, b = torch.zeros(2, 2, 512, device=DEV), torch.zeros(2, 2, 512, device=DEV)
    want, x = st.attend(q, table, i32(lens), 0.2, weights=a), q.clone()
    assert st.attend(x, table, i32(lens), 0.2, out=x, weights=b) is x
    assert torch.equal(x, want) and torch.equal(a, b)
    g, q, k, v, cu, cu_k = prompts(17, [60, 40], 0, 2, 4, 64, torch.float16)
    with pytest.raises(ValueError, match="out cannot be q"):
        ops.prompt_attention(q, k, v, i32(cu), 0.1, out=q, weights=torch.zeros(2, 2, 60, device=DEV))


def test_prompt_out_is_taken():
    """An out of its own, of other strides than a new one's, holds the output, and its weights are a new one's."""
    g, q, k, v, cu, cu_k = prompts(18, [60, 400], 0, 2, 4, 64, torch.bfloat16)
    a, b = torch.zeros(2, 2, 400, device=DEV), torch.zeros(2, 2, 400, device=DEV)
    want = ops.prompt_attention(q, k, v, i32(cu), 0.1, weights=a)
    out = torch.zeros(460, 8, 64, dtype=torch.bfloat16, device=DEV)[:, ::2]
    assert ops.prompt_attention(q, k, v, i32(cu), 0.1, out=out, weights=b) is out
    assert torch.equal(out, want) and torch.equal(a, b)


@pytest.mark.parametrize("lens,past,head", [([150], [0], (1000, 0)), ([70, 200], [0, 40], (1000, 0)), ([2900], [0], (1000, 0)),
                                            ([3, 2], [1500, 4000], (100, 900))])
@pytest.mark.parametrize("causal", [True, False])
def test_prompt_sequences_inside(lens, past, head, causal):
    """Rows and keys before the first sequence and behind the last one take no part, and no weight is written beside the
    sequences' own."""
    g, q, k, v, cu, cu_k = prompts(19, [head[0], *lens, 90], [head[1], *past, 0], 2, 4, 64, torch.float16)
    cu, cu_k = cu[1:-1], cu_k[1:-1]
    S, T = len(lens), max(b - a for a, b in zip(cu_k, cu_k[1:])) + 5
    held_all = held(g, S + 2, 2, T)
    before, w = held_all.cpu().clone(), held_all[1:-1]
    out = torch.full_like(q, 7.0)
    ops.prompt_attention(q, k, v, i32(cu), 0.2, i32(cu_k), causal=causal, out=out, weights=w)
    got, qc, kc = held_all.cpu(), q.cpu(), k.cpu()
    assert torch.equal(got[0], before[0]) and torch.equal(got[-1], before[-1])
    assert bool((out[:cu[0]] == 7).all()) and bool((out[cu[-1]:] == 7).all())
    for s in range(S):
        n = cu_k[s + 1] - cu_k[s]
        assert torch.equal(got[1 + s, :, n:], before[1 + s, :, n:])
        want, bound = E.weights(qc[cu[s]:cu[s + 1]], kc[cu_k[s]:cu_k[s + 1]], 0.2, causal, 0)
        check(got[1 + s, :, :n], before[1 + s, :, :n], want, bound, s)


@pytest.mark.parametrize("Hq", [3, 5, 8])
@pytest.mark.parametrize("kw", [dict(), dict(causal=False), dict(window=100), dict(window=1000)])
def test_prompt_alone(Hq, kw):
    """One long prompt, whose keys several workgroups share in small chunks of rows, at heads that do and do not divide them."""
    check_prompts(*prompts(20 + Hq, [1100], 0, 1, Hq, 64, torch.float16), 0.125, **kw)
