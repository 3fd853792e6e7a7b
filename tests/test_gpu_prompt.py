"""ops.prompt_attention on the GPU against attention in 64 bits (oracle/serving_ref.py)."""
import random

import pytest
import torch

from innerq_amd import ops
from oracle import serving_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float16, torch.bfloat16]


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def starts(lens):
    return [sum(lens[:i]) for i in range(len(lens) + 1)]


def inputs(seed, lq, lk, Hq, H, D, dtype):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(sum(lq), Hq, D, generator=g).to(dtype)
    k = torch.randn(sum(lk), H, D, generator=g)
    k[..., :3] *= 4
    v = torch.randn(sum(lk), H, D, generator=g)
    return q, k.to(dtype), v.to(dtype)


def check(q, k, v, lq, lk, scale, causal=True, window=None, **kw):
    cu, cu_k = starts(lq), starts(lk)
    out = ops.prompt_attention(q.to(DEV), k.to(DEV), v.to(DEV), i32(cu), scale, cu_seqlens_k=i32(cu_k), causal=causal,
                               window=window, **kw)
    compare(out, q, k, v, cu, cu_k, scale, causal, window)
    return out


def compare(out, q, k, v, cu, cu_k, scale, causal=True, window=None):
    got = out.cpu().double()
    for s in range(len(cu) - 1):
        want, bound = R.attention(q[cu[s]:cu[s + 1]], k[cu_k[s]:cu_k[s + 1]], v[cu_k[s]:cu_k[s + 1]], scale, causal,
                                  window or 0)
        d = (got[cu[s]:cu[s + 1]] - want).abs() - bound
        assert d.numel() == 0 or d.max() <= 0, (s, float(d.max()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,Hq,H", [(128, 4, 1), (64, 2, 2), (128, 3, 1), (64, 8, 2)])
@pytest.mark.parametrize("lens", [[1], [31, 32, 33], [63, 64, 65, 1, 0, 2], [127, 128, 129], [300, 5, 257]])
def test_lengths(dtype, D, Hq, H, lens):
    q, k, v = inputs(sum(lens) + D, lens, lens, Hq, H, D, dtype)
    check(q, k, v, lens, lens, D ** -0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lq,lk", [([5, 1], [200, 64]), ([130], [131]), ([70, 3, 0], [10, 3, 5]), ([1, 1, 1], [1, 65, 0]),
                                   ([200], [33]), ([64, 64], [192, 64])])
@pytest.mark.parametrize("causal,window", [(True, None), (False, None), (True, 1), (True, 20), (True, 64), (True, 130)])
def test_chunks_and_windows(dtype, D, lq, lk, causal, window):
    """More keys than rows, fewer (rows that see none are 0), windows that start inside a tile."""
    q, k, v = inputs(sum(lk), lq, lk, 2, 1, D, dtype)
    check(q, k, v, lq, lk, D ** -0.5, causal, window)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [-0.3, 0.0, 2.0])
def test_scales(dtype, scale):
    lens = [100, 40]
    q, k, v = inputs(3, lens, lens, 2, 2, 64, dtype)
    check(q, k, v, lens, lens, scale)


def test_long():
    """Many tiles of keys, running maxima that rise to the last; a few rows of it checked."""
    D, n = 128, 5000
    g = torch.Generator().manual_seed(5)
    k = torch.randn(n, 1, D, generator=g) * torch.linspace(0.2, 2, n)[:, None, None]
    q, k, v = torch.randn(n, 2, D, generator=g).half(), k.half(), torch.randn(n, 1, D, generator=g).half()
    out = ops.prompt_attention(q.to(DEV), k.to(DEV), v.to(DEV), i32([0, n]), 0.09).cpu().double()
    for i in (0, 1, 63, 64, 127, 128, 2047, 4095, 4999):
        want, bound = R.attention(q[i:i + 1], k[:i + 1], v[:i + 1], 0.09)
        assert bool(((out[i] - want[0]).abs() <= bound[0]).all()), i


def test_windows_past_every_length():
    lq, lk = [70, 3], [20, 90]
    q, k, v = inputs(6, lq, lk, 2, 1, 64, torch.float16)
    for window in (90, 110, 2 ** 31 - 1):
        check(q, k, v, lq, lk, 0.125, True, window)


@pytest.mark.parametrize("S", [64, 65, 256, 257, 4097, 5000])
def test_more_sequences_than_one_search_step(S):
    rng = random.Random(S)
    lens = [rng.choice([0, 0, 1, 2]) for _ in range(S)]
    lens[S - 2] = 150
    q, k, v = inputs(S, lens, lens, 2, 1, 64, torch.float16)
    check(q, k, v, lens, lens, 0.125)


def test_many_sequences():
    rng = random.Random(2)
    lens = [rng.choice([0, 1, 2, 7, 40]) for _ in range(200)]
    lens[131] = 300
    q, k, v = inputs(7, lens, lens, 2, 1, 64, torch.float16)
    check(q, k, v, lens, lens, 0.125)


def test_strides_rows_behind_and_out():
    """Views of one projection's output; rows before and behind the sequences are left as they were."""
    lens = [50, 140]
    g = torch.Generator().manual_seed(8)
    x = torch.randn(200, 8, 64, generator=g).half().to(DEV)
    x[:4] = float("nan")
    x[194:] = float("nan")
    q, k, v = x[:, :4], x[:, 4:6], x[:, 6:]
    wide = torch.full((200, 6, 64), 3.0, dtype=torch.float16, device=DEV)
    out = wide[:, 1:5]
    cu = [4, 54, 194]
    got = ops.prompt_attention(q, k, v, i32(cu), 0.125, out=out)
    assert got is out and bool((wide[:4] == 3).all()) and bool((wide[194:] == 3).all()) and bool((wide[:, 0] == 3).all())
    assert bool((wide[:, 5] == 3).all())
    compare(out[4:194], q[4:194].cpu(), k[4:194].cpu(), v[4:194].cpu(), starts(lens), starts(lens), 0.125)
    # a head-major view, one that the kernel cannot read as it is, and keys shared by all heads
    qt = q.transpose(0, 1).contiguous().transpose(0, 1)
    odd = torch.randn(200, 2, 65, device=DEV).half()[..., 1:]
    odd.copy_(k)
    assert torch.equal(ops.prompt_attention(qt, odd, v, i32(cu), 0.125)[4:194], out[4:194])
    shared = ops.prompt_attention(q, k[:, :1].expand(200, 2, 64), v[:, :1].expand(200, 2, 64), i32(cu), 0.125)
    assert torch.equal(shared[4:194], ops.prompt_attention(q, k[:, :1], v[:, :1], i32(cu), 0.125)[4:194])


def test_bounds_outside_the_tensors():
    """Cumulative lengths outside the tensors are moved to their ends: nothing outside is read or written."""
    q, k, v = (t.to(DEV) for t in inputs(9, [80], [80], 2, 1, 64, torch.float16))
    want = ops.prompt_attention(q, k, v, i32([0, 80]), 0.125)
    out = torch.zeros_like(q)
    ops.prompt_attention(q, k, v, i32([-5, 2 ** 31 - 1]), 0.125, out=out)
    assert torch.equal(out, want)
    out.zero_()
    ops.prompt_attention(q, k, v, i32([0, 50, 20, 80]), 0.125, out=out)  # rows 20 .. 49 are claimed by two sequences
    assert torch.equal(out[:20], ops.prompt_attention(q, k, v, i32([0, 50]), 0.125)[:20])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_infinities_stay_where_they_are_seen(dtype, D, bad):
    """Infinite or NaN values reach the rows that see their key and no other: causal rows before it, windows past it,
    the neighbouring sequence."""
    lens = [150, 90]
    q, k, v = inputs(11, lens, lens, 2, 1, D, dtype)
    v[100, 0, 7] = bad
    v[149, 0, 33] = bad
    v[150 + 10, 0, 1] = bad
    k[150 + 40, 0, 5] = float("nan")
    for window in (None, 30):
        out = ops.prompt_attention(q.to(DEV), k.to(DEV), v.to(DEV), i32(starts(lens)), D ** -0.5, window=window)
        got, cu = out.cpu().double(), starts(lens)
        for s in range(2):
            a, b = cu[s], cu[s + 1]
            want, bound = R.attention(q[a:b], k[a:b], v[a:b], D ** -0.5, True, window or 0)
            fine = want.isfinite()
            assert torch.equal(want.isnan(), got[a:b].isnan()), (s, window)
            assert torch.equal(fine, got[a:b].isfinite())
            assert bool(((got[a:b] - want).abs() <= bound)[fine].all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_extreme_logits(dtype):
    """Logits of the type's largest values: one weight is 1, the rest 0, and nothing overflows to NaN."""
    n = 70
    q, k, v = inputs(12, [n], [n], 1, 1, 64, dtype)
    q, k = (q.float() * 300).to(dtype), (k.float() * 300).to(dtype)
    out = ops.prompt_attention(q.to(DEV), k.to(DEV), v.to(DEV), i32([0, n]), 1.0).cpu()
    assert bool(torch.isfinite(out).all())
    s = torch.einsum("qd,kd->qk", q[:, 0].double(), k[:, 0].double()).masked_fill(torch.ones(n, n).triu(1).bool(), -1e300)
    top = s.topk(2, -1).values
    sure = top[:, 0] - top[:, 1] > 100
    sure[0] = True
    assert int(sure.sum()) > 40 and torch.equal(out[sure, 0], v[s.argmax(-1)[sure], 0])


def test_graph_follows_lengths():
    q, k, v = (t.to(DEV) for t in inputs(13, [400], [400], 4, 2, 128, torch.bfloat16))
    cu = i32([0, 400, 400, 400])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    ops.prompt_attention(q, k, v, cu, 0.09)
    with torch.cuda.graph(graph):
        out = ops.prompt_attention(q, k, v, cu, 0.09)
    for lens in ([400, 0, 0], [1, 200, 199], [130, 140, 130], [10, 20, 0]):
        cu.copy_(i32(starts(lens)))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        want = torch.zeros_like(out)
        ops.prompt_attention(q, k, v, cu, 0.09, out=want)
        assert torch.equal(out, want), lens


def test_another_stream_same_result():
    q, k, v = (t.to(DEV) for t in inputs(14, [900], [900], 2, 1, 128, torch.float16))
    want = ops.prompt_attention(q, k, v, i32([0, 900]), 0.09)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        for _ in range(3):
            assert torch.equal(ops.prompt_attention(q, k, v, i32([0, 900]), 0.09), want)
    torch.cuda.synchronize()


@pytest.mark.parametrize("D", [64, 128])
def test_tiles_are_waited_for(D):
    """Tiles reach LDS behind the program's back: many runs, each on memory that was just written, give the same bits."""
    lens = [900, 5, 257, 640]
    q, k, v = (t.to(DEV) for t in inputs(16, lens, lens, 8, 2, D, torch.float16))
    cu = i32(starts(lens))
    want = ops.prompt_attention(q, k, v, cu, 0.09)
    for _ in range(30):
        a, b, c = q.clone(), k.clone(), v.clone()
        assert torch.equal(ops.prompt_attention(a, b, c, cu, 0.09), want)


@pytest.mark.parametrize("Hq,H", [(4, 1), (2, 2), (6, 2)])
def test_into_its_queries(Hq, H):
    lens = [300, 1, 0, 129]
    q, k, v = (t.to(DEV) for t in inputs(17, lens, lens, Hq, H, 128, torch.bfloat16))
    cu = i32(starts(lens))
    want = ops.prompt_attention(q, k, v, cu, 0.09)
    assert ops.prompt_attention(q, k, v, cu, 0.09, out=q) is q and torch.equal(q, want)


def test_refusals():
    q, k, v = (t.to(DEV) for t in inputs(15, [20], [20], 4, 2, 64, torch.float16))
    cu = i32([0, 20])
    ok = dict(q=q, k=k, v=v, cu_seqlens=cu, scale=1.0)
    ops.prompt_attention(**ok)
    for kw, err in [(dict(q=q[:, :3]), ValueError), (dict(k=k[:19]), ValueError), (dict(v=v[:19]), ValueError),
                    (dict(k=k.bfloat16()), TypeError), (dict(q=q.float()), TypeError), (dict(v=v.cpu()), TypeError),
                    (dict(cu_seqlens=cu.long()), TypeError), (dict(cu_seqlens=cu[:1]), ValueError),
                    (dict(cu_seqlens=cu.cpu()), TypeError), (dict(cu_seqlens_k=i32([0, 1, 20])), ValueError),
                    (dict(window=0), ValueError), (dict(window=5, causal=False), ValueError), (dict(out=q[:5]), ValueError),
                    (dict(out=q.float()), TypeError), (dict(q=q[..., :32], k=k[..., :32], v=v[..., :32]), ValueError),
                    (dict(q=q[0]), ValueError), (dict(q=q[:, :0]), ValueError),
                    (dict(q=q.clone().requires_grad_()), NotImplementedError),
                    (dict(v=v.clone().requires_grad_()), NotImplementedError)]:
        with pytest.raises(err):
            ops.prompt_attention(**{**ok, **kw})
    with pytest.raises(ValueError):  # rows in one place
        ops.prompt_attention(**ok, out=q[:, :1].expand(20, 4, 64))
    with torch.autograd.forward_ad.dual_level(), pytest.raises(NotImplementedError):
        ops.prompt_attention(**{**ok, "k": torch.autograd.forward_ad.make_dual(k, k)})
    assert ops.prompt_attention(q[:0], k, v, cu, 1.0, cu_seqlens_k=cu).shape == (0, 4, 64)
    none = ops.prompt_attention(q, k[:0], v[:0], cu, 1.0, cu_seqlens_k=i32([0, 0]))
    assert bool((none == 0).all())
