"""Differential attention over packed prompts on the GPU against 64 bits (oracle/diff_ref.py)."""
import random

import pytest
import torch

from innerq_amd import ops
from oracle import diff_ref as X

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float16, torch.bfloat16]


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def prompts(seed, lens, past, H, Hq, D, dtype):
    g = torch.Generator().manual_seed(seed)
    past = past if isinstance(past, list) else [past] * len(lens)
    N, Nk = sum(lens), sum(max(a + b, 0) for a, b in zip(lens, past))
    q, k, v = torch.randn(N, Hq, D, generator=g), torch.randn(Nk, H, D, generator=g), torch.randn(Nk, H // 2, 2 * D, generator=g)
    k[..., :3] *= 4
    lam = torch.rand(Hq // 2, generator=g) * 0.8 + 0.1
    cu, cu_k = [0], [0]
    for a, b in zip(lens, past):
        cu.append(cu[-1] + a)
        cu_k.append(cu_k[-1] + max(a + b, 0))
    return *(x.to(dtype).to(DEV) for x in (q, k, v)), lam.to(DEV), cu, cu_k


def check(q, k, v, lam, cu, cu_k, scale, **kw):
    out = ops.diff_prompt_attention(q, k, v, i32(cu), lam, scale, i32(cu_k), **kw)
    assert out.shape == (q.shape[0], q.shape[1] // 2, 2 * q.shape[2]) and out.dtype == q.dtype
    got, q, k, v, lam = out.cpu().double(), *(x.cpu() for x in (q, k, v, lam))
    for s in range(len(cu) - 1):
        r, j = slice(cu[s], cu[s + 1]), slice(cu_k[s], cu_k[s + 1])
        if cu[s + 1] == cu[s]:
            continue
        want, bound = X.attention(q[r], k[j], v[j], lam, scale, kw.get("causal", True), kw.get("window") or 0)
        worst = ((got[r] - want).abs() - bound).max()
        assert worst <= 0, (s, float(worst))
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,H,Hq", [(128, 2, 8), (64, 4, 4), (128, 2, 2), (64, 2, 6), (64, 2, 10)])
@pytest.mark.parametrize("lens", [[1], [63, 0, 64, 65, 1], [300, 17], [31, 32, 33, 128, 129]])
@pytest.mark.parametrize("past", [0, 1, 100])
def test_lengths(dtype, D, H, Hq, lens, past):
    check(*prompts(sum(lens) + past, lens, past, H, Hq, D, dtype), D ** -0.5)


@pytest.mark.parametrize("window", [1, 2, 31, 32, 64, 65, 130, 400, 2 ** 31 - 1])
@pytest.mark.parametrize("past", [0, 150])
@pytest.mark.parametrize("D,Hq", [(64, 4), (128, 12)])
def test_windows(window, past, D, Hq):
    check(*prompts(window % 1000, [200, 1, 90, 257], past, 4, Hq, D, torch.float16), 0.125, window=window)


@pytest.mark.parametrize("past", [[0, 70, -20], [-39, 300, -89], [-40, 0, 0]])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D", [64, 128])
def test_fewer_and_more_keys(past, causal, D):
    """More rows than keys (the first see none and are 0), more keys than rows, no keys, and every row all keys."""
    q, k, v, lam, cu, cu_k = prompts(9, [40, 100, 90], past, 2, 4, D, torch.bfloat16)
    out = check(q, k, v, lam, cu, cu_k, 0.09, causal=causal)
    if causal and past[2] == -20:
        assert bool((out[140:160] == 0).all())


@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0, 50.0])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
def test_scales(scale, dtype, D):
    check(*prompts(10, [150, 40], 0, 2, 4, D, dtype), scale)


@pytest.mark.parametrize("D", [64, 128])
def test_factors(D):
    """0 (the first map alone: as prompt_attention up to its rounding), negative, 1 for equal maps, one number for all heads."""
    q, k, v, lam, cu, cu_k = prompts(11, [150, 70], 30, 4, 8, D, torch.float16)
    for x in (torch.zeros_like(lam), -lam, lam * 10, lam[:1].expand(4), torch.stack([lam, lam], 1)[:, 0]):
        check(q, k, v, x, cu, cu_k, 0.1)
    q[:, 1::2], k[:, 1::2] = q[:, ::2], k[:, ::2]
    out = ops.diff_prompt_attention(q, k, v, i32(cu), torch.ones_like(lam), 0.1, i32(cu_k))
    assert bool((out == 0).all())  # the same sums, taken from each other


def test_many_sequences():
    rng = random.Random(12)
    lens = [rng.choice([0, 0, 1, 3, 40]) for _ in range(400)]
    lens[7] = 300
    check(*prompts(12, lens, [rng.choice([0, 0, 5, 130]) for _ in lens], 2, 4, 64, torch.float16), 0.125)


@pytest.mark.parametrize("D", [64, 128])
def test_long(D):
    check(*prompts(13, [900], 700, 2, 4, D, torch.bfloat16), 0.09)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_special_values(D, dtype):
    """NaN and infinities reach the rows that see them and no other."""
    q, k, v, lam, cu, cu_k = prompts(14, [200, 100], 0, 4, 8, D, dtype)
    want = ops.diff_prompt_attention(q, k, v, i32(cu), lam, 0.1)
    # (a tile with such a V adds its keys one by one: the other values' sums may round otherwise, and are held to the
    # definition's bound, not to the same bits)
    exact, bound = (torch.cat(x).to(DEV) for x in zip(*(X.attention(*(x[a:b].cpu() for x in (q, k, v)), lam.cpu(), 0.1)
                                                       for a, b in zip(cu, cu[1:]))))
    for value in (float("nan"), float("inf"), float("-inf")):
        bad = v.clone()
        bad[120, 1, D + 5] = value  # of pair 1: output heads 2 and 3
        out = ops.diff_prompt_attention(q, k, bad, i32(cu), lam, 0.1)
        hit = torch.zeros_like(out, dtype=torch.bool)
        hit[120:200, 2:, D + 5] = True
        assert not bool(out[hit].isfinite().any())
        assert bool(((out.double() - exact).abs() <= bound)[~hit].all())
        bad = q.clone()
        bad[50, 5, 7] = value  # the second map of output head 2
        out = ops.diff_prompt_attention(bad, k, v, i32(cu), lam, 0.1)
        hit = torch.zeros_like(out, dtype=torch.bool)
        hit[50, 2] = True
        assert torch.equal(out[~hit], want[~hit]) and bool(out[50, 2].isnan().all()) == (value != value) or value == value
    bad = k.clone()
    bad[120, 2, 3] = float("nan")  # the first map of pair 1
    out = ops.diff_prompt_attention(q, bad, v, i32(cu), lam, 0.1)
    assert bool(out[120:200, 2:].isnan().all()) and torch.equal(out[:120], want[:120]) and torch.equal(out[200:], want[200:])
    assert torch.equal(out[:, :2], want[:, :2])
    # a map whose logits are all minus infinity counts as 0
    x, y = torch.ones_like(q), k.clone()
    y[:, 1::2] = 0
    y[:, 1::2, 0] = float("-inf")
    out = ops.diff_prompt_attention(x, y, v, i32(cu), lam, 0.1)
    first = ops.diff_prompt_attention(x, y, v, i32(cu), torch.zeros_like(lam), 0.1)
    assert torch.equal(out, first) and bool(out.isfinite().all())


def test_padding_outputs_and_strides():
    """Rows outside the sequences are left as they were; strided views, and views that are copied."""
    q, k, v, lam, cu, cu_k = prompts(15, [100, 40, 27], 0, 4, 8, 64, torch.bfloat16)
    want = check(q, k, v, lam, cu, cu_k, 0.1)
    cu2 = i32([20, 90, 130])
    out = torch.full_like(want, 7.0)
    assert ops.diff_prompt_attention(q, k, v, cu2, lam, 0.1, out=out) is out
    assert bool((out[:20] == 7).all()) and bool((out[130:] == 7).all()) and not bool((out[20:130] == 7).all(-1).any())
    wide = torch.zeros(167, 8 + 4 + 4, 64, dtype=q.dtype, device=DEV)
    wide[:, :8], wide[:, 8:12], wide[:, 12:] = q, k, v.view(167, 4, 64)
    vv = wide[:, 12:].unflatten(1, (2, 2)).flatten(2)
    assert vv.data_ptr() == wide[:, 12:].data_ptr()
    o = torch.zeros(167, 2, 4, 128, dtype=q.dtype, device=DEV)[:, 1]
    assert torch.equal(ops.diff_prompt_attention(wide[:, :8], wide[:, 8:12], vv, i32(cu), lam, 0.1, out=o), want)
    qt, kt, vt = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v))
    assert torch.equal(ops.diff_prompt_attention(qt, kt, vt, i32(cu), lam, 0.1), want)
    odd = torch.zeros(167, 8, 66, dtype=q.dtype, device=DEV)[..., 1:65]
    odd.copy_(q)
    assert torch.equal(ops.diff_prompt_attention(odd, k, v, i32(cu), lam, 0.1), want)


def test_streams_and_graphs():
    q, k, v, lam, cu, cu_k = prompts(16, [300, 40, 7], 0, 2, 4, 128, torch.float16)
    ints = i32(cu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out = torch.zeros(347, 2, 256, dtype=q.dtype, device=DEV)
    with torch.cuda.stream(side):
        ops.diff_prompt_attention(q, k, v, ints, lam, 0.1, out=out)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        ops.diff_prompt_attention(q, k, v, ints, lam, 0.1, out=out)
    for c, f in ((cu, 1.0), ([0, 0, 300, 347], -0.5), ([40, 41, 60, 300], 0.3)):
        ints.copy_(i32(c))
        lam.fill_(f)
        out.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        want = ops.diff_prompt_attention(q, k, v, ints, lam, 0.1, out=torch.full_like(out, 3.0))
        assert torch.equal(out, want)


def test_refusals():
    q, k, v, lam, cu, cu_k = prompts(17, [60, 40], 0, 4, 8, 64, torch.float16)
    c = i32(cu)
    f = ops.diff_prompt_attention
    for a in ((q[:, :6], k, v, c, lam[:3]), (q, k[:, :3], v, c, lam), (q, k, v[:, :1], c, lam), (q, k, v[..., :64], c, lam),
              (q, k, v, c, lam[:3]), (q, k, v, c, lam[None]), (q[:, :0], k, v, c, lam[:0]), (q, k[:, :0], v[:, :0], c, lam),
              (q, k[:50], v[:50], c, lam), (q[..., :32], k[..., :32], v[..., :64], c, lam), (q[0], k, v, c, lam),
              (q, k, v, c[:1], lam)):
        with pytest.raises(ValueError):
            f(*a, 0.1)
    for a in ((q.float(), k, v, c, lam), (q, k.bfloat16(), v, c, lam), (q, k, v, c.long(), lam), (q, k, v, c, lam.half()),
              (q, k, v, c, 0.5), (q, k, v.cpu(), c, lam), (q, k, v, c, lam.cpu())):
        with pytest.raises(TypeError):
            f(*a, 0.1)
    for kw in (dict(window=0), dict(window=-3), dict(window=5, causal=False), dict(out=q), dict(out=torch.empty_like(q[:, :4])),
               dict(out=torch.empty(1, 4, 128, dtype=q.dtype, device=DEV).expand(100, 4, 128))):
        with pytest.raises(ValueError):
            f(q, k, v, c, lam, 0.1, **kw)
    for a in ((q.clone().requires_grad_(), k, v, c, lam), (q, k, v, c, lam.clone().requires_grad_())):
        with pytest.raises(NotImplementedError):
            f(*a, 0.1)
    assert f(q[:0], k, v, i32([0, 0, 0]), lam, 0.1, c).shape == (0, 4, 128)
    assert bool((f(q, k[:0], v[:0], c, lam, 0.1, i32([0, 0, 0])) == 0).all())


@pytest.mark.parametrize("keys", [[70], [3], [70, 100], [64, 127, 130], [199]])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,Hq", [(64, 4), (128, 4), (128, 12)])
def test_infinities_in_some_tiles(D, Hq, dtype, keys):
    """Tiles of keys with and without an infinity in V follow one another at the ends of the rows' keys."""
    q, k, v, lam, cu, cu_k = prompts(17, [200, 100], 0, 4, Hq, D, dtype)
    exact, bound = (torch.cat(x).to(DEV) for x in zip(*(X.attention(*(x[a:b].cpu() for x in (q, k, v)), lam.cpu(), 0.1)
                                                       for a, b in zip(cu, cu[1:]))))
    bad, hit = v.clone(), torch.zeros_like(exact, dtype=torch.bool)
    for n, key in enumerate(keys):
        bad[key, 1, 7 * n + 1] = float("inf") if n % 2 == 0 else float("-inf")  # of pair 1
        hit[key:200, Hq // 4:, 7 * n + 1] = True
    out = ops.diff_prompt_attention(q, k, bad, i32(cu), lam, 0.1)
    assert not bool(out[hit].isfinite().any())
    assert bool(((out.double() - exact).abs() <= bound)[~hit].all())
