"""The launches that weigh a prompt's keys, each at sizes that reach it (the rule: iq_prompt_weights.h), on the GPU against 64
bits (oracle/evict_ref.py: gathered)."""
import pytest
import torch

from innerq_amd import ops
from oracle import diff_ref as X
from oracle import evict_ref as E
from oracle import serving_ref as R
from test_prompt_weights_plan import plan  # noqa: F401

DEV = "cuda:0"
DTYPES = [torch.float16, torch.bfloat16]

# rows and keys of the sequences, query and KV heads: all of them few rows over many keys, but for the last three
SIZES = {
    "few": ([20, 3, 64, 1], [4000, 3700, 5000, 1700], 8, 8),
    "few, grouped heads": ([20, 3, 31, 1], [4000, 3700, 5000, 1700], 24, 8),
    "few, one sequence": ([50], [15001], 32, 8),
    "few, steps": ([33, 7], [9000, 12345], 16, 8),
    "few, more steps": ([1, 4, 2], [9000, 1, 51007], 16, 8),
    "few, rows in turns": ([100, 1], [9000, 6000], 32, 8),
    "few, a turn of a row": ([257, 0, 0, 5], [7000, 0, 300, 8000], 8, 8),
    "few, more rows than keys": ([40, 2, 30], [10, 14500, 0], 8, 8),
    "few, 16 heads": ([9, 0, 130], [3000, 100, 4200], 16, 16),
    "shares": ([1500], [1500], 2, 2),
    "shares, grouped heads": ([700, 5, 300], [900, 2005, 300], 12, 2),
    "shares of whole chunks": ([2100, 100], [2100, 1100], 8, 2),
}


def sizes(name):
    rows, keys, Hq, H = SIZES[name]
    return len(rows), sum(rows), sum(keys), Hq, H


def test_sizes_reach_their_launches(plan):  # noqa: F811
    found = dict(zip(SIZES, plan([sizes(name) for name in SIZES])))
    for name, (few, steps, shares, chunk) in found.items():
        assert few == name.startswith("few"), name
        assert few or shares > 1, name
    assert found["few"][1] == 1 and found["few, steps"][1] == 2 and found["few, more steps"][1] == 4
    S, N, Nk, Hq, H = sizes("few, rows in turns")
    assert max(SIZES["few, rows in turns"][0]) * Hq // H > 256 and max(SIZES["few, a turn of a row"][0]) == 257
    assert found["shares"][3] == 256 and found["shares of whole chunks"][3] < max(SIZES["shares of whole chunks"][0]) * 4


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def starts(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def made(name, D, dtype, wide=1):
    """q, k, v (its heads ``wide`` D) and the starts of the sequences' rows and keys."""
    rows, keys, Hq, H = SIZES[name]
    g = torch.Generator().manual_seed(sum(rows) + D)
    q, k = torch.randn(sum(rows), Hq, D, generator=g), torch.randn(sum(keys), H, D, generator=g)
    v = torch.randn(sum(keys), H // wide, wide * D, generator=g)
    return *(x.to(dtype).to(DEV) for x in (q, k, v)), starts(rows), starts(keys)


def check_weights(w, before, q, k, cu, cu_k, scale, maps=1, **kw):
    """w = before + what the keys gather: within the bound, and nothing else changed."""
    T = w.shape[2]
    for s in range(len(cu) - 1):
        r, j, n = slice(cu[s], cu[s + 1]), slice(cu_k[s], cu_k[s + 1]), min(cu_k[s + 1] - cu_k[s], T)
        assert torch.equal(w[s, :, n:], before[s, :, n:]), s
        for i in range(maps):
            want, bound = E.gathered(q[r, i::maps], k[j, i::maps], scale, **kw)
            want, bound, old = want[:, :n], bound[:, :n], before[s, i::maps, :n].double()
            worst = ((w[s, i::maps, :n].double() - old - want).abs() - bound - 2.0 ** -24 * (old + want)).amax() if n else 0
            assert worst <= 0, (s, i, float(worst))
            # (a key that no row sees is left as it is)
            assert torch.equal(w[s, i::maps, :n][want == 0], before[s, i::maps, :n][want == 0]), s


@pytest.mark.gpu
@pytest.mark.parametrize("D,dtype", [(64, torch.float16), (128, torch.bfloat16)])
@pytest.mark.parametrize("kw", [dict(), dict(causal=False), dict(window=700), dict(window=1), dict(window=3001)])
@pytest.mark.parametrize("name", SIZES)
def test_weights(name, D, dtype, kw):
    q, k, v, cu, cu_k = made(name, D, dtype)
    S, longest = len(cu) - 1, max(SIZES[name][1])
    for T, held in ((longest + 5, 0.0), (longest * 2 // 3 + 1, 1.0)):
        w = torch.rand(S, k.shape[1], T, device=DEV, generator=torch.Generator(DEV).manual_seed(T)) * held
        before = w.clone()
        ops.prompt_attention(q, k, v, i32(cu), D ** -0.5, i32(cu_k), weights=w, **kw)
        check_weights(w, before, q, k, cu, cu_k, D ** -0.5, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("D,dtype", [(64, torch.bfloat16), (128, torch.float16)])
@pytest.mark.parametrize("kw", [dict(), dict(window=700)])
@pytest.mark.parametrize("name", SIZES)
def test_weights_of_two_maps(name, D, dtype, kw):
    q, k, v, cu, cu_k = made(name, D, dtype, wide=2)
    S, longest = len(cu) - 1, max(SIZES[name][1])
    lam = torch.rand(q.shape[1] // 2, device=DEV)
    w = torch.rand(S, k.shape[1], longest + 5, device=DEV)
    before = w.clone()
    want = ops.diff_prompt_attention(q, k, v, i32(cu), lam, D ** -0.5, i32(cu_k), **kw)
    out = ops.diff_prompt_attention(q, k, v, i32(cu), lam, D ** -0.5, i32(cu_k), weights=w, **kw)
    assert torch.equal(out, want)
    check_weights(w, before, q, k, cu, cu_k, D ** -0.5, maps=2, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["few", "few, rows in turns", "shares", "shares, grouped heads"])
def test_rows_of_nan_and_infinities(name):
    """NaN stays with the keys that its row and KV head see; a key of minus infinity gathers nothing."""
    q, k, v, cu, cu_k = made(name, 64, torch.float16)
    S, H, r, longest = len(cu) - 1, k.shape[1], q.shape[1] // k.shape[1], max(SIZES[name][1])
    clean = torch.zeros(S, H, longest + 5, device=DEV)
    want = clean.clone()
    ops.prompt_attention(q, k, v, i32(cu), 0.125, i32(cu_k), weights=want, window=901)
    for value in (float("nan"), float("inf"), float("-inf")):
        bad, w = q.clone(), clean.clone()
        row = cu[1] - 2  # the last but one of sequence 0
        bad[row, r - 1, 3] = value  # of KV head 0
        ops.prompt_attention(bad, k, v, i32(cu), 0.125, i32(cu_k), weights=w, window=901)
        keys = cu_k[1] - cu_k[0]
        low, high = max(keys - 1 - 901, 0), keys - 1
        assert bool(w[0, 0, low:high].isnan().all())
        # what only other rows see is theirs (a wave with an infinite base rounds its other logits otherwise)
        rest = torch.ones_like(w, dtype=torch.bool)
        rest[0, 0, low:high] = False
        assert bool(((w - want).abs() <= 1e-4 * want + 1e-30)[rest].all())
        assert torch.equal(w[1:], want[1:]) and torch.equal(w[0, 1:], want[0, 1:])
    low = clean.clone()
    x, y = q.abs(), k.clone()
    y[cu_k[0] + 5:cu_k[1]:3, :, 0] = float("-inf")
    x[..., 0] += 1
    ops.prompt_attention(x, y, v, i32(cu), 0.125, i32(cu_k), weights=low)
    assert bool(low.isfinite().all()) and bool((low[0, :, 5:cu_k[1]:3] == 0).all()) and bool((low[0, :, :5] > 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["few", "few, steps", "few, rows in turns", "shares, grouped heads"])
def test_sequences_inside_and_graphs(name):
    """Rows and keys beside the sequences take no part; a captured call follows its lengths, over several replays."""
    q, k, v, cu, cu_k = made(name, 64, torch.float16)
    S, H, longest = len(cu) - 1, k.shape[1], max(SIZES[name][1])
    ints, ints_k = i32(cu), i32(cu_k)
    clean = torch.rand(S, H, longest + 5, device=DEV)
    w = clean.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.prompt_attention(q, k, v, ints, 0.1, ints_k, weights=w)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        o = ops.prompt_attention(q, k, v, ints, 0.1, ints_k, weights=w)
    inside = [min(max(c, 2), cu[-1] - 1) for c in cu]
    inside_k = [min(max(c, 700), cu_k[-1] - 900) for c in cu_k]
    for a, b in ((cu, cu_k), (inside, inside_k), ([0] * S + [cu[-1]], [0] * S + [min(longest, cu_k[-1])]), (cu, cu_k)):
        ints.copy_(i32(a))
        ints_k.copy_(i32(b))
        w.copy_(clean)
        o.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        x, y = clean.clone(), torch.full_like(o, 7.0)
        ops.prompt_attention(q, k, v, ints, 0.1, ints_k, weights=x, out=y)
        assert torch.equal(w, x) and torch.equal(o, y)
        assert bool((o[:a[0]] == 7).all()) and bool((o[a[-1]:] == 7).all())
        check_weights(w, clean, q, k, a, b, 0.1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,H,Hq", [(64, 4, 8), (128, 2, 4)])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_queries_that_are_not_finite(D, H, Hq, dtype, value):
    """A row whose query holds NaN or an infinity is NaN, in its own map's head alone, and no other row leaves its bound."""
    g = torch.Generator().manual_seed(14)
    q, k, v = torch.randn(300, Hq, D, generator=g), torch.randn(300, H, D, generator=g), torch.randn(300, H, D, generator=g)
    q, k, v = (x.to(dtype) for x in (q, k, v))
    lam, cu = torch.rand(Hq // 2, generator=g), [0, 200, 300]
    bad = q.clone()
    bad[50, Hq - 1, 7] = value  # of the last head, which is the second map of the last output head
    parts = [R.attention(*(x[a:b] for x in (q, k, v)), 0.1) for a, b in zip(cu, cu[1:])]
    want, bound = (torch.cat(x) for x in zip(*parts))
    out = ops.prompt_attention(bad.to(DEV), k.to(DEV), v.to(DEV), i32(cu), 0.1).cpu().double()
    assert bool(out[50, Hq - 1].isnan().all())
    out[50, Hq - 1] = want[50, Hq - 1]
    assert bool(((out - want).abs() <= bound).all())
    vv = v.reshape(300, H // 2, 2 * D)
    parts = [X.attention(*(x[a:b] for x in (q, k, vv)), lam, 0.1) for a, b in zip(cu, cu[1:])]
    want, bound = (torch.cat(x) for x in zip(*parts))
    out = ops.diff_prompt_attention(bad.to(DEV), k.to(DEV), vv.to(DEV), i32(cu), lam.to(DEV), 0.1).cpu().double()
    assert bool(out[50, Hq // 2 - 1].isnan().all())
    out[50, Hq // 2 - 1] = want[50, Hq // 2 - 1]
    assert bool(((out - want).abs() <= bound).all())
