"""4-bit pages on the GPU: append, read and attend against plain definitions (oracle/serving_ref.py)."""
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


def normal(g, *shape, dtype=torch.float16, outliers=True):
    x = torch.randn(*shape, generator=g)
    if outliers and len(shape) == 3:
        x[..., :3] *= 6
    return x.to(dtype)


def tables(rng, lens, spare=3, width=None):
    """(pool size, table): pages in random order, unused entries out of range."""
    need = sum(-(-n // 64) for n in lens)
    ids = rng.sample(range(need + spare), need)
    P = width or max(1, max(-(-n // 64) for n in lens))
    t, at = [], 0
    for n in lens:
        k = -(-n // 64)
        t.append(ids[at:at + k] + [-1] * (P - k))
        at += k
    return need + spare, i32(t)


def angles(n, half):
    a = torch.arange(n)[:, None] * 10000.0 ** (-torch.arange(half) / half)
    return a.cos().float(), a.sin().float()


def filled(g, rng, lens, H, D, dtype, width=None, stale=True):
    """A store whose sequences hold random tokens; rows behind their ends hold anything."""
    pool, table = tables(rng, lens, width=width)
    st = paged.PagedStore(pool, H, D, DEV, dtype)
    if stale:
        st.pages.fill_(-1)  # codes 15, scales and zeros NaN
    N = sum(lens)
    k, v = normal(g, N, H, D, dtype=dtype), normal(g, N, H, D, dtype=dtype)
    cu = i32([sum(lens[:i]) for i in range(len(lens) + 1)])
    if N:
        st.append(k.to(DEV), v.to(DEV), table, i32([0] * len(lens)), cu)
    return st, table, cu, k, v


def held(st, table, cu, lens):
    """K and V of every token as the store holds them, on the CPU."""
    k, v = st.read(table, i32([0] * len(lens)), cu, sum(lens))
    return k.cpu(), v.cpu()


def check_attend(st, table, cu, lens, q, scale, window=None, causal_rows=None):
    k, v = held(st, table, cu, lens)
    out = st.attend(q.to(DEV), table, i32(lens), scale, window=window).cpu().double()
    qq = q if q.dim() == 4 else q[:, None]
    got = out if q.dim() == 4 else out[:, None]
    at = 0
    for s, n in enumerate(lens):
        want, bound = R.attention(qq[s], k[at:at + n], v[at:at + n], scale, window=window or 0)
        at += n
        worst = ((got[s] - want).abs() - bound).max()
        assert worst <= 0, (s, n, float(worst), float((got[s] - want).abs().max()))
    st.check()


# ---- append and read -------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,H,Hq", [(128, 2, 8), (64, 3, 3), (128, 1, 3)])
@pytest.mark.parametrize("new,held0", [([1, 1, 1], [0, 63, 64]), ([5, 0, 130], [7, 20, 61]), ([64], [0]), ([1], [31]),
                                       ([33, 1, 2, 97], [0, 127, 190, 15])])
@pytest.mark.parametrize("rot", ["full", "part", "none"])
def test_append_is_bit_exact(dtype, D, H, Hq, new, held0, rot):
    g, rng = torch.Generator().manual_seed(D + H + sum(new)), random.Random(5)
    N, S = sum(new), len(new)
    pool, table = tables(rng, [a + b for a, b in zip(new, held0)])
    st = paged.PagedStore(pool, H, D, DEV, dtype)
    st.pages.fill_(0x5A5A5A5A)
    wide = normal(g, N, Hq + 2 * H, D, dtype=dtype).to(DEV)  # one projection's output
    q, k, v = wide[:, :Hq], wide[:, Hq:Hq + H], wide[:, Hq + H:]
    cu = None if new == [1] * S else i32([sum(new[:i]) for i in range(S + 1)])
    half = {"full": D // 2, "part": 24 if D == 128 else 8, "none": 0}[rot]
    cos, sin = angles(300, half) if half else (None, None)
    got = st.append(k, v, table, i32(held0), cu, None if cos is None else cos.to(DEV),
                    None if sin is None else sin.to(DEV), q=q)
    st.check()
    at = torch.tensor([h + i for h, n in zip(held0, new) for i in range(n)])
    seq = [s for s, n in enumerate(new) for _ in range(n)]
    q, k, v = q.cpu(), k.cpu(), v.cpu()
    if half:
        q, k = R.rotate(q, cos[at], sin[at]), R.rotate(k, cos[at], sin[at])
    assert torch.equal(got.cpu(), q)
    want = [R.quantize(k), R.quantize(v)]
    pages, tab = st.pages.cpu(), table.cpu()
    touched = set()
    for n in range(N):
        page, row = int(tab[seq[n], int(at[n]) // 64]), int(at[n]) % 64
        touched.add((page, row))
        for (c, s, z), w in zip(R.page_rows(pages, page, row, D, dtype), want):
            assert torch.equal(c, w[0][n]) and torch.equal(s, w[1][n]) and torch.equal(z, w[2][n]), (n, page, row)
    for page in range(pool):  # and no other row
        for row in range(64):
            if (page, row) not in touched:
                for c, s, z in R.page_rows(pages, page, row, D, dtype):
                    assert bool((c.view(c.shape[0], -1, 2) == torch.tensor([10, 5], dtype=torch.int32)).all())
    kk, vv = st.read(table, i32(held0), cu, N)
    assert torch.equal(kk.cpu(), R.value(*want[0])) and torch.equal(vv.cpu(), R.value(*want[1]))


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_odd_groups(dtype):
    """Constant groups, zeros, infinities, NaN, the type's extremes and its smallest values."""
    big = float(torch.finfo(dtype).max)
    tiny = 2.0 ** -24 if dtype == torch.float16 else 2.0 ** -130
    x = torch.zeros(12, 1, 128)
    x[1] = 3.0
    x[2, 0, 5] = float("inf")
    x[3, 0, 40] = float("-inf")
    x[4, 0, 70] = float("nan")
    x[5, 0, :64] = big
    x[5, 0, 3] = -big
    x[6] = torch.arange(128) * tiny
    x[7] = -0.0
    x[8] = torch.linspace(-big / 4, big / 4, 128)
    x[9] = 1000 + torch.arange(128) % 2
    x[10, 0, ::2] = -tiny
    x[11] = torch.linspace(0, 15, 128)
    x = x.to(dtype)
    st = paged.PagedStore(2, 1, 128, DEV, dtype)
    table, lens, cu = i32([[1]]), i32([0]), i32([0, 12])
    st.append(x.to(DEV), x.to(DEV), table, lens, cu)
    c, s, z = R.quantize(x)
    pages = st.pages.cpu()
    for n in range(12):
        for cc, ss, zz in R.page_rows(pages, 1, n, 128, dtype):
            assert torch.equal(cc, c[n]), n
            assert torch.equal(ss.isnan(), s[n].isnan()) and torch.equal(zz.isnan(), z[n].isnan()), n
            assert torch.equal(ss.nan_to_num(), s[n].nan_to_num()) and torch.equal(zz.nan_to_num(), z[n].nan_to_num()), n


def test_append_pads_in_place_and_outputs():
    """Rows outside the sequences are left out and left as they were; q rotated in place; given outputs are used."""
    g = torch.Generator().manual_seed(0)
    st = paged.PagedStore(4, 2, 64, DEV)
    st.pages.zero_()
    N = 9  # rows 0, 1 before the first sequence, 6 .. 8 behind the last
    q, k, v = (normal(g, N, 2, 64).to(DEV) for _ in range(3))
    cos, sin = (t.to(DEV) for t in angles(80, 32))
    table, lens, cu = i32([[0, 1], [2, 3]]), i32([62, 5]), i32([2, 5, 6])
    q0 = q.clone()
    out = st.append(k, v, table, lens, cu, cos, sin, q=q, q_out=q)
    assert out is q
    at = torch.tensor([62, 63, 64, 5])
    assert torch.equal(q[2:6].cpu(), R.rotate(q0[2:6].cpu(), cos.cpu()[at], sin.cpu()[at]))
    assert torch.equal(q[:2], q0[:2]) and torch.equal(q[6:], q0[6:])
    kk, vv = torch.full((9, 2, 64), 7.0, dtype=torch.float16, device=DEV), torch.full((9, 2, 64), 8.0, device=DEV).half()
    a, b = st.read(table, lens, cu, N, k_out=kk, v_out=vv)
    assert a is kk and b is vv
    assert bool((kk[:2] == 7).all()) and bool((kk[6:] == 7).all()) and bool((vv[6:] == 8).all())
    assert torch.equal(vv[2:6].cpu(), R.value(*R.quantize(v[2:6].cpu())))
    assert int((st.pages != 0).any(-1).any(-1).sum()) == 3  # page 3 is untouched
    # strided views, and views that the kernels cannot read as they are
    base = normal(g, 4, 2, 66)[..., 1:65]
    st.append(base.to(DEV)[..., :], base.to(DEV), table, i32([0, 0]), i32([0, 2, 4]))
    kk, _ = st.read(table, i32([0, 0]), i32([0, 2, 4]), 4)
    assert torch.equal(kk.cpu(), R.value(*R.quantize(base)))


def test_bad_tokens_and_pages():
    """Entries outside the pool and tokens past the table or the rotation's rows are left out, read as NaN, and told."""
    g = torch.Generator().manual_seed(1)
    H, D = 2, 128
    st = paged.PagedStore(3, H, D, DEV)
    st.pages.fill_(0x11111111)
    before = st.pages.clone()
    k, v = normal(g, 4, H, D).to(DEV), normal(g, 4, H, D).to(DEV)
    table = i32([[3, 0], [-1, 0], [1, 2 ** 31 - 1], [2, 0]])
    st.append(k, v, table, i32([0, 5, 64, 128]))
    with pytest.raises(RuntimeError, match="outside the pool and a token past"):
        st.check()
    st.check()
    assert torch.equal(st.pages, before)
    st.append(k, v, table, i32([64, 64, 3, -1]))
    with pytest.raises(RuntimeError, match="negative length"):
        st.check()
    cos, sin = (t.to(DEV) for t in angles(60, 64))
    st.append(k, v, i32([[0], [1], [2], [0]]), i32([59, 60, 10, 61]), cos=cos, sin=sin)
    with pytest.raises(RuntimeError, match="rotation"):
        st.check()
    kk, _ = st.read(table, i32([0, 64, 64, 0]), None, 4)
    nan = kk.isnan().all(-1).all(-1).tolist()
    assert nan == [True, False, True, False]
    with pytest.raises(RuntimeError, match="outside the pool"):
        st.check()
    # attention: the sequences that need such a page are NaN, the others right
    st, table, cu, k, v = filled(torch.Generator().manual_seed(2), random.Random(2), [100, 700, 30], H, D, torch.float16)
    want = st.attend(normal(g, 3, 4, D).to(DEV) * 0, table, i32([100, 700, 30]), 1.0)
    table[1, 4] = 99
    got = st.attend(normal(g, 3, 4, D).to(DEV) * 0, table, i32([100, 700, 30]), 1.0)
    assert bool(got[1].isnan().all()) and torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])
    with pytest.raises(RuntimeError, match="outside the pool"):
        st.check()


# ---- attend ----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,H,Hq", [(128, 2, 8), (64, 2, 2), (128, 1, 3), (64, 1, 32), (128, 3, 3)])
@pytest.mark.parametrize("lens", [[1], [2, 63, 64, 65], [0, 5, 0, 300], [1000, 17, 128, 511], [255, 256, 257]])
def test_attend_lengths(dtype, D, H, Hq, lens):
    g, rng = torch.Generator().manual_seed(sum(lens)), random.Random(1)
    st, table, cu, _, _ = filled(g, rng, lens, H, D, dtype)
    check_attend(st, table, cu, lens, normal(g, len(lens), Hq, D, dtype=dtype, outliers=False), D ** -0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("m,Hq", [(2, 8), (4, 8), (5, 6), (16, 2), (16, 16)])
@pytest.mark.parametrize("window", [None, 1, 50, 64, 200])
def test_attend_drafts_and_windows(dtype, D, m, Hq, window):
    g, rng = torch.Generator().manual_seed(m), random.Random(m)
    lens = [m, 3, 0, 64 + m - 1, 333, 1, 600]
    st, table, cu, _, _ = filled(g, rng, lens, 2, D, dtype, width=11)
    check_attend(st, table, cu, lens, normal(g, len(lens), m, Hq, D, dtype=dtype, outliers=False), D ** -0.5, window)


@pytest.mark.parametrize("window", [None, 1, 64, 700, 2 ** 31 - 1])
def test_attend_one_token_windows(window):
    g, rng = torch.Generator().manual_seed(3), random.Random(3)
    lens = [1, 64, 65, 1500, 0, 129]
    st, table, cu, _, _ = filled(g, rng, lens, 2, 128, torch.float16)
    check_attend(st, table, cu, lens, normal(g, len(lens), 4, 128, outliers=False), 0.1, window)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0])
def test_attend_scales(dtype, scale):
    """Negative, zero and large scales: flat rows and rows of one weight."""
    g, rng = torch.Generator().manual_seed(4), random.Random(4)
    lens = [300, 1, 64]
    st, table, cu, _, _ = filled(g, rng, lens, 2, 64, dtype)
    check_attend(st, table, cu, lens, normal(g, len(lens), 4, 64, dtype=dtype, outliers=False), scale)


def test_attend_many_sequences():
    """More sequences than a wave has lanes, most of them short, some empty; a table wider than any needs."""
    g, rng = torch.Generator().manual_seed(6), random.Random(6)
    lens = [rng.choice([0, 1, 2, 40, 64, 130]) for _ in range(150)]
    lens[77] = 900
    st, table, cu, _, _ = filled(g, rng, lens, 1, 64, torch.float16, width=40)
    check_attend(st, table, cu, lens, normal(g, len(lens), 2, 64, outliers=False), 0.125)


@pytest.mark.parametrize("S", [257, 700])
def test_attend_more_sequences_than_one_chunk(S):
    """Past the 256 sequences that a wave takes at a time; runs of empty ones, one long one near the end."""
    g, rng = torch.Generator().manual_seed(S), random.Random(S)
    lens = [rng.choice([0, 0, 0, 1, 3]) for _ in range(S)]
    lens[0], lens[S - 2] = 70, 1300
    st, table, cu, _, _ = filled(g, rng, lens, 1, 64, torch.float16, width=21)
    check_attend(st, table, cu, lens, normal(g, S, 2, 64, outliers=False), 0.125)


@pytest.mark.parametrize("width", [5, 40])
def test_attend_into_its_queries(width):
    """Whole items, and items that several workgroups share."""
    g, rng = torch.Generator().manual_seed(11), random.Random(11)
    lens = [300, 0, 64 * width, 7]
    st, table, cu, _, _ = filled(g, rng, lens, 2, 128, torch.bfloat16)
    for m in (1, 5):
        q = normal(g, 4, m, 8, 128, dtype=torch.bfloat16, outliers=False).to(DEV)
        want = st.attend(q, table, i32(lens), 0.09)
        got = st.attend(q, table, i32(lens), 0.09, out=q)
        assert got is q and torch.equal(q, want)


@pytest.mark.parametrize("S,H,width", [(2, 1, 8), (2, 1, 9), (16, 4, 16), (16, 4, 17), (64, 4, 32), (64, 4, 33), (257, 1, 40),
                                       (700, 1, 40)])
def test_attend_table_widths(S, H, width):
    """Both sides of the widths up to which a workgroup takes a whole sequence and head."""
    g, rng = torch.Generator().manual_seed(width), random.Random(S)
    lens = [rng.choice([0, 1, 64, 130]) for _ in range(S)]
    lens[0], lens[S - 1] = width * 64, 200
    st, table, cu, _, _ = filled(g, rng, lens, H, 64, torch.float16)
    assert table.shape[1] == width
    check_attend(st, table, cu, lens, normal(g, S, 2 * H, 64, outliers=False), 0.125)


@pytest.mark.parametrize("H,Hq,D,N", [(8, 32, 128, 2100), (2, 8, 64, 9000), (32, 32, 64, 700)])
def test_append_and_read_of_many_tokens(H, Hq, D, N):
    """Enough tokens for blocks of several heads: as a few tokens at a time, which take one head per block."""
    g, rng = torch.Generator().manual_seed(N), random.Random(N)
    lens = [N // 2 + 3, 0, N - N // 2 - 3]
    k, v, q = (normal(g, N, h, D).to(DEV) for h in (H, H, Hq))
    cos, sin = (x.to(DEV) for x in angles(N, D // 2))
    pool, table = tables(rng, lens)
    one, few = (paged.PagedStore(pool, H, D, DEV) for _ in range(2))
    for st in (one, few):
        st.pages.zero_()
    cu = i32([0, lens[0], lens[0], N])
    turned = one.append(k, v, table, i32([0, 0, 0]), cu, cos, sin, q)
    parts = torch.empty_like(q)
    for s, a in ((0, 0), (2, lens[0])):
        for i in range(0, lens[s], 60):
            n = min(60, lens[s] - i)
            row = slice(a + i, a + i + n)
            few.append(k[row], v[row], table[s:s + 1], i32([i]), i32([0, n]), cos, sin, q[row], parts[row])
    assert torch.equal(one.pages, few.pages) and torch.equal(turned, parts)
    kk, vv = one.read(table, i32([0, 0, 0]), cu, N)
    for i in range(0, lens[2], 61):
        n = min(61, lens[2] - i)
        a, b = few.read(table[2:], i32([i]), i32([0, n]), n)
        assert torch.equal(a, kk[lens[0] + i:lens[0] + i + n]) and torch.equal(b, vv[lens[0] + i:lens[0] + i + n])
    one.check(), few.check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("m,Hq", [(5, 8), (16, 4), (16, 16), (3, 22), (2, 32)])
@pytest.mark.parametrize("window", [None, 1, 50, 200])
def test_attend_rows_of_two_groups(dtype, D, m, Hq, window):
    """Tables wide enough for tiles of 32 rows: 20, 32, 128, 33 and 32 rows per KV head."""
    g, rng = torch.Generator().manual_seed(m), random.Random(m)
    lens = [m, 3, 0, 64 + m - 1, 333, 1, 1600]
    st, table, cu, _, _ = filled(g, rng, lens, 2, D, dtype, width=300)
    check_attend(st, table, cu, lens, normal(g, len(lens), m, Hq, D, dtype=dtype, outliers=False), D ** -0.5, window)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
def test_attend_rows_of_two_groups_whole(dtype, D):
    """The same where a workgroup takes a whole sequence and head."""
    S, H, m = 64, 4, 4
    g, rng = torch.Generator().manual_seed(D), random.Random(D)
    lens = [rng.choice([0, 1, 3, 64, 130]) for _ in range(S)]
    lens[5], lens[S - 1] = 2048, 777
    st, table, cu, _, _ = filled(g, rng, lens, H, D, dtype)
    assert table.shape[1] == 32
    check_attend(st, table, cu, lens, normal(g, S, m, 8 * H, D, dtype=dtype, outliers=False), D ** -0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_attend_infinities_in_rows_of_two_groups(dtype, D, bad):
    """As below, for drafts in both groups of a tile; a bad page and a length past the table are told there too."""
    g, rng = torch.Generator().manual_seed(18), random.Random(18)
    lens, m, width = [130, 68, 5], 7, 1400
    st, table, cu, k, v = filled(g, rng, lens, 1, D, dtype, width=width)
    v = v.clone()
    v[127, 0, 5] = bad            # sequence 0: seen by the drafts from 127 on
    v[130 + 20, 0, 40] = bad      # sequence 1: outside the window of every row
    v[130 + 66, 0, 3] = bad       # and its sixth draft's token
    st.append(k.to(DEV), v.to(DEV), table, i32([0] * 3), cu)
    q = normal(g, 3, m, 4, D, dtype=dtype, outliers=False)
    kk, vv = held(st, table, cu, lens)
    for window in (None, 40):
        out = st.attend(q.to(DEV), table, i32(lens), D ** -0.5, window=window).cpu().double()
        at = 0
        for s, n in enumerate(lens):
            want, bound = R.attention(q[s], kk[at:at + n], vv[at:at + n], D ** -0.5, window=window or 0)
            at += n
            fine = want.isfinite()
            assert torch.equal(fine, out[s].isfinite()), (s, window)
            assert bool(((out[s] - want).abs() <= bound)[fine].all()), (s, window)
            assert torch.equal(want.isnan(), out[s].isnan())
    st.check()
    table[0, 1] = 12345
    got = st.attend(q.to(DEV), table, i32([130, width * 64 + 1, 5]), D ** -0.5).cpu()
    assert bool(got[:2].isnan().all()) and bool(torch.isfinite(got[2]).all())
    with pytest.raises(RuntimeError, match="outside the pool.*past"):
        st.check()


def test_lengths_past_the_table_are_told():
    """A length that the table has no pages for, and a negative one: NaN and 0, told by check(); the others right."""
    g, rng = torch.Generator().manual_seed(20), random.Random(20)
    for width in (2, 30):  # a workgroup per sequence and head, and shares
        st, table, cu, _, _ = filled(g, rng, [100, 128, 60], 1, 64, torch.float16, width=width)
        q = normal(g, 3, 2, 64, outliers=False).to(DEV)
        want = st.attend(q, table, i32([100, 128, 60]), 0.125)
        st.check()
        got = st.attend(q, table, i32([100, width * 64 + 1, 60]), 0.125)
        assert torch.equal(got[::2], want[::2]) and bool(got[1].isnan().all())
        with pytest.raises(RuntimeError, match="past"):
            st.check()
        got = st.attend(q, table, i32([100, -7, 60]), 0.125)
        assert torch.equal(got[::2], want[::2]) and bool((got[1] == 0).all())
        with pytest.raises(RuntimeError, match="negative"):
            st.check()


def test_attend_strides_and_out():
    g, rng = torch.Generator().manual_seed(7), random.Random(7)
    lens = [70, 300]
    st, table, cu, _, _ = filled(g, rng, lens, 2, 64, torch.float16)
    wide = torch.full((2, 8, 64), 5.0, dtype=torch.float16, device=DEV)
    q = normal(g, 2, 4, 64, outliers=False).to(DEV)
    want = st.attend(q, table, i32(lens), 0.125)
    got = st.attend(q, table, i32(lens), 0.125, out=wide[:, 2:6])
    assert torch.equal(got, want) and bool((wide[:, :2] == 5).all()) and bool((wide[:, 6:] == 5).all())
    qt = torch.empty(4, 2, 64, dtype=torch.float16, device=DEV).transpose(0, 1)
    qt.copy_(q)
    big = torch.cat([table, table], 1)[:, :table.shape[1]]  # a table with a row stride of its own
    assert torch.equal(st.attend(qt, big, i32(lens), 0.125), want)
    q4 = q[:, None].expand(2, 3, 4, 64)  # stride 0
    one = st.attend(q4, table, i32(lens), 0.125)
    assert torch.equal(one[:, 2], want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_attend_infinities_stay_where_they_are_seen(dtype, D, bad):
    """A token whose values are infinite or NaN reaches the rows that see it and no other (drafts before it, windows
    past it); a page's rows behind the sequence's end are NaN throughout (filled())."""
    g, rng = torch.Generator().manual_seed(8), random.Random(8)
    lens, m = [130, 68, 5], 4
    st, table, cu, k, v = filled(g, rng, lens, 1, D, dtype)
    v = v.clone()
    v[128, 0, 5] = bad            # sequence 0: seen by the drafts from 128 on
    v[130 + 20, 0, 40] = bad      # sequence 1: outside the window of every row
    v[130 + 66, 0, 3] = bad       # and the third draft's token
    st.append(k.to(DEV), v.to(DEV), table, i32([0] * 3), cu)
    q = normal(g, 3, m, 2, D, dtype=dtype, outliers=False)
    for window in (None, 40):
        out = st.attend(q.to(DEV), table, i32(lens), D ** -0.5, window=window).cpu().double()
        kk, vv = held(st, table, cu, lens)
        at = 0
        for s, n in enumerate(lens):
            want, bound = R.attention(q[s], kk[at:at + n], vv[at:at + n], D ** -0.5, window=window or 0)
            at += n
            fine = want.isfinite()
            assert torch.equal(fine, out[s].isfinite()), (s, window)
            assert bool(((out[s] - want).abs() <= bound)[fine].all()), (s, window)
            assert torch.equal(want.isnan(), out[s].isnan())
    assert bool(torch.isfinite(out[2]).all())


def test_attend_infinite_logits():
    """Keys of minus infinity count for nothing; a row of only such keys is 0, as one that sees no key."""
    st = paged.PagedStore(1, 1, 64, DEV)
    st.pages.zero_()
    k = torch.zeros(3, 1, 64, dtype=torch.float16)
    k[:, 0, :32] = torch.finfo(torch.float16).max
    v = torch.ones(3, 1, 64, dtype=torch.float16)
    table, cu = i32([[0]]), i32([0, 3])
    st.append(k.to(DEV), v.to(DEV), table, i32([0]), cu)
    q = torch.full((1, 1, 64), -torch.finfo(torch.float16).max, dtype=torch.float16)
    out = st.attend(q.to(DEV), table, i32([3]), 1.0)  # -1.4e11 each: finite, and far below 0
    assert torch.equal(out.cpu(), torch.ones(1, 1, 64, dtype=torch.float16))


def test_far_pages():
    """A pool past 4 GiB: page offsets of more than 32 bits."""
    D, H = 128, 8
    n = (9 << 29) // paged.PagedStore.page_bytes(H, D)  # 4.5 GiB
    st = paged.PagedStore(n, H, D, DEV)
    g = torch.Generator().manual_seed(9)
    lens = [150]
    table = i32([[n - 1, 3, n - 2]])
    k, v = normal(g, 150, H, D), normal(g, 150, H, D)
    cu = i32([0, 150])
    st.append(k.to(DEV), v.to(DEV), table, i32([0]), cu)
    kk, _ = held(st, table, cu, lens)
    assert torch.equal(kk, R.value(*R.quantize(k)))
    check_attend(st, table, cu, lens, normal(g, 1, 8, D, outliers=False), 0.1)


# ---- together --------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_serving_run(dtype):
    """Prompts, their appends, decode steps, a second chunk of one prompt, drafts: every output against 64 bits over the
    values that the cache holds."""
    g, rng = torch.Generator().manual_seed(10), random.Random(10)
    D, H, Hq, S = 64, 2, 4, 3
    prompts = [70, 9, 40]
    pool, table = tables(rng, [p + 90 for p in prompts])
    st = paged.PagedStore(pool, H, D, DEV, dtype)
    cos, sin = (t.to(DEV) for t in angles(400, D // 2))
    lens = i32([0] * S)

    def chunk(new):
        """Appends new[s] tokens each and attends for all of them over what the cache holds."""
        nonlocal lens
        N, cu = sum(new), i32([sum(new[:i]) for i in range(S + 1)])
        q, k, v = (normal(g, N, h, D, dtype=dtype).to(DEV) for h in (Hq, H, H))
        q = st.append(k, v, table, lens, cu, cos, sin, q=q)
        total = lens + i32(new)
        cu_k = torch.cat([i32([0]), total.cumsum(0, dtype=torch.int32)])
        kk, vv = st.read(table, torch.zeros_like(lens), cu_k, int(total.sum()))
        out = ops.prompt_attention(q, kk, vv, cu, D ** -0.5, cu_seqlens_k=cu_k)
        compare(out, q, kk, vv, cu.tolist(), cu_k.tolist())
        lens = total

    def compare(out, q, kk, vv, cu, cu_k):
        for s in range(S):
            want, bound = R.attention(q[cu[s]:cu[s + 1]].cpu(), kk[cu_k[s]:cu_k[s + 1]].cpu(),
                                      vv[cu_k[s]:cu_k[s + 1]].cpu(), D ** -0.5)
            assert bool(((out[cu[s]:cu[s + 1]].cpu().double() - want).abs() <= bound).all())

    chunk(prompts)
    for step in range(4):
        q, k, v = (normal(g, S, h, D, dtype=dtype).to(DEV) for h in (Hq, H, H))
        q = st.append(k, v, table, lens, cos=cos, sin=sin, q=q)
        lens = lens + 1
        out = st.attend(q, table, lens, D ** -0.5)
        cu_k = torch.cat([i32([0]), lens.cumsum(0, dtype=torch.int32)])
        kk, vv = st.read(table, torch.zeros_like(lens), cu_k, int(lens.sum()))
        compare(out, q, kk, vv, [0, 1, 2, 3], cu_k.tolist())
    chunk([0, 33, 1])
    m = 3
    q, k, v = (normal(g, S * m, h, D, dtype=dtype).to(DEV) for h in (Hq, H, H))
    cu = i32([0, m, 2 * m, 3 * m])
    q = st.append(k, v, table, lens, cu, cos, sin, q=q)
    lens = lens + m
    out = st.attend(q.view(S, m, Hq, D), table, lens, D ** -0.5)
    cu_k = torch.cat([i32([0]), lens.cumsum(0, dtype=torch.int32)])
    kk, vv = st.read(table, torch.zeros_like(lens), cu_k, int(lens.sum()))
    compare(out.view(S * m, Hq, D), q, kk, vv, cu.tolist(), cu_k.tolist())
    st.check()


def test_graph_follows_lengths_and_tables():
    """A captured step (append, attend) replayed with other tokens, lengths and tables gives the eager results; two
    graphs of one store, replayed in turn on two streams, keep apart."""
    g, rng = torch.Generator().manual_seed(11), random.Random(11)
    D, H, Hq, S = 128, 2, 8, 4
    lens0 = [500, 3, 64, 0]
    st, _, _, _, _ = filled(g, rng, [700] * S, H, D, torch.float16, width=12)
    pool = st.n_pages
    cos, sin = (t.to(DEV) for t in angles(800, D // 2))

    def buffers():
        return dict(q=torch.zeros(S, Hq, D, dtype=torch.float16, device=DEV), k=torch.zeros(S, H, D, dtype=torch.float16, device=DEV),
                    v=torch.zeros(S, H, D, dtype=torch.float16, device=DEV), lens=i32([0] * S),
                    table=torch.zeros(S, 12, dtype=torch.int32, device=DEV))

    def step(b):
        q = st.append(b["k"], b["v"], b["table"], b["lens"], cos=cos, sin=sin, q=b["q"])
        return st.attend(q, b["table"], b["lens"] + 1, 0.09)

    graphs = []
    for _ in range(2):
        b = buffers()
        step(b)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(b)
        graphs.append((graph, b, out))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(4):
        wants = []
        for (graph, b, out), stream in zip(graphs, streams):
            for x in ("q", "k", "v"):
                b[x].copy_(normal(g, *b[x].shape))
            ids = rng.sample(range(pool), S * 11)
            b["table"][:, :11].copy_(i32(ids).view(S, 11))
            b["lens"].copy_(i32([(n * (turn + 1)) % 690 for n in lens0]))
        # both steps write pages: their tables must not meet
        ids = rng.sample(range(pool), pool)
        for i, (graph, b, out) in enumerate(graphs):
            b["table"][:, :11].copy_(i32([[ids[(i * S + s) * 5 + p % 5] for p in range(11)] for s in range(S)]))
            b["lens"].copy_(i32([(n * (turn + 1) + i) % 319 for n in lens0]))
        pages = st.pages.clone()
        wants = [step(b).clone() for _, b, _ in graphs]
        after = st.pages.clone()
        st.pages.copy_(pages)
        torch.cuda.synchronize()
        for (graph, b, out), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for (graph, b, out), want in zip(graphs, wants):
            assert torch.equal(out.view(torch.int16), want.view(torch.int16)), turn  # bit for bit: NaN among them
        assert torch.equal(st.pages, after), turn


def test_same_result_every_time_and_on_another_stream():
    g, rng = torch.Generator().manual_seed(12), random.Random(12)
    lens = [3000, 17, 900]
    st, table, cu, _, _ = filled(g, rng, lens, 2, 128, torch.bfloat16)
    q = normal(g, 3, 8, 128, dtype=torch.bfloat16).to(DEV)
    want = st.attend(q, table, i32(lens), 0.09)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        for _ in range(3):
            assert torch.equal(st.attend(q, table, i32(lens), 0.09), want)


def test_refusals():
    st = paged.PagedStore(4, 2, 64, DEV)
    k = torch.zeros(3, 2, 64, dtype=torch.float16, device=DEV)
    table, lens, cu = i32([[0, 1], [2, 3]]), i32([0, 0]), i32([0, 1, 3])
    cos = torch.ones(10, 32, device=DEV)
    ok = dict(k=k, v=k, table=table, lens=lens, cu_seqlens=cu)
    st.append(**ok)
    for kw, err in [(dict(k=k[:2]), ValueError), (dict(v=k.float()), TypeError), (dict(v=k.bfloat16()), TypeError),
                    (dict(k=k.cpu()), TypeError), (dict(k=k[:, :1]), ValueError), (dict(table=table.long()), TypeError),
                    (dict(lens=i32([0])), ValueError), (dict(lens=lens.cpu()), TypeError), (dict(cu_seqlens=None), ValueError),
                    (dict(cu_seqlens=i32([0, 3])), ValueError), (dict(cu_seqlens=cu.long()), TypeError),
                    (dict(table=table[:, :0]), ValueError), (dict(table=table.t()), ValueError), (dict(cos=cos), ValueError),
                    (dict(cos=cos, sin=cos[:5]), ValueError), (dict(cos=cos.half(), sin=cos.half()), TypeError),
                    (dict(cos=cos[:, :12].contiguous(), sin=cos[:, :12].contiguous()), ValueError),
                    (dict(cos=torch.ones(4, 64, device=DEV), sin=torch.ones(4, 64, device=DEV)), ValueError),
                    (dict(q=k[:2]), ValueError), (dict(q_out=k), ValueError), (dict(q=k, q_out=k[:2]), ValueError),
                    (dict(q=k[:, :0]), ValueError), (dict(k=k.float().requires_grad_().half()), NotImplementedError)]:
        with pytest.raises(err):
            st.append(**{**ok, **kw})
    q = torch.zeros(2, 4, 64, dtype=torch.float16, device=DEV)
    ok = dict(q=q, table=table, lens=lens, scale=1.0)
    st.attend(**ok)
    for kw, err in [(dict(q=q[:1]), ValueError), (dict(q=q[:, :3]), ValueError), (dict(q=q[..., :32]), ValueError),
                    (dict(q=q.bfloat16()), TypeError), (dict(q=q[0]), ValueError), (dict(q=q[:, None].expand(2, 17, 4, 64)), ValueError),
                    (dict(window=0), ValueError), (dict(window=-3), ValueError), (dict(out=q[:1]), ValueError),
                    (dict(out=q.float()), TypeError), (dict(out=torch.zeros(2, 4, 66, device=DEV).half()[..., 1:65]), ValueError),
                    (dict(q=q[:, :0]), ValueError), (dict(q=q.clone().requires_grad_()), NotImplementedError)]:
        with pytest.raises(err):
            st.attend(**{**ok, **kw})
    with torch.no_grad():
        st.attend(q.clone().requires_grad_(), table, lens, 1.0)
    with pytest.raises(ValueError):  # rows in one place
        st.attend(q, table, lens, 1.0, out=q[:, :1].expand(2, 4, 64))
    with torch.autograd.forward_ad.dual_level(), pytest.raises(NotImplementedError):
        st.attend(torch.autograd.forward_ad.make_dual(q, q), table, lens, 1.0)
    for bad in (torch.zeros(4, 2, 100, dtype=torch.int32, device=DEV), torch.zeros(0, 2, 640, dtype=torch.int32, device=DEV),
                torch.zeros(4, 2, 1280, dtype=torch.int32, device=DEV)[..., ::2]):
        with pytest.raises(ValueError):
            paged.PagedStore.over(bad, 64)
    with pytest.raises(ValueError):
        paged.PagedStore(0, 2, 64, DEV)
    with pytest.raises(TypeError):
        paged.PagedStore(4, 2, 64, DEV, torch.float32)
    with pytest.raises(ValueError):
        st.read(table, lens, cu, 3, k_out=k[:2])


def test_the_native_front_and_the_general_path_agree(monkeypatch):
    """The same calls through csrc/iq_pyfast.cpp and through the Python path: the same bits."""
    g, rng = torch.Generator().manual_seed(13), random.Random(13)
    H, Hq, D, lens = 2, 8, 64, [70, 3, 129]
    cos, sin = (t.to(DEV) for t in angles(200, 32))
    k, v = normal(g, 202, H, D).to(DEV), normal(g, 202, H, D).to(DEV)
    q = normal(g, 202, Hq, D).to(DEV)
    _, table = tables(rng, [n + 1 for n in lens])
    cu = i32([0, 70, 73, 202])
    results = []
    for general in (False, True):
        with monkeypatch.context() as m:
            if general:
                m.setattr(ops, "_native", lambda t: None)
            st = paged.PagedStore(int(table.max()) + 1, H, D, DEV)
            st.pages.zero_()
            a = st.append(k, v, table, i32([0] * 3), cu, cos, sin, q=q)
            b = st.append(k[:3], v[:3], table, i32(lens), q=q[:3], q_out=torch.empty_like(q[:3]))
            c = st.read(table, i32([0] * 3), cu, 202)
            d = st.attend(b, table, i32(lens) + 1, 0.125)
            e = st.attend(q[:6].view(3, 2, Hq, D), table, i32(lens) + 1, 0.125, window=40, out=torch.empty(3, 2, Hq, D, device=DEV).half())
            f = ops.prompt_attention(a, c[0], c[1], cu, 0.125)
            h = ops.prompt_attention(a, c[0], c[1], cu, 0.125, cu_seqlens_k=cu, window=30, out=torch.empty_like(a))
            n = ops.prompt_attention(a, c[0], c[1], cu, 0.125, causal=False)
            assert st.append(k[:3], v[:3], table, i32(lens)) is None
            results.append([st.pages, a, b, *c, d, e, f, h, n])
    for x, y in zip(*results):
        assert torch.equal(x, y)
