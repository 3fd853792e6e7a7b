"""Caches that drop tokens, run as a serving program does: prompts, steps and evictions one behind the other, for plain and
for differential attention, each call held to its definition over what the store then holds."""
import random

import pytest
import torch

from innerq_amd import ops, paged
from oracle import diff_ref as X
from oracle import evict_ref as E
from oracle import serving_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.fixture(params=["native", "general"])
def front(request, monkeypatch):
    """The same calls through csrc/iq_pyfast.cpp and through the Python path alone."""
    if request.param == "general":
        monkeypatch.setattr(ops, "_native", lambda t: None)


class Program:
    """Three sequences, a budget of tokens each; what the store holds is read back and kept beside it on the CPU."""

    def __init__(self, seed, H, Hq, D, dtype, diff):
        self.g = torch.Generator().manual_seed(seed)
        self.H, self.Hq, self.D, self.dtype, self.diff = H, Hq, D, dtype, diff
        self.S, self.P = 3, 4
        self.store = paged.PagedStore(12, H, D, DEV, dtype)
        self.table = i32(random.Random(seed).sample(range(12), 12)).view(3, 4)
        self.lens = torch.zeros(3, dtype=torch.int32, device=DEV)
        self.gone = torch.zeros_like(self.lens)
        self.weights = torch.zeros(3, H, 256, device=DEV)
        a = torch.arange(400)[:, None] * 10000.0 ** (-torch.arange(D // 2) / (D // 2))
        self.cos, self.sin = a.cos().float().to(DEV), a.sin().float().to(DEV)
        self.lam = (torch.rand(Hq // 2, generator=self.g) + 0.1).to(DEV)
        self.scale = D ** -0.5

    def new(self, n):
        x = [torch.randn(n, h, self.D, generator=self.g).to(self.dtype).to(DEV) for h in (self.Hq, self.H, self.H)]
        x[1][..., :3] *= 4
        return x

    def held(self):
        """K and V of every token that the sequences hold, and their starts."""
        n = self.lens.tolist()
        cu = [0, n[0], n[0] + n[1], sum(n)]
        k, v = self.store.read(self.table, torch.zeros_like(self.lens), i32(cu), cu[3])
        return k, v, cu

    def check(self, q, out, before, rows, k, v, cu):
        """out and the weights' growth of the last rows[s] tokens of every sequence (q: theirs, one behind the other)."""
        q, out, k, v, now, before = (x.cpu() for x in (q, out, k, v, self.weights, before))
        at = 0
        for s, m in enumerate(rows):
            n = cu[s + 1] - cu[s]
            qq, kk, vv = q[at:at + m], k[cu[s]:cu[s + 1]], v[cu[s]:cu[s + 1]]
            if self.diff:
                want, bound = X.attention(qq, kk, vv.reshape(n, self.H // 2, 2 * self.D), self.lam.cpu(), self.scale)
                parts = [E.weights(qq[:, i::2], kk[:, i::2], self.scale) for i in (0, 1)]
            else:
                want, bound = R.attention(qq, kk, vv, self.scale)
                parts = [E.weights(qq, kk, self.scale)]
            assert ((out[at:at + m].double() - want).abs() - bound).max() <= 0
            for i, (w, b) in enumerate(parts):
                heads = slice(i, None, len(parts))
                add = now[s, heads, :n].double() - before[s, heads, :n].double()
                assert ((add - w).abs() <= b + 2.0 ** -24 * now[s, heads, :n].double()).all()
            assert torch.equal(now[s, :, n:], before[s, :, n:])
            at += m

    def prompt(self, new):
        N, cu = sum(new), i32([0, new[0], new[0] + new[1], sum(new)])
        q, k, v = self.new(N)
        q = self.store.append(k, v, self.table, self.lens, cu, self.cos, self.sin, q)
        self.lens += cu.diff()
        k, v, cu_k = self.held()
        before = self.weights.clone()
        if self.diff:
            vv = v.view(-1, self.H // 2, 2 * self.D)
            out = ops.diff_prompt_attention(q, k, vv, cu, self.lam, self.scale, weights=self.weights)
        else:
            out = ops.prompt_attention(q, k, v, cu, self.scale, weights=self.weights)
        self.check(q, out, before, new, k, v, cu_k)

    def step(self):
        q, k, v = self.new(3)
        raw_q, raw_k, at = q.cpu(), k.cpu(), (self.lens + self.gone).tolist()
        q = self.store.append(k, v, self.table, self.lens, None, self.cos, self.sin, q, evicted=self.gone)
        want = R.rotate(raw_q, self.cos.cpu()[at], self.sin.cpu()[at])
        assert torch.equal(q.cpu(), want)
        held = self.lens.tolist()
        self.lens += 1
        k, v, cu = self.held()
        turned = R.value(*R.quantize(R.rotate(raw_k, self.cos.cpu()[at], self.sin.cpu()[at])))
        assert all(torch.equal(k[cu[s] + n].cpu(), turned[s]) for s, n in enumerate(held))
        before = self.weights.clone()
        call = (self.store.diff_attend, (self.lam, self.scale)) if self.diff else (self.store.attend, (self.scale,))
        out = call[0](q, self.table, self.lens, *call[1], weights=self.weights)
        self.check(q, out, before, [1, 1, 1], k, v, cu)

    def evict(self, keep, recent, sinks):
        k, v, cu = (x.cpu() if isinstance(x, torch.Tensor) else x for x in self.held())
        w, shared, was = self.weights.cpu().numpy(), 2 if self.diff else 1, self.lens.clone()
        self.store.evict(self.table, self.lens, self.weights, keep, recent, sinks, shared, out=self.weights, lens_out=self.lens)
        self.gone += was - self.lens
        kk, vv, cc = self.held()
        kk, vv, now = kk.cpu(), vv.cpu(), self.weights.cpu().numpy()
        for s, n in enumerate(was.tolist()):
            for h in range(self.H):
                h0 = h // shared * shared
                total = w[s, h0] if shared == 1 else w[s, h0] + w[s, h0 + 1]
                src = E.kept(total[:n], keep, recent, sinks)
                assert len(src) == cc[s + 1] - cc[s]
                assert torch.equal(kk[cc[s]:cc[s + 1], h], k[cu[s]:cu[s + 1], h][src])
                assert torch.equal(vv[cc[s]:cc[s + 1], h], v[cu[s]:cu[s + 1], h][src])
                assert (now[s, h, :len(src)] == w[s, h, src]).all()
        self.store.check()


@pytest.mark.parametrize("diff", [False, True])
@pytest.mark.parametrize("D,H,Hq,dtype", [(64, 2, 4, torch.float16), (128, 4, 8, torch.bfloat16)])
def test_a_run(front, diff, D, H, Hq, dtype):
    p = Program(D + H + diff, H, Hq, D, dtype, diff)
    p.prompt([130, 40, 66])
    p.evict(60, 10, 2)
    for _ in range(5):
        p.step()
    p.evict(62, 20, 2)
    p.step()
    assert p.lens.tolist() == [63, 46, 63] and p.gone.tolist() == [73, 0, 9]
    p.evict(30, 30, 0)
    p.evict(30, 0, 4)
    for _ in range(2):
        p.step()
    p.evict(1, 0, 0)
    p.step()
    assert p.lens.tolist() == [2, 2, 2] and p.gone.tolist() == [137, 47, 73]


@pytest.mark.parametrize("width", [3, 30])
def test_both_fronts_agree(monkeypatch, width):
    """The same results through the native front and the general path, outputs given or not."""
    g = torch.Generator().manual_seed(1)
    H, Hq, D, S = 4, 8, 64, 3
    st = paged.PagedStore(S * width, H, D, DEV)
    table, lens = torch.arange(S * width, dtype=torch.int32, device=DEV).view(S, width), i32([150, 64 * width, 1])
    k = torch.randn(S * width * 64, H, D, generator=g).half().to(DEV)
    st.append(k, k.flip(0), table, i32([0] * S), i32([0, width * 64, width * 128, width * 192]))
    q, lam = torch.randn(S, Hq, D, generator=g).half().to(DEV), torch.rand(Hq // 2, generator=g).to(DEV)
    w = torch.rand(S, H, width * 64 + 1, generator=g).to(DEV)
    n = 200
    x, cu, v = torch.randn(n, Hq, D, generator=g).half().to(DEV), i32([0, 90, 90, n]), k[:n].flip(1)
    pages = st.pages.clone()

    def calls(given):
        r = []
        a, b, c, d = (w.clone() for _ in range(4))
        o = [torch.zeros(S, Hq, D, dtype=torch.half, device=DEV), torch.zeros(S, Hq // 2, 2 * D, dtype=torch.half, device=DEV),
             torch.zeros(n, Hq, D, dtype=torch.half, device=DEV), torch.zeros(n, Hq // 2, 2 * D, dtype=torch.half, device=DEV)]
        o = [y if given else None for y in o]
        r += [st.attend(q, table, lens, 0.1, out=o[0], weights=a), a]
        r += [st.diff_attend(q, table, lens, lam, 0.1, window=100, out=o[1], weights=b), b]
        r += [ops.prompt_attention(x, k[:n], v, cu, 0.1, out=o[2], weights=c), c]
        r += [ops.diff_prompt_attention(x, k[:n], v.reshape(n, H // 2, 2 * D), cu, lam, 0.1, out=o[3], weights=d), d]
        assert not given or all(y is z for y, z in zip(r[::2], o))
        ll, ww = lens.clone(), w.clone()
        new = st.evict(table, ll, ww, 100, 30, 2, 2, *((ww, ll) if given else ()))
        assert (new[0] is ll and new[1] is ww) == given
        r += [*new, st.pages.clone()]
        st.pages.copy_(pages)
        return r

    want = calls(False)
    assert torch.equal(want[0], st.attend(q, table, lens, 0.1))
    for given in (False, True):
        for native in (True, False):
            with monkeypatch.context() as m:
                if not native:
                    m.setattr(ops, "_native", lambda t: None)
                for i, (a, b) in enumerate(zip(calls(given), want)):
                    assert torch.equal(a, b), (given, native, i)
