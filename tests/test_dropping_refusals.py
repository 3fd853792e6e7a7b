"""The C ABI of gathered attention weights, of dropping tokens and of differential attention refuses bad arguments on
the host, before any launch (no GPU here: each case has one invalid argument), workspaces are as large as what they
hold, and CPU tensors raise."""
import ctypes

import pytest
import torch

from innerq_amd import _lib, ops, paged

FAKE, OUT = ctypes.c_void_p(0x1000), ctypes.c_void_p(0x2000)  # never dereferenced
ODD, ODD4 = ctypes.c_void_p(0x1008), ctypes.c_void_p(0x1002)


def _paged(**kw):
    a = dict(pages=0x1000, n_pages=8, table=0x1000, s_table=4, lens=0x1000, status=0x1000, S=3, P=4, H=8, D=128, mode=0)
    a.update(kw)
    p = _lib.iq_paged()
    for name, x in a.items():
        setattr(p, name, x)
    return ctypes.byref(p)


BAD_STORES = [(dict(pages=None), -1), (dict(table=None), -1), (dict(lens=None), -1), (dict(status=None), -1),
              (dict(mode=1), -7), (dict(mode=2), -7), (dict(D=96), -4), (dict(H=0), -4), (dict(S=0), -4), (dict(P=0), -4),
              (dict(n_pages=0), -4), (dict(pages=0x1008), -5), (dict(table=0x1002), -5), (dict(lens=0x1002), -5)]
ROOM = dict(ws=FAKE, wsb=1 << 40, stream=None)
GATHERED = dict(weights=FAKE, sw_s=2048, sw_h=256, T=256)


def _append(store=None, **kw):
    a = dict(cu=FAKE, N=5, k=FAKE, sk_n=1024, sk_h=128, v=FAKE, sv_n=1024, sv_h=128, cos=FAKE, sin=FAKE, n_pos=100, R=128,
             evicted=FAKE, q=FAKE, sq_n=4096, sq_h=128, Hq=32, q_out=FAKE, so_n=4096, so_h=128, stream=None)
    a.update(kw)
    return _lib.lib().iq_paged_append_at(store or _paged(), *a.values())


def _evict(store=None, **kw):
    a = dict(weights=FAKE, sw_s=2048, sw_h=256, weights_out=FAKE, so_s=2048, so_h=256, T=256, keep=100, recent=20, sinks=4,
             shared=1, lens_out=FAKE, **ROOM)
    a.update(kw)
    return _lib.lib().iq_paged_evict(store or _paged(), *a.values())


def _attend(store=None, **kw):
    a = dict(q=FAKE, sq_s=4096, sq_h=128, Hq=32, scale=1.0, window=0, out=FAKE, so_s=4096, so_h=128, **GATHERED, **ROOM)
    a.update(kw)
    return _lib.lib().iq_paged_attention_weights(store or _paged(), *a.values())


def _diff_attend(store=None, **kw):
    a = dict(q=FAKE, sq_s=4096, sq_m=4096, sq_h=128, m=1, Hq=32, lam=FAKE, s_lam=1, scale=1.0, window=0, out=OUT, so_s=4096,
             so_m=4096, so_h=256, **GATHERED, **ROOM)
    a.update(kw)
    return _lib.lib().iq_diff_paged_attention(store or _paged(), *a.values())


QKV = dict(q=FAKE, sq_n=4096, sq_h=128, k=FAKE, sk_n=1024, sk_h=128, v=FAKE, sv_n=1024, sv_h=128)
SIZES = dict(cu_q=FAKE, cu_k=FAKE, S=3, N=50, Nk=50, Hq=32, H=8, D=128, mode=0, scale=1.0, causal=1, window=0)


def _prompt(**kw):
    a = dict(**QKV, **SIZES, out=OUT, so_n=4096, so_h=128, **GATHERED, **ROOM)
    a.update(kw)
    return _lib.lib().iq_prompt_attention_weights(*a.values())


def _diff_prompt(**kw):
    a = dict(**QKV, lam=FAKE, s_lam=1, **SIZES, out=OUT, so_n=4096, so_h=256, **GATHERED, **ROOM)
    a.update(kw)
    return _lib.lib().iq_diff_prompt_attention(*a.values())


@pytest.mark.parametrize("kw,err", BAD_STORES)
@pytest.mark.parametrize("fn", [_append, _evict, _attend, _diff_attend])
def test_bad_stores(fn, kw, err):
    assert fn(_paged(**kw)) == err


@pytest.mark.parametrize("kw,err", [(dict(k=None), -1), (dict(cos=None), -1), (dict(evicted=ODD4), -5), (dict(N=-1), -4),
                                    (dict(R=24), -4), (dict(q=ODD), -5)])
def test_append_at_rejects(kw, err):
    assert _append(**kw) == err


@pytest.mark.parametrize("store,kw,err", [
    ({}, dict(weights=None), -1), ({}, dict(weights_out=None), -1), ({}, dict(lens_out=None), -1), ({}, dict(keep=0), -4),
    ({}, dict(keep=-5), -4), ({}, dict(recent=-1), -4), ({}, dict(sinks=-1), -4), ({}, dict(recent=97), -4),
    ({}, dict(recent=2 ** 31 - 1, sinks=2 ** 31 - 1), -4), ({}, dict(sinks=81), -4), ({}, dict(shared=0), -4),
    ({}, dict(shared=3), -4), ({}, dict(T=255), -4), ({}, dict(sw_s=-1), -4), ({}, dict(so_h=-1), -4),
    ({}, dict(so_h=512), -4),                                        # in place, but at other strides
    ({}, dict(weights=ODD4), -5), ({}, dict(lens_out=ODD4), -5), ({}, dict(ws=None), -6), ({}, dict(wsb=8), -6),
    ({}, dict(ws=ODD4), -5), (dict(S=1 << 20), dict(), -4),          # 2^23 (sequence, head) pairs
    (dict(P=1 << 25), dict(T=1 << 40), -4)])
def test_evict_rejects(store, kw, err):
    assert _evict(_paged(**store), **kw) == err


WEIGHTS = [(dict(T=255), -4), (dict(sw_s=-1), -4), (dict(sw_h=-1), -4), (dict(weights=ODD4), -5), (dict(ws=None), -6),
           (dict(wsb=1000), -6), (dict(ws=ODD), -5)]
PAGED_Q = [(dict(q=None), -1), (dict(out=None), -1), (dict(Hq=0), -4), (dict(Hq=12), -4), (dict(Hq=8192), -4),
           (dict(window=-1), -4), (dict(q=ODD), -5), (dict(sq_h=4), -5), (dict(so_s=12), -5)]


@pytest.mark.parametrize("kw,err", [(dict(weights=None), -1), *PAGED_Q, *WEIGHTS])
def test_attend_weights_rejects(kw, err):
    assert _attend(**kw) == err


@pytest.mark.parametrize("store,kw,err", [
    *(({}, *x) for x in PAGED_Q + WEIGHTS), ({}, dict(lam=None), -1), ({}, dict(lam=ODD4), -5), ({}, dict(s_lam=-1), -4),
    ({}, dict(out=FAKE), -4), ({}, dict(m=0), -4), ({}, dict(m=17), -4), ({}, dict(m=2), -4),  # weights of drafted tokens
    (dict(H=7), dict(Hq=28), -4), (dict(H=1), dict(Hq=8), -4)])
def test_diff_attend_rejects(store, kw, err):
    assert _diff_attend(_paged(**store), **kw) == err


PROMPT = [(dict(q=None), -1), (dict(k=None), -1), (dict(v=None), -1), (dict(out=None), -1), (dict(cu_q=None), -1),
          (dict(cu_k=None), -1), (dict(mode=1), -7), (dict(D=96), -4), (dict(Hq=30), -4), (dict(H=0), -4), (dict(S=0), -4),
          (dict(N=-1), -4), (dict(Nk=-1), -4), (dict(window=-1), -4), (dict(causal=0, window=5), -7), (dict(sk_n=1 << 23), -4),
          (dict(sv_n=-8), -4), (dict(q=ODD), -5), (dict(out=ODD), -5), (dict(sq_n=4100), -5), (dict(so_h=4), -5),
          (dict(out=FAKE), -4),                                      # q: it is read again behind the attention
          (dict(sq_n=1 << 23), -4), (dict(sq_n=-8), -4), (dict(sq_h=1 << 27), -4), (dict(T=-1), -4), (dict(sw_s=-1), -4),
          (dict(sw_h=-1), -4), (dict(weights=ODD4), -5), (dict(ws=None), -6), (dict(wsb=1000), -6), (dict(ws=ODD), -5)]


@pytest.mark.parametrize("kw,err", [(dict(weights=None), -1), *PROMPT])
def test_prompt_weights_rejects(kw, err):
    assert _prompt(**kw) == err


@pytest.mark.parametrize("kw,err", [*PROMPT, (dict(lam=None), -1), (dict(lam=ODD4), -5), (dict(s_lam=-1), -4),
                                    (dict(H=7, Hq=28), -4), (dict(H=1), -4)])
def test_diff_prompt_rejects(kw, err):
    assert _diff_prompt(**kw) == err


def test_nothing_to_do_is_no_error():
    assert _append(N=0) == 0 and _prompt(N=0) == 0 and _diff_prompt(N=0) == 0


def test_workspaces():
    lib = _lib.lib()
    evict = lib.iq_paged_evict_workspace_bytes
    for bad in ((0, 4, 8, 100, 20, 1), (3, 0, 8, 100, 20, 1), (3, 4, 8, 0, 0, 1), (3, 4, 8, 100, 101, 1), (3, 4, 8, 100, 20, 3)):
        assert evict(*bad) == 0
    # two numbers per (sequence, run of heads), and two lists of the rows that can come: those below keep - recent, or what
    # the table holds past keep
    assert evict(3, 4, 8, 100, 20, 1) == 3 * 8 * (2 + 2 * 80) * 4
    assert evict(3, 4, 8, 100, 20, 2) == 3 * 4 * (2 + 2 * 80) * 4
    assert evict(3, 4, 8, 250, 20, 1) == 3 * 8 * (2 + 2 * 6) * 4
    assert evict(3, 4, 8, 300, 20, 1) == 3 * 8 * 2 * 4
    plain, weights = lib.iq_paged_attention_workspace_bytes, lib.iq_paged_attention_weights_workspace_bytes
    assert weights(3, 4, 30, 8, 128) == 0
    assert weights(3, 4, 32, 8, 128) == plain(3, 4, 1, 32, 8, 128) + 3 * 32 * 8 + 3 * 32 * 256 * 4
    diff = lib.iq_diff_paged_attention_workspace_bytes
    assert diff(3, 4, 1, 32, 7, 128, 0) == diff(3, 4, 1, 32, 1, 128, 1) == 0
    assert diff(3, 4, 1, 32, 8, 128, 1) == diff(3, 4, 1, 32, 8, 128, 0) + 3 * 32 * 8 + 3 * 32 * 256 * 4
    prompt = lib.iq_prompt_weights_workspace_bytes
    assert prompt(3, 50, 50, 30, 8, 128) == prompt(3, 0, 50, 32, 8, 128) == prompt(3, 50, 50, 32, 8, 96) == 0
    assert prompt(3, 50, 50, 32, 8, 128) == 50 * 32 * 8
    assert prompt(4, 256, 64256, 32, 8, 128) > 256 * 32 * 8    # few rows over many keys: the parts of workgroups too


def test_cpu_tensors_raise():
    x, cu, lam = torch.zeros(4, 2, 64, dtype=torch.float16), torch.tensor([0, 4], dtype=torch.int32), torch.zeros(1)
    with pytest.raises(TypeError):
        ops.prompt_attention(x, x, x, cu, 1.0, weights=torch.zeros(1, 2, 4))
    with pytest.raises(TypeError):
        ops.diff_prompt_attention(x, x, x.view(4, 1, 128), cu, lam, 1.0)
