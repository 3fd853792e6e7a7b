"""The C ABI of pages and packed prompts refuses bad arguments on the host, before any launch (no GPU here: each case
has one invalid argument), sizes are what the layout says, and CPU tensors raise."""
import ctypes

import pytest
import torch

from innerq_amd import _lib, ops, paged

FAKE = ctypes.c_void_p(0x1000)  # never dereferenced
ODD = ctypes.c_void_p(0x1008)


def _paged(**kw):
    a = dict(pages=0x1000, n_pages=8, table=0x1000, s_table=4, lens=0x1000, status=0x1000, S=3, P=4, H=8, D=128, mode=0)
    a.update(kw)
    p = _lib.iq_paged()
    for name, x in a.items():
        setattr(p, name, x)
    return ctypes.byref(p)


BAD_STORES = [(dict(pages=None), -1), (dict(table=None), -1), (dict(lens=None), -1), (dict(status=None), -1),
              (dict(mode=1), -7), (dict(mode=2), -7), (dict(D=96), -4), (dict(D=256), -4), (dict(H=0), -4), (dict(S=0), -4),
              (dict(P=0), -4), (dict(n_pages=0), -4), (dict(n_pages=1 << 31), -4), (dict(P=1 << 26), -4),
              (dict(s_table=-1), -4), (dict(pages=0x1008), -5), (dict(table=0x1002), -5), (dict(lens=0x1002), -5)]


def _append(store=None, **kw):
    a = dict(cu=FAKE, N=5, k=FAKE, sk_n=1024, sk_h=128, v=FAKE, sv_n=1024, sv_h=128, cos=FAKE, sin=FAKE, n_pos=100, R=128,
             q=FAKE, sq_n=4096, sq_h=128, Hq=32, q_out=FAKE, so_n=4096, so_h=128, stream=None)
    a.update(kw)
    return _lib.lib().iq_paged_append(store or _paged(), *a.values())


def _read(store=None, **kw):
    a = dict(cu=FAKE, N=5, k=FAKE, sk_n=1024, sk_h=128, v=FAKE, sv_n=1024, sv_h=128, stream=None)
    a.update(kw)
    return _lib.lib().iq_paged_read(store or _paged(), *a.values())


def _attend(store=None, **kw):
    a = dict(q=FAKE, sq_s=4096, sq_m=4096, sq_h=128, m=1, Hq=32, scale=1.0, window=0, out=FAKE, so_s=4096, so_m=4096,
             so_h=128, ws=FAKE, wsb=1 << 40, stream=None)
    a.update(kw)
    return _lib.lib().iq_paged_attention(store or _paged(), *a.values())


def _prompt(**kw):
    a = dict(q=FAKE, sq_n=4096, sq_h=128, k=FAKE, sk_n=1024, sk_h=128, v=FAKE, sv_n=1024, sv_h=128, cu_q=FAKE, cu_k=FAKE,
             S=3, N=50, Nk=50, Hq=32, H=8, D=128, mode=0, scale=1.0, causal=1, window=0, out=FAKE, so_n=4096, so_h=128,
             stream=None)
    a.update(kw)
    return _lib.lib().iq_prompt_attention(*a.values())


@pytest.mark.parametrize("kw,err", BAD_STORES)
@pytest.mark.parametrize("fn", [_append, _read, _attend])
def test_bad_stores(fn, kw, err):
    assert fn(_paged(**kw)) == err


def test_null_store():
    lib = _lib.lib()
    assert lib.iq_paged_read(None, FAKE, 5, FAKE, 1024, 128, FAKE, 1024, 128, None) == -1


@pytest.mark.parametrize("kw,err", [
    (dict(k=None), -1), (dict(v=None), -1), (dict(q_out=None), -1), (dict(cos=None), -1), (dict(sin=None), -1),
    (dict(N=-1), -4), (dict(cu=None, N=5), -4), (dict(Hq=0), -4), (dict(Hq=5000), -4), (dict(R=0), -4), (dict(R=136), -4),
    (dict(R=24), -4), (dict(R=144), -4), (dict(n_pos=0), -4), (dict(k=ODD), -5), (dict(v=ODD), -5), (dict(q=ODD), -5),
    (dict(q_out=ODD), -5), (dict(cos=ODD), -5), (dict(sk_n=1020), -5), (dict(sv_h=100), -5), (dict(sq_n=4097), -5),
    (dict(so_h=129), -5)])
def test_append_rejects(kw, err):
    assert _append(**kw) == err


@pytest.mark.parametrize("kw,err", [
    (dict(k=None), -1), (dict(v=None), -1), (dict(N=-1), -4), (dict(cu=None, N=4), -4), (dict(k=ODD), -5),
    (dict(sv_n=1023), -5)])
def test_read_rejects(kw, err):
    assert _read(**kw) == err


@pytest.mark.parametrize("store,kw,err", [
    ({}, dict(q=None), -1), ({}, dict(out=None), -1), ({}, dict(m=0), -4), ({}, dict(m=17), -4), ({}, dict(Hq=0), -4),
    ({}, dict(Hq=12), -4), ({}, dict(window=-1), -4), ({}, dict(q=ODD), -5), ({}, dict(sq_h=4), -5), ({}, dict(so_s=12), -5),
    (dict(P=4000, S=100000, H=8), dict(), -4),                       # more than 2^31 pages to read
    (dict(P=300, s_table=300), dict(ws=None), -6), (dict(P=300, s_table=300), dict(wsb=64), -6),
    (dict(P=300, s_table=300), dict(ws=ODD), -5)])
def test_attend_rejects(store, kw, err):
    assert _attend(_paged(**store), **kw) == err


@pytest.mark.parametrize("kw,err", [
    (dict(q=None), -1), (dict(k=None), -1), (dict(v=None), -1), (dict(out=None), -1), (dict(cu_q=None), -1),
    (dict(cu_k=None), -1), (dict(mode=1), -7), (dict(mode=0x102), -7), (dict(D=96), -4), (dict(Hq=30), -4), (dict(H=0), -4),
    (dict(S=0), -4), (dict(N=-1), -4), (dict(Nk=-1), -4), (dict(window=-1), -4), (dict(causal=0, window=5), -7),
    (dict(sk_n=1 << 23), -4), (dict(sv_n=-8), -4), (dict(q=ODD), -5), (dict(out=ODD), -5), (dict(sq_n=4100), -5),
    (dict(so_h=4), -5), (dict(N=2 ** 31 - 1, Hq=4096), -4)])
def test_prompt_rejects(kw, err):
    assert _prompt(**kw) == err


def test_nothing_to_do_is_no_error():
    assert _append(N=0) == 0 and _read(N=0) == 0 and _prompt(N=0) == 0


def test_sizes():
    assert paged.PagedStore.page_bytes(8, 128) == 64 * 8 * 2 * (64 + 16)
    assert paged.PagedStore.page_bytes(1, 64) == 64 * 2 * (32 + 8)
    with pytest.raises(_lib.IQError):
        paged.PagedStore.page_bytes(0, 128)
    with pytest.raises(_lib.IQError):
        paged.PagedStore.page_bytes(8, 96)
    ws = _lib.lib().iq_paged_attention_workspace_bytes
    assert ws(0, 4, 1, 32, 8, 128) == 0 and ws(8, 512, 1, 30, 8, 128) == 0
    assert ws(8, 512, 1, 32, 8, 128) == ws(64, 100, 4, 32, 8, 128) > 0  # by the grid, not by the lengths


def test_cpu_tensors_raise():
    x = torch.zeros(4, 2, 64, dtype=torch.float16)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(TypeError):
        ops.prompt_attention(x, x, x, cu, 1.0)
    with pytest.raises(TypeError):
        paged.PagedStore(4, 2, 64, "cpu")
    with pytest.raises(TypeError):
        paged.PagedStore.over(torch.zeros(4, 2, 640, dtype=torch.int32), 64)
