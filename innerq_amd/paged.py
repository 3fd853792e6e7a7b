"""A 4-bit KV cache in pages, shared by many sequences of different lengths.

``PagedStore`` holds a pool of pages, each of 64 tokens of every KV head, K and V in 4-bit asymmetric groups of 32
along head_dim (the codes, scales and zero points of quant.quantize_channeldim_asym of each token; layout:
include/innerq_abi.h).  Which pages are a sequence's is the caller's ``table``, how many tokens it holds the caller's
``lens``, both int32 device tensors that the kernels read: a captured call follows their values.

* ``append`` quantizes the new tokens of every sequence into its pages, rotating keys (and the step's queries) on
  the way;
* ``attend`` is decode attention of one or a few new tokens per sequence over its pages;
* ``read`` gives back the values of some tokens, dense.

A prompt attends with ops.prompt_attention over its dense K and V; a later chunk of it over what ``read`` gives.

    store = PagedStore(n_pages, Hkv, 128, "cuda:0")
    q = store.append(k, v, table, lens, cu_seqlens, cos=cos, sin=sin, q=q)    # prompts: tokens lens[s] ..
    ...
    q = store.append(k, v, table, lens, cos=cos, sin=sin, q=q)                # a step: one token per sequence
    out = store.attend(q, table, lens + 1, scale)

Inference only: tensors that autograd follows are refused, outputs too.  Device tensors only; there is no CPU path.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch.autograd import forward_ad

from . import _lib, ops
from ._lib import call

PAGE_TOKENS = 64
GROUP = 32
MAX_NEW = 16  # new tokens per sequence of an attend()


def _no_grad(*tensors) -> None:
    if ops.autograd_follows(*tensors):
        raise NotImplementedError("paged KV calls have no backward: call them under torch.no_grad()")


def _rows(t: torch.Tensor, name: str, shape: tuple, dtype, device) -> torch.Tensor:
    """``t`` as the kernels read it: of this shape, dtype and device, D contiguous, rows 16-byte aligned (copied if not)."""
    ops.require_device(t, name, dtype)
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the store on {device}")
    ops.check_out(t.shape, shape, name)
    return ops.readable_rows(t)


def _out_rows(t: torch.Tensor, name: str, shape: tuple, dtype, device) -> torch.Tensor:
    ops.require_device(t, name, dtype)
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the store on {device}")
    ops.check_out(t.shape, shape, name)
    if not ops.writable_rows(t):
        raise ValueError(f"{name} needs a contiguous head_dim and rows of their own on 16-byte boundaries")
    return t


class PagedStore:
    """``n_pages`` pages of H KV heads of head_dim D (64 or 128) for fp16 or bf16 activations."""

    def __init__(self, n_pages: int, H: int, D: int, device, dtype=torch.float16):
        ops.act_flag(dtype)
        if n_pages <= 0:
            raise ValueError(f"a store needs at least one page, got {n_pages}")
        device = torch.device(device)
        if device.type != "cuda":
            raise TypeError("PagedStore lives on a HIP device (innerq_amd has no CPU path)")
        pages = torch.empty(n_pages, H, self.page_bytes(H, D) // (4 * H), dtype=torch.int32, device=device)
        self._set(pages, D, dtype)

    @classmethod
    def over(cls, pages: torch.Tensor, D: int, dtype=torch.float16) -> "PagedStore":
        """A store over existing pages: int32 [n_pages, H, words], contiguous (as ``store.pages``)."""
        ops.require_device(pages, "pages", torch.int32)
        ops.act_flag(dtype)
        if pages.dim() != 3 or not pages.is_contiguous() or pages.shape[0] == 0:
            raise ValueError(f"pages must be a contiguous [n_pages, H, words] tensor, got {tuple(pages.shape)}")
        words = cls.page_bytes(pages.shape[1], D) // (4 * pages.shape[1])
        ops.check_out(pages.shape, (pages.shape[0], pages.shape[1], words), "pages")
        if pages.data_ptr() % 16:
            raise ValueError("pages must start on a 16-byte boundary")
        st = cls.__new__(cls)
        st._set(pages, D, dtype)
        return st

    def _set(self, pages, D, dtype) -> None:
        self.pages, self.D, self.dtype = pages, D, dtype
        self.n_pages, self.H = pages.shape[0], pages.shape[1]
        self.device = pages.device
        self.status = torch.zeros(1, dtype=torch.int32, device=pages.device)

    @staticmethod
    def page_bytes(H: int, D: int) -> int:
        """Bytes of one page: 64 tokens of H heads, K and V."""
        n = ctypes.c_int64()
        call("iq_page_bytes", H, D, ctypes.byref(n))
        return n.value

    def check(self) -> None:
        """Raises RuntimeError if a call since the last check needed a page outside the pool or a token past the
        table (takes the status word on the current stream: waits for it, and for calls that it waits for; what a call
        on another stream tells meanwhile is kept for the next check)."""
        with ops.on_device(self.device):
            taken = torch.empty(1, dtype=torch.int32, device=self.device)
            call("iq_paged_take_status", ops._p(self.status), ops._p(taken), ops._stream(self.device))
        bad = int(taken.item())
        if bad:
            why = [w for b, w in ((1, "a table entry outside the pool"),
                                  (2, "a token past the table's pages or the rotation's rows, or a negative length"))
                   if bad & b]
            raise RuntimeError("PagedStore: a call met " + " and ".join(why))

    def _args(self, table: torch.Tensor, lens: torch.Tensor) -> "_lib.iq_paged":
        for t, name, dim in ((table, "table", 2), (lens, "lens", 1)):
            ops.require_device(t, name, torch.int32)
            if t.dim() != dim or t.device != self.device:
                raise ValueError(f"{name} must be a {dim}-d int32 tensor on {self.device}, got {tuple(t.shape)} on "
                                 f"{t.device}")
        S, P = table.shape
        if lens.shape[0] != S or not S or not P:
            raise ValueError(f"table [S, P] and lens [S] do not fit: {tuple(table.shape)}, {tuple(lens.shape)}")
        if (P > 1 and table.stride(1) != 1) or not lens.is_contiguous():
            raise ValueError("table rows and lens must be contiguous")
        p = _lib.iq_paged()
        p.pages, p.n_pages = self.pages.data_ptr(), self.n_pages
        p.table, p.s_table, p.lens, p.status = table.data_ptr(), table.stride(0), lens.data_ptr(), self.status.data_ptr()
        p.S, p.P, p.H, p.D, p.mode = S, P, self.H, self.D, ops.act_flag(self.dtype)
        return p

    def _cu(self, cu: Optional[torch.Tensor], S: int, N: int) -> Optional[torch.Tensor]:
        if cu is None:
            if N != S:
                raise ValueError(f"without cu_seqlens there is one token per sequence: {N} tokens, {S} sequences")
            return None
        return ops.check_cu(cu, "cu_seqlens", S, self.device)

    def append(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, lens: torch.Tensor,
               cu_seqlens: Optional[torch.Tensor] = None, cos: Optional[torch.Tensor] = None,
               sin: Optional[torch.Tensor] = None, q: Optional[torch.Tensor] = None,
               q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
        """Appends k and v [N, H, D]: rows cu_seqlens[s] .. cu_seqlens[s+1] (int32 [S+1]; None: one row per sequence)
        become tokens lens[s], lens[s] + 1, ... of sequence s (lens: tokens held before the call, which it leaves as
        they are).  cos, sin: fp32 [positions, R/2]; the first R dims of each key and query are rotated by their
        token's row (pairs d, d + R/2).  Returns q [N, Hq, D] rotated, written to ``q_out`` (q itself, or memory that no
        other argument uses) or a new tensor; None without q.  Rows outside the sequences are neither appended nor
        written to q_out.  A token that cannot be appended (check()) has NaN queries, and one that only the rotation has
        no row for NaN in its page, so that read() and attend() give NaN.  Sequences that append must not share the
        pages they append to."""
        fast = ops._native(k) if forward_ad._current_level < 0 else None
        if fast is not None:
            r = fast.paged_append(self.pages, self.D, self.dtype, self.status, table, lens, k, v, cu_seqlens, cos, sin, q,
                                  q_out)
            if r is not None:
                return r[0]
        _no_grad(k, v, q, cos, sin, q_out)
        p = self._args(table, lens)
        if k.dim() != 3:
            raise ValueError(f"append: k must be [N, H, D], got {tuple(k.shape)}")
        N, want = k.shape[0], (k.shape[0], self.H, self.D)
        k = _rows(k, "k", want, self.dtype, self.device)
        v = _rows(v, "v", want, self.dtype, self.device)
        cu = self._cu(cu_seqlens, p.S, N)
        if (cos is None) != (sin is None):
            raise ValueError("append: cos and sin come together")
        n_pos = R = 0
        if cos is not None:
            for t, name in ((cos, "cos"), (sin, "sin")):
                ops.require_device(t, name, torch.float32)
                if t.dim() != 2 or t.shape != cos.shape or t.device != self.device or not t.is_contiguous() \
                        or t.data_ptr() % 16:
                    raise ValueError(f"append: {name} must be a contiguous fp32 [positions, R/2] tensor on {self.device}")
            n_pos, R = cos.shape[0], 2 * cos.shape[1]
            if R % 16 or not 0 < R <= self.D or not n_pos:
                raise ValueError(f"append: the rotation covers R dims, a multiple of 16 up to {self.D}, got {R} "
                                 f"({n_pos} positions)")
        Hq, qs, qos = 0, (0, 0), (0, 0)
        if q is not None:
            if q.dim() != 3 or q.shape[1] == 0:
                raise ValueError(f"append: q must be [N, Hq, D], got {tuple(q.shape)}")
            Hq = q.shape[1]
            q = _rows(q, "q", (N, Hq, self.D), self.dtype, self.device)
            if q_out is None:
                q_out = torch.empty(N, Hq, self.D, dtype=self.dtype, device=self.device)
            else:
                _out_rows(q_out, "q_out", (N, Hq, self.D), self.dtype, self.device)
            qs, qos = q.stride(), q_out.stride()
        elif q_out is not None:
            raise ValueError("append: q_out without q")
        with ops.on_device(self.device):
            call("iq_paged_append", ctypes.byref(p), ops._p(cu), N, ops._p(k), k.stride(0), k.stride(1), ops._p(v),
                 v.stride(0), v.stride(1), ops._p(cos), ops._p(sin), n_pos, R, ops._p(q), qs[0], qs[1], Hq,
                 ops._p(q_out), qos[0], qos[1], ops._stream(self.device))
        return q_out

    def read(self, table: torch.Tensor, lens: torch.Tensor, cu_seqlens: Optional[torch.Tensor], n: int,
             k_out: Optional[torch.Tensor] = None, v_out: Optional[torch.Tensor] = None):
        """K and V [n, H, D] of tokens lens[s] + i of every sequence, at rows cu_seqlens[s] + i (as ``append`` takes
        them; n rows in all), in ``k_out`` and ``v_out`` (memory of their own) or new tensors.  Rows outside the
        sequences are not written."""
        fast = ops._native(self.pages)
        if fast is not None and k_out is None and v_out is None:
            r = fast.paged_read(self.pages, self.D, self.dtype, self.status, table, lens, cu_seqlens, n)
            if r is not None:
                return r
        _no_grad(k_out, v_out)
        p = self._args(table, lens)
        cu = self._cu(cu_seqlens, p.S, n)
        want = (n, self.H, self.D)
        outs = []
        for t, name in ((k_out, "k_out"), (v_out, "v_out")):
            outs.append(torch.empty(want, dtype=self.dtype, device=self.device) if t is None else
                        _out_rows(t, name, want, self.dtype, self.device))
        k, v = outs
        if not ops.apart(k, v):
            raise ValueError("read: k_out and v_out share memory")
        with ops.on_device(self.device):
            call("iq_paged_read", ctypes.byref(p), ops._p(cu), n, ops._p(k), k.stride(0), k.stride(1), ops._p(v),
                 v.stride(0), v.stride(1), ops._stream(self.device))
        return k, v

    def attend(self, q: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, scale: float,
               window: Optional[int] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """softmax(q K^T * scale) V over each sequence's first lens[s] tokens, the new ones among them.  q [S, Hq, D]
        (one new token) or [S, m, Hq, D] (m <= 16: token j sees all but the m - 1 - j after it); window: only the last
        ``window`` tokens up to its own.  The table's width plans the work: pass ``table[:, :pages that the longest
        sequence needs]`` where tables are wider than any sequence.  Rows that see no token, or only tokens whose logits
        are minus infinity, are 0.  Returns ``out`` (q itself, or memory that no other argument uses) or a new tensor of
        q's shape."""
        fast = ops._native(q) if forward_ad._current_level < 0 else None
        if fast is not None:
            r = fast.paged_attend(self.pages, self.D, self.dtype, self.status, table, lens, q, scale, window, out)
            if r is not None:
                return r
        _no_grad(q, out)
        p = self._args(table, lens)
        if q.dim() not in (3, 4) or q.shape[0] != p.S:
            raise ValueError(f"attend: q must be [S, Hq, D] or [S, m, Hq, D] with S = {p.S}, got {tuple(q.shape)}")
        m, Hq = (1, q.shape[1]) if q.dim() == 3 else (q.shape[1], q.shape[2])
        if not 0 < m <= MAX_NEW:
            raise ValueError(f"attend: 1 to {MAX_NEW} new tokens per sequence, got {m} (more: read() and "
                             "ops.prompt_attention)")
        ops.check_gqa(Hq, self.H)
        if not Hq:
            raise ValueError("attend: q has no heads")
        if window is not None and not 0 < window < 2 ** 31:
            raise ValueError(f"attend: window must be positive, got {window}")
        q = _rows(q, "q", (*q.shape[:-1], self.D), self.dtype, self.device)
        if out is None:
            out = torch.empty(q.shape, dtype=self.dtype, device=self.device)
        else:
            _out_rows(out, "out", tuple(q.shape), self.dtype, self.device)
        qs, os = (t.stride() if m > 1 or t.dim() == 4 else (t.stride(0), 0, t.stride(1)) for t in (q, out))
        nbytes = _lib.lib().iq_paged_attention_workspace_bytes(p.S, p.P, m, Hq, self.H, self.D)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device) if nbytes else None
        with ops.on_device(self.device):
            call("iq_paged_attention", ctypes.byref(p), ops._p(q), qs[0], qs[1], qs[2], m, Hq, float(scale), window or 0,
                 ops._p(out), os[0], os[1], os[2], ops._p(ws), nbytes, ops._stream(self.device))
        return out
