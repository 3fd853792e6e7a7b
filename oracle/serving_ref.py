"""References for the operators of many sequences (4-bit pages, packed prompts) -- TEST ORACLE ONLY.

Plain definitions on the CPU: the rotation in fp32 op by op, the quantizer through quant_ref, the page layout by index
arithmetic token by token (include/innerq_abi.h), attention in 64 bits with an error bound for the kernels.
"""
from __future__ import annotations

import numpy as np
import torch

from . import quant_ref as Q

PAGE, GROUP = 64, 32


def act_of(dtype) -> str:
    return "bf16" if dtype == torch.bfloat16 else "f16"


def rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """x [n, H, D] rotated by rows cos, sin [n, R/2]: pairs (d, d + R/2), fp32 ops, one rounding to x's dtype."""
    h = cos.shape[-1]
    y = x.float()
    a, b = y[..., :h], y[..., h:2 * h]
    c, s = cos[:, None], sin[:, None]
    return torch.cat([a * c - b * s, b * c + a * s, y[..., 2 * h:]], -1).to(x.dtype)


def quantize(x: torch.Tensor):
    """(codes int32, scale, zero) of x [n, H, D] by quant.py's quantize_channeldim_asym (numpy; NaN codes as 0)."""
    act = act_of(x.dtype)
    arr = x.numpy() if x.dtype == torch.float16 else x.float().numpy()
    with np.errstate(all="ignore"):
        c, s, z = Q.quantize_channeldim_asym(arr, GROUP, 4, act)
    c = np.where(c == Q.INT32_MIN, 0, c)
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a).astype(np.float32)).to(x.dtype)  # noqa: E731
    return torch.from_numpy(c.astype(np.int32)), t(s), t(z)


def value(codes, scale, zero) -> torch.Tensor:
    """c * s + z in fp32, rounded to the scales' dtype."""
    rep = lambda a: a.float().repeat_interleave(GROUP, -1)  # noqa: E731
    return (codes.float() * rep(scale) + rep(zero)).to(scale.dtype)


def page_rows(pages: torch.Tensor, page: int, row: int, D: int, dtype):
    """((codes, scale, zero) of K, the same of V), each [H, D] / [H, D/32], of one token of int32 pages [n, H, words]."""
    U, G = D // 8, D // GROUP
    w = pages[page].numpy().view(np.uint32)                       # [H, words]
    half = w.view(np.uint16)
    km, vc = PAGE * U, PAGE * (U + G)
    vm = vc + PAGE * U
    b, p = row // 32 * 4 + row % 16 // 4, row % 4 + row // 16 % 2 * 4
    out = []
    for role in "KV":
        words = np.stack([w[:, row * U + o] if role == "K" else w[:, vc + (b * U + o) * 8 + p] for o in range(U)], -1)
        codes = (words[..., None] >> np.arange(0, 32, 4, dtype=np.uint32)) & 15
        at = [(2 * (km + row * G + g), 2 * (km + row * G + g) + 1) if role == "K" else
              (2 * vm + (b * G + g) * 16 + p, 2 * vm + (b * G + g) * 16 + 8 + p) for g in range(G)]
        meta = [torch.from_numpy(np.stack([half[:, a[i]] for a in at], -1).astype(np.int16)).view(dtype) for i in (0, 1)]
        out.append((torch.from_numpy(codes.reshape(w.shape[0], D).astype(np.int32)), *meta))
    return out


def attention(q, k, v, scale: float, causal=True, window=0):
    """softmax(q k^T scale) v in 64 bits for one sequence: q [lq, Hq, D], k, v [lk, H, D].  A row's keys are those it
    sees: what the others hold plays no part.  Returns (out, bound): bound holds, value by value, how far a kernel may
    be that sums in fp32 and rounds the weights to q's dtype:

      every weight is rounded once (u = eps/2 of the dtype, relative; fp16 weights below 2^-14 by 2^-25 absolutely, the
      running maximum's weight being 1), the result once (u; 2^-25 absolutely for small fp16);
      a logit's fp32 dot product is off by D + 8 roundings of its products' absolute sum, and the exponential's argument
      and result by a few more, which moves weights by as much relatively: (D + 16) 2^-23 (1 + |logit|);
      sums over n weights, rescaled by at most n running maxima: (2 n + 64) 2^-24 each for numerator and sum.
    """
    lq, Hq, D = q.shape
    lk, H = k.shape[:2]
    r = Hq // H
    u = torch.finfo(q.dtype).eps / 2
    out = torch.zeros(lq, Hq, D, dtype=torch.float64)
    bound = torch.zeros_like(out)
    qd, kd, vd = q.double(), k.double(), v.double()
    for i in range(lq):
        end = i + lk - lq + 1 if causal else lk
        j0, j1 = max(0, end - window) if window else 0, min(max(end, 0), lk)
        if j1 <= j0:
            continue
        n = j1 - j0
        kk, vv = (x[j0:j1].repeat_interleave(r, 1) for x in (kd, vd))
        s = torch.einsum("hd,khd->hk", qd[i], kk) * scale
        p = torch.softmax(s, -1)
        out[i] = torch.einsum("hk,khd->hd", p, vv)
        size = (torch.einsum("hd,khd->hk", qd[i].abs(), kk.abs()) * abs(scale)).amax(-1)  # [Hq]
        a = torch.einsum("hk,khd->hd", p, vv.abs())
        rel = (D + 16) * 2.0 ** -23 * (1 + size)[:, None] + (2 * n + 64) * 2.0 ** -23
        b = (u + rel) * a + (u + rel) * out[i].abs() + 1e-30
        if q.dtype == torch.float16:
            b = b + n * 2.0 ** -25 * vv.abs().amax(0) + 2.0 ** -25
        bound[i] = 1.01 * b
    return out, bound
