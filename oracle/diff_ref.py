"""References for differential attention -- TEST ORACLE ONLY.  Two maps in 64 bits, with an error bound for the kernels."""
from __future__ import annotations

import torch

from . import serving_ref as R


def attention(q, k, v, lam, scale: float, causal=True, window=0):
    """(softmax(q_2j k_2g^T scale) - lam_j softmax(q_2j+1 k_2g+1^T scale)) v_g in 64 bits for one sequence: q [lq, Hq, D],
    k [lk, H, D], v [lk, H/2, 2 D].  Returns (out [lq, Hq/2, 2 D], bound): the maps' own bounds (serving_ref.attention: each
    weight rounded once to q's dtype, its result's rounding u |map| included, of which this operator has none: it rounds the
    difference) added up, and the difference's rounding (u = eps/2; 2^-25 absolutely for small fp16)."""
    lq, Hq, D = q.shape
    H = k.shape[1]
    u = torch.finfo(q.dtype).eps / 2
    parts = []
    for i in (0, 1):
        halves = [R.attention(q[:, i::2], k[:, i::2], x, scale, causal, window) for x in (v[..., :D], v[..., D:])]
        parts.append([torch.cat(x, -1) for x in zip(*halves)])
    f = lam.double()[None, :, None]
    (a, ba), (b, bb) = parts
    out = a - f * b
    bound = ba + f.abs() * bb + (u + 2.0 ** -22) * out.abs() + 2.0 ** -22 * (f * b).abs() + 2.0 ** -25
    return out, 1.01 * bound
