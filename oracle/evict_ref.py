"""References for caches that drop tokens by the attention weight they have gathered -- TEST ORACLE ONLY.

Plain definitions on the CPU: which tokens a head keeps and where they go, the rows of pages as raw words, the weights
that attention gives its keys in 64 bits with an error bound for the kernels.
"""
from __future__ import annotations

import numpy as np
import torch

PAGE, GROUP = 64, 32


def kept(w, keep: int, recent: int, sinks: int):
    """The old places [keep] of the tokens that a run of heads keeps, by new place; w: fp32 [n] (summed over the run)."""
    w = np.asarray(w, dtype=np.float32)
    n = len(w)
    if n <= keep:
        return list(range(n))
    old, base = n - recent, keep - recent
    rank = lambda i: (0, 0.0) if i < sinks or np.isnan(w[i]) else (1, -float(w[i]))  # noqa: E731
    best = sorted(range(old), key=lambda i: (*rank(i), i))[:base]  # equal weights (-0 and 0 too): the first
    stay, come = set(best), iter(sorted(i for i in best if i >= base))
    return [i if i in stay else next(come) for i in range(base)] + list(range(old, n))


def token_words(pages, table_row, n: int, D: int):
    """[H, n, *] uint32: every word and half word of the tokens 0 .. n-1 of one sequence (pages int32 [N, H, words])."""
    U, G = D // 8, D // GROUP
    km, vc = PAGE * U, PAGE * (U + G)
    vm = vc + PAGE * U
    w = pages.numpy().view(np.uint32)
    half = w.view(np.uint16)
    t = np.arange(n)
    page, row = np.asarray(table_row)[t // PAGE].astype(np.int64), t % PAGE
    b, p = row // 32 * 4 + row % 16 // 4, row % 4 + row // 16 % 2 * 4
    o, g = np.arange(U), np.arange(G)
    H = w.shape[1]
    pick = lambda x, at: np.stack([x[page[:, None], h, at] for h in range(H)])  # noqa: E731
    vs = 2 * vm + (b[:, None] * G + g) * 16 + p[:, None]
    return np.concatenate([pick(w, row[:, None] * U + o), pick(w, km + row[:, None] * G + g),
                           pick(w, vc + (b[:, None] * U + o) * 8 + p[:, None]), pick(half, vs).astype(np.uint32),
                           pick(half, vs + 8).astype(np.uint32)], -1)


def weights(q, k, scale: float, causal=True, window=0):
    """What attention of q [lq, Hq, D] over k [lk, H, D] gives each key: (sum over rows and a group's heads of the softmax
    weights [H, lk], bound), in 64 bits.  The bound, for a kernel whose logits, statistics and sums are fp32, is a coarse one
    (gathered() has one that tells rounded weights from unrounded ones): every weight by (D + 16) 2^-23 (1 + the largest of
    its row's logits' absolute sums of products) relatively, which is more than its own logit and its row's sum are off by; its
    row's sum over n keys, rescaled by at most n running maxima, by (2 n + 64) 2^-23; the sum over the rows by one rounding of
    2^-24 each."""
    lq, Hq, D = q.shape
    lk, H = k.shape[:2]
    r = Hq // H
    out = torch.zeros(H, lk, dtype=torch.float64)
    bound = torch.zeros_like(out)
    qd, kd = q.double(), k.double()
    for i in range(lq):
        end = i + lk - lq + 1 if causal else lk
        j0, j1 = max(0, end - window) if window else 0, min(max(end, 0), lk)
        if j1 <= j0:
            continue
        kk = kd[j0:j1].repeat_interleave(r, 1)
        s = torch.einsum("hd,khd->hk", qd[i], kk) * scale
        size = (torch.einsum("hd,khd->hk", qd[i].abs(), kk.abs()) * abs(scale)).amax(-1, keepdim=True)
        p = torch.softmax(s, -1)
        rel = (D + 16) * 2.0 ** -23 * (1 + size) + (2 * (j1 - j0) + 64) * 2.0 ** -23
        out[:, j0:j1] += p.view(H, r, -1).sum(1)
        bound[:, j0:j1] += (p * rel).view(H, r, -1).sum(1)
    return out, 1.01 * (bound + (lq * r + 2) * 2.0 ** -24 * out) + 1e-30


def gathered(q, k, scale: float, causal=True, window=0):
    """weights() of the same arguments, on q's device, with the bound that follows from what the kernels do, small enough
    that weights rounded to 16 bits break it.  Relatively, with u = 2^-24:

      a logit: its products are exact, their sum in fp32 is off by D roundings (2 u each: the matrix unit may cut) of the
      products' absolute sum, the factor c = RN(scale log2 e), the multiply-add and what is subtracted by 8 more; the
      exponential by 16 u:                                 e_j = 2 u ((D + 8) sum |q k| scale + 8), which moves weight j by e_j
      the row's sum: of weights that are off by e_j:                                            sum_j p_j e_j
      and of its own roundings.  n keys are taken in tiles of 32 at least, each of which adds once to the sum and may change
      the base: 2 u for the exponential of the change, u for the product, u for the change itself times what it is, and all
      changes together are at most twice the row's largest logit; within a tile, between lanes, waves and shares fewer than
      64 sums:                                             u (6 (n / 32 + 1) + 2 max |logit| + 64)
      the sum over R rows and heads: in lanes of 32, then between lanes, shares and turns:       u (R / 32 + 64)"""
    (lq, Hq, D), (lk, H) = q.shape, k.shape[:2]
    u = 2.0 ** -24
    out = torch.zeros(H, lk, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    if not lq or not lk:
        return out, bound
    i, j = torch.arange(lq, device=q.device)[:, None], torch.arange(lk, device=q.device)[None]
    end = i + (lk - lq + 1) if causal else torch.full_like(i, lk)
    seen = (j < end) & ((j >= end - window) if window else (j >= 0))
    n = seen.sum(1, keepdim=True)
    for g in range(Hq):
        h = g // (Hq // H)
        x, y = q[:, g].double().contiguous(), k[:, h].double().t().contiguous()
        s = torch.where(seen, (x @ y) * scale, -torch.inf)
        size = torch.where(seen, (x.abs() @ y.abs()) * abs(scale), 0.0)
        p = torch.where(seen, (s - s.amax(1, keepdim=True).clamp(min=-1e300)).exp(), 0.0)
        p = p / p.sum(1, keepdim=True).clamp(min=1e-300)
        e = 2 * u * ((D + 8) * size + 8)
        rel = e + (p * e).sum(1, keepdim=True) + u * (6 * (n / 32 + 1) + 2 * size.amax(1, keepdim=True) + 64)
        out[h] += p.sum(0)
        bound[h] += (p * rel).sum(0)
    return out, 1.01 * (bound + u * (lq * (Hq // H) / 32 + 64) * out) + 1e-30
