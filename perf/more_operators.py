"""Operators beside those of perf/operators.py: caches that drop what is not attended to, and differential attention.

Five kinds of call (``kind``):

* ``weigh_prompt``  ops.prompt_attention(weights=): causal attention over packed prompts that also adds up, key by key,
  the weights that the prompt's rows gave it;
* ``weigh_attend``  paged.PagedStore.attend(weights=): the same for a step's new token over its 4-bit pages;
* ``evict``         paged.PagedStore.evict: of each sequence and KV head, the tokens of most weight (and the first and the
  last ones) stay, in the sequence's first pages; what is kept is read back (PagedStore.read);
* ``diff_prompt``   ops.diff_prompt_attention: (softmax(q1 k1) - lam softmax(q2 k2)) v over packed prompts;
* ``diff_attend``   paged.PagedStore.diff_attend: the same for one token (or a few drafted ones) over 4-bit pages.

Heads: ``Hq`` query and ``Hkv`` key heads of ``D``.  For the differential kinds two neighbouring heads are the two maps of
one output head, and V's heads are 2 D wide (two neighbouring heads of a page).

A page holds 64 tokens of every KV head.  One (page, head) is one run of 32-bit words,

    K codes [64 tokens][D/8]   K scales/zeros [64][D/32]   V codes [8 blocks][D/8][8 tokens]   V scales/zeros [8][D/32][s x 8, z x 8]

a word being 8 codes of one token (code i at bits 4i).  Token t of a page is token t%4 + 4*(t//16%2) of V block
t//32*4 + t%16//4.  A code c stands for c*s + z, rounded to the cache's type.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
DT = {"fp16": torch.float16, "bf16": torch.bfloat16}
PAGE, GROUP = 64, 32
# (query, KV) elements of the largest listed prompt and tokens of its largest cache: no drawn case is larger
MOST_PAIRS, MOST_HELD = 32 * 8192 * 8192, 8 * 32768


def listed():
    return [
        # one user's short question whose cache will be cut down later: launches and latency
        dict(name="weigh_prompt_one_short", kind="weigh_prompt", seqs=1, longest=77, mix=0, past=0, window=0, Hq=32, Hkv=8,
             D=128, dtype="fp16"),
        # a step's prompts of different lengths, packed
        dict(name="weigh_prompt_packed", kind="weigh_prompt", seqs=16, longest=2000, mix=3, past=0, window=0, Hq=32, Hkv=8,
             D=128, dtype="bf16"),
        # the last rows of four long prompts choose what their caches keep
        dict(name="weigh_prompt_last_rows", kind="weigh_prompt", seqs=4, longest=64, mix=0, past=16000, window=0, Hq=32,
             Hkv=8, D=128, dtype="fp16"),
        # a decode step of a batch of 8 at 32k tokens: the cache's stream, and its logits once more
        dict(name="weigh_attend_batch", kind="weigh_attend", seqs=8, longest=32768, mix=0, window=0, Hq=32, Hkv=8, D=128,
             dtype="fp16"),
        # a serving batch of very different lengths, bf16
        dict(name="weigh_attend_ragged", kind="weigh_attend", seqs=48, longest=16001, mix=7, window=0, Hq=32, Hkv=8, D=128,
             dtype="bf16"),
        # a batch at its budget, a page over it: each sequence drops 64 tokens
        dict(name="evict_step", kind="evict", seqs=32, longest=2112, mix=0, keep=2048, recent=256, sinks=0, Hkv=8, D=128,
             dtype="fp16"),
        # long prompts cut down to a budget
        dict(name="evict_prompts", kind="evict", seqs=8, longest=32768, mix=0, keep=2048, recent=512, sinks=4, Hkv=8, D=128,
             dtype="bf16"),
        # packed prompts of a differential model
        dict(name="diff_prompt_packed", kind="diff_prompt", seqs=16, longest=2000, mix=3, past=0, window=0, Hq=32, Hkv=8,
             D=64, dtype="bf16"),
        # a long document in one call: the matrix cores' work
        dict(name="diff_prompt_long", kind="diff_prompt", seqs=1, longest=8192, mix=0, past=0, window=0, Hq=32, Hkv=8,
             D=128, dtype="fp16"),
        # one user, a short chat: latency
        dict(name="diff_attend_one_short", kind="diff_attend", seqs=1, longest=1000, mix=0, new=1, window=0, Hq=32, Hkv=8,
             D=64, dtype="bf16"),
        # a batch of 8 at 32k tokens: the cache's stream
        dict(name="diff_attend_batch", kind="diff_attend", seqs=8, longest=32768, mix=0, new=1, window=0, Hq=32, Hkv=8,
             D=64, dtype="fp16"),
        # three drafted tokens per sequence checked at once, lengths of all kinds, bf16
        dict(name="diff_attend_drafts", kind="diff_attend", seqs=24, longest=6001, mix=2, new=3, window=0, Hq=32, Hkv=8,
             D=128, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["weigh_prompt", "weigh_attend", "evict", "diff_prompt", "diff_attend"])
    Hq, Hkv = rng.choice([(32, 8), (32, 8), (8, 8), (16, 2), (32, 4), (12, 4)])
    c = dict(kind=kind, mix=rng.choice([0, rng.randrange(1, 1000)]), Hq=Hq, Hkv=Hkv, D=rng.choice([64, 128]),
             dtype=rng.choice(["fp16", "bf16"]))
    if kind.endswith("prompt"):
        c["seqs"] = _log_int(rng, 1, 48)
        c["past"] = rng.choice([0, 0, _log_int(rng, 1, 8000)])
        c["longest"] = _log_int(rng, 1, 8200)
        while c["seqs"] * Hq * c["longest"] * (c["longest"] + c["past"]) > MOST_PAIRS // 2:
            c["longest"] = c["longest"] * 3 // 4
        c["window"] = rng.choice([0, 0, _log_int(rng, 1, 8000)])
        return c
    c["seqs"] = _log_int(rng, 1, 128)
    c["longest"] = _log_int(rng, 1, MOST_HELD // c["seqs"])
    if kind == "evict":
        del c["Hq"]
        c["keep"] = _log_int(rng, 1, c["longest"])
        c["recent"] = rng.choice([0, rng.randrange(c["keep"] + 1) // 2])
        c["sinks"] = rng.choice([0, min(4, c["keep"] - c["recent"])])
    else:
        c["window"] = rng.choice([0, 0, _log_int(rng, 1, 8000)])
        if kind == "diff_attend":
            c["new"] = min(rng.choice([1, 1, rng.randrange(1, 9)]), c["longest"])
    return c


def _lengths(c):
    """Tokens of each sequence: all ``longest``, or (mix > 0) a long one and others down to a hundredth of it."""
    n = c["seqs"]
    if not c["mix"]:
        return [c["longest"]] * n
    r = random.Random(c["mix"])
    out = [max(1, int(c["longest"] * r.uniform(0.1, 1) ** 2)) for _ in range(n)]
    out[r.randrange(n)] = c["longest"]
    return out


def _starts(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _page_words(D):
    U, G = D // 8, D // GROUP
    return 2 * PAGE * (U + G)


# ---- prepare ---------------------------------------------------------------------------------------------------
def _normal(g, shape, dtype, outliers=0):
    x = torch.randn(shape, generator=g, device=DEV, dtype=torch.float32)
    if outliers:  # a few channels of each head are larger, as a model's keys have them
        H, D = shape[-2], shape[-1]
        ch = torch.rand((H, D), generator=g, device=DEV).argsort(-1)[:, :outliers]
        x *= torch.ones(H, D, device=DEV).scatter_(1, ch, 6.0)
    return x.to(dtype)


def _tables(g, lens):
    """Pages of sequences of ``lens`` tokens, in any order of a pool a little larger than they need."""
    P = max(1, max(-(-n // PAGE) for n in lens))
    need = sum(-(-n // PAGE) for n in lens)
    pool = need + 7
    order = torch.randperm(pool, generator=g, device=DEV).to(torch.int32)
    table = torch.zeros(len(lens), P, dtype=torch.int32)
    host, at = order.cpu(), 0
    for s, n in enumerate(lens):
        k = -(-n // PAGE)
        table[s, :k] = host[at:at + k]
        at += k
    return pool, table.to(DEV)


def _int32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _gathered(g, lens, Hkv, T):
    """Weights [S, Hkv, T] that each token has gathered in a few steps (a few tokens get most of it); 0 past the ends."""
    n = _int32(lens)[:, None, None]
    w = torch.rand((len(lens), Hkv, T), generator=g, device=DEV).clamp_(min=1e-6).log_().neg_()
    w = w.pow_(3) / n.clamp(min=1)
    return w.masked_fill_(torch.arange(T, device=DEV) >= n, 0.0)


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt, Hkv, D = DT[c["dtype"]], c["Hkv"], c["D"]
    lens = _lengths(c)
    S, N = len(lens), sum(lens)
    st = dict(c, dt=dt, scale=D ** -0.5)
    diff = c["kind"].startswith("diff")
    if diff:  # learned: one number per output head
        st["lam"] = torch.rand(c["Hq"] // 2, generator=g, device=DEV) * 0.6 + 0.2
    if c["kind"].endswith("prompt"):
        st["cu"], st["longest"] = _int32(_starts(lens)), max(lens)
        st["q"] = _normal(g, (N, c["Hq"], D), dt)
        if not c["past"]:  # keys and values of one projection: strided views
            x = _normal(g, (N, 2 * Hkv, D), dt, 4)
            st["k"], st["v"] = x[:, :Hkv], x[:, Hkv:]
            st["cu_k"] = None
        else:
            st["k"] = _normal(g, (N + S * c["past"], Hkv, D), dt, 4)
            st["v"] = _normal(g, (N + S * c["past"], Hkv, D), dt)
            st["cu_k"] = _int32(_starts([n + c["past"] for n in lens]))
        if diff:
            st["v"] = st["v"].unflatten(1, (Hkv // 2, 2)).flatten(2)  # [Nk, Hkv/2, 2 D]: a view
        else:
            st["weights"] = _gathered(g, [c["past"]] * S, Hkv, max(lens) + c["past"])
        return st
    pool, st["table"] = _tables(g, lens)
    st["lens"] = _int32(lens)
    st["pages"] = torch.empty(pool, Hkv, _page_words(D), dtype=torch.int32, device=DEV)
    rows = torch.arange(PAGE, device=DEV)
    for p0 in range(0, pool, 512):
        n = min(512, pool - p0)
        page = torch.arange(p0, p0 + n, device=DEV).repeat_interleave(PAGE)
        row = rows.repeat(n)
        _put(st["pages"], page, row, _normal(g, (n * PAGE, Hkv, D), dt, 4), _normal(g, (n * PAGE, Hkv, D), dt))
    T = st["table"].shape[1] * PAGE
    if c["kind"] == "evict":
        st["weights"] = _gathered(g, lens, Hkv, T)
        kept = [min(n, c["keep"]) for n in lens]  # (a program knows how many tokens its sequences hold)
        st["none"], st["cu"], st["tokens"] = torch.zeros_like(st["lens"]), _int32(_starts(kept)), sum(kept)
        return st
    if c["kind"] == "weigh_attend":
        st["weights"] = _gathered(g, [n - 1 for n in lens], Hkv, T)
    m = c.get("new", 1)
    st["q"] = _normal(g, (S, m, c["Hq"], D), dt)
    if m == 1:
        st["q"] = st["q"][:, 0]
    return st


# ---- the plain forms -------------------------------------------------------------------------------------------
def _quantize(x):
    """4-bit codes, scales and minima of groups of 32 of x [..., D], each step rounded to x's type (as quant.py's ops)."""
    t = x.dtype
    x = x.float().unflatten(-1, (-1, GROUP))
    mn = x.amin(-1, keepdim=True)
    s = ((x.amax(-1, keepdim=True) - mn).to(t).float() / 15.0).to(t).float()
    y = ((x - mn).to(t).float() / s).to(t).float()
    c = torch.where(s > 0, y, torch.zeros_like(y)).clamp(0, 15).round().to(torch.int32)
    return c.flatten(-2), s[..., 0].to(t), mn[..., 0].to(t)


def _value(c, s, z, t):
    """What codes [..., D] with scales and minima [..., D/32] stand for, in fp32."""
    v = c.unflatten(-1, (-1, GROUP)).float() * s.float()[..., None] + z.float()[..., None]
    return v.to(t).float().flatten(-2)


def _words(c):
    c = c.unflatten(-1, (-1, 8)).to(torch.int64)
    w = (c << (4 * torch.arange(8, device=c.device))).sum(-1)
    return torch.where(w >= 2 ** 31, w - 2 ** 32, w).to(torch.int32)


def _codes(w):
    return ((w[..., None] >> (4 * torch.arange(8, device=w.device, dtype=torch.int32))) & 15).flatten(-2)


def _places(D, row):
    """Word offsets of K codes and K scales, then of V codes and half offsets of V scales, of page rows [...]."""
    U, G = D // 8, D // GROUP
    o, g = torch.arange(U, device=row.device), torch.arange(G, device=row.device)
    block, at = row // 32 * 4 + row % 16 // 4, row % 4 + row // 16 % 2 * 4
    row, block, at = (x[..., None] for x in (row, block, at))
    km, vc = PAGE * U, PAGE * (U + G)
    vm = vc + PAGE * U
    return row * U + o, km + row * G + g, vc + (block * U + o) * 8 + at, 2 * vm + (block * G + g) * 16 + at


def _put(pages, page, row, k, v):
    """Quantizes k and v [n, H, D] into the rows ``row`` of the pages ``page`` [n]."""
    H, D = k.shape[1:]
    t = k.dtype
    kc, ks, vc, vs = (x[:, None] for x in _places(D, row))
    p, h = page[:, None, None], torch.arange(H, device=k.device)[None, :, None]
    half = pages.view(torch.int16)
    c, s, z = _quantize(k)
    pages[p, h, kc] = _words(c)
    half[p, h, 2 * ks] = s.view(torch.int16)
    half[p, h, 2 * ks + 1] = z.view(torch.int16)
    c, s, z = _quantize(v)
    pages[p, h, vc] = _words(c)
    half[p, h, vs] = s.view(torch.int16)
    half[p, h, vs + 8] = z.view(torch.int16)


def _get(pages, page, row, D, t):
    """The values [n, H, D] of K and V in the rows ``row`` of the pages ``page`` [n], fp32."""
    H = pages.shape[1]
    kc, ks, vc, vs = (x[:, None] for x in _places(D, row))
    p, h = page[:, None, None], torch.arange(H, device=row.device)[None, :, None]
    half = pages.view(torch.int16)
    k = _value(_codes(pages[p, h, kc]), half[p, h, 2 * ks].view(t), half[p, h, 2 * ks + 1].view(t), t)
    v = _value(_codes(pages[p, h, vc]), half[p, h, vs].view(t), half[p, h, vs + 8].view(t), t)
    return k, v


def _sequence_of(cu, n):
    i = torch.arange(n, device=cu.device)
    s = torch.searchsorted(cu[1:].contiguous(), i.to(cu.dtype), right=True)
    return s, i - cu[s]


def _map(q, k, scale, hide):
    """softmax(q k^T scale) over the last dim, in fp32; ``hide`` broadcasts over the logits, rows of no key are 0."""
    s = torch.matmul(q, k.transpose(-1, -2)).mul_(scale).masked_fill_(hide, -math.inf)
    m = s.amax(-1, keepdim=True).clamp_(min=-3e38)
    s.sub_(m).exp_()
    return s.div_(s.sum(-1, keepdim=True).clamp_(min=1e-38))


def _hidden(lq, lk, Lq, Lk, window):
    """[S, Lq, Lk]: key j is hidden from query i of a sequence of lq queries and lk keys."""
    i, j = torch.arange(Lq, device=lq.device)[None, :, None], torch.arange(Lk, device=lq.device)[None, None, :]
    last = i + (lk - lq)[:, None, None]
    hide = (j > last) | (j >= lk[:, None, None]) | (i >= lq[:, None, None])
    return hide | (j <= last - window) if window else hide


def _attention(st, q, k, v, hide):
    """q [S, m, Hq, D], k, v [S, Hkv, T, D]: the output and, for plain attention, the keys' summed weights.  ``hide``
    [S, m, T]."""
    (S, m, Hq, D), (Hkv, T) = q.shape, k.shape[1:3]
    r = Hq // Hkv
    if not st["kind"].startswith("diff"):
        q = q.float().view(S, m, Hkv, r, D).permute(0, 2, 3, 1, 4).reshape(S, Hkv, r * m, D)
        p = _map(q, k, st["scale"], hide[:, None].repeat(1, 1, r, 1))
        o = torch.matmul(p, v).view(S, Hkv, r, m, D).permute(0, 3, 1, 2, 4).reshape(S, m, Hq, D)
        return o, p.sum(-2)
    G = Hkv // 2
    q = q.float().view(S, m, G, r, 2, D).permute(4, 0, 2, 3, 1, 5).reshape(2, S, G, r * m, D)
    k = k.view(S, G, 2, T, D)
    v = v.view(S, G, 2, T, D).transpose(2, 3).reshape(S, G, T, 2 * D)
    hide = hide[:, None].repeat(1, 1, r, 1)
    first, second = (torch.matmul(_map(q[i], k[:, :, i].contiguous(), st["scale"], hide), v) for i in (0, 1))
    lam = st["lam"].view(G, r, 1).expand(G, r, m).reshape(G, r * m, 1)
    o = (first - lam * second).view(S, G, r, m, 2 * D)
    return o.permute(0, 3, 1, 2, 4).reshape(S, m, G * r, 2 * D), None


def _plain_prompt(st):
    q, k, v, cu = st["q"], st["k"], st["v"], st["cu"]
    cu_k = cu if st["cu_k"] is None else st["cu_k"]
    Lq, Lk, Hkv, D = st["longest"], st["longest"] + st["past"], k.shape[1], k.shape[2]
    lq, lk = cu[1:] - cu[:-1], cu_k[1:] - cu_k[:-1]
    at = (cu[:-1, None] + torch.arange(Lq, device=cu.device)).clamp(max=q.shape[0] - 1)
    at_k = (cu_k[:-1, None] + torch.arange(Lk, device=cu.device)).clamp(max=k.shape[0] - 1)
    v = v.reshape(v.shape[0], Hkv, D)
    kp, vp = (x[at_k].float().permute(0, 2, 1, 3).contiguous() for x in (k, v))
    o, w = _attention(st, q[at], kp, vp, _hidden(lq, lk, Lq, Lk, st["window"]))
    s, i = _sequence_of(cu, q.shape[0])
    o = o[s, i].to(q.dtype)
    if w is None:
        return o
    st["weights"] += w
    return o, st["weights"]


def _plain_attend(st):
    t, D, table, lens = st["dt"], st["D"], st["table"], st["lens"]
    S, P = table.shape
    T = P * PAGE
    row = torch.arange(T, device=table.device).repeat(S)
    k, v = _get(st["pages"], table.repeat_interleave(PAGE, 1).reshape(-1).long(), row % PAGE, D, t)
    Hkv = k.shape[1]
    # rows behind a sequence's end are anything: they count for nothing
    gone = (row.view(S, T) >= lens[:, None])[:, None, :, None]
    k, v = (x.view(S, T, Hkv, D).transpose(1, 2).masked_fill(gone, 0.0).contiguous() for x in (k, v))
    m = st.get("new", 1)
    q = st["q"].view(S, m, -1, D)
    hide = _hidden(torch.full_like(lens, m), lens, m, T, st["window"])
    o, w = _attention(st, q, k, v, hide)
    o = (o if st["q"].dim() == 4 else o[:, 0]).to(t)
    if w is None:
        return o
    st["weights"] += w
    return o, st["weights"]


def _plain_evict(st):
    w, lens, table, pages = st["weights"], st["lens"], st["table"], st["pages"]
    keep, recent, sinks, D, t = st["keep"], st["recent"], st["sinks"], st["D"], st["dt"]
    (S, H, T), dev = w.shape, w.device
    B, K = keep - recent, min(keep, T)
    place = torch.arange(T, device=dev)
    n, full = lens[:, None, None], (lens > keep)[:, None, None]
    # the B chosen ones: the sinks, then those of most weight (ties: the first) of what is not among the last `recent`
    order = torch.where(place < n - recent, w, torch.full_like(w, -1.0))
    order = torch.where(place < sinks, torch.full_like(w, math.inf), order).sort(dim=-1, descending=True, stable=True).indices
    chosen = torch.zeros_like(w, dtype=torch.bool).scatter_(-1, order[..., :B], True)
    # the places below B that a token leaves free are taken, in order, by the chosen ones past B
    come = torch.where(chosen & (place >= B), place.expand_as(w), torch.full_like(order, T)).sort(-1).values
    free = ~chosen & (place < B)
    rank = (free.cumsum(-1) - 1).clamp_(min=0)
    src = torch.where(free, come.gather(-1, rank), place.expand_as(w))
    src = torch.where(place >= B, place + n - keep, src)[..., :K]
    src = torch.where(full, src, place[:K].expand(S, H, K)).clamp(max=T - 1)
    # rows and weights to their places
    s, h = torch.arange(S, device=dev)[:, None, None], torch.arange(H, device=dev)[None, :, None]
    at = place[:K].expand(S, H, K)
    half, move = pages.view(torch.int16), []
    for j in (src, at):
        page, row = table.long()[s, j // PAGE], j % PAGE
        kc, ks, vc, vs = _places(D, row)
        i, hh = page[..., None], h[..., None]
        move.append([(pages, i, hh, kc), (pages, i, hh, ks), (pages, i, hh, vc), (half, i, hh, vs), (half, i, hh, vs + 8)])
    held = (at < n) & full
    for (x, *a), (_, *b) in zip([(x, i[held], hh.expand(S, H, K, 1)[held], j[held]) for x, i, hh, j in move[1]],
                                [(x, i[held], hh.expand(S, H, K, 1)[held], j[held]) for x, i, hh, j in move[0]]):
        x[tuple(a)] = x[tuple(b)]
    out = torch.where(full, torch.zeros_like(w), w)
    out[..., :K] = torch.where(full, w.gather(-1, src), w[..., :K])
    s, i = _sequence_of(st["cu"], st["tokens"])
    k, v = _get(pages, table[s, i // PAGE].long(), i % PAGE, D, t)
    return lens.clamp(max=keep), out, k.to(t), v.to(t)


# ---- one pass --------------------------------------------------------------------------------------------------
def run(state):
    st = state
    if not own:
        return (_plain_prompt if st["kind"].endswith("prompt") else _plain_evict if st["kind"] == "evict" else _plain_attend)(st)
    from innerq_amd import ops, paged
    window = st.get("window") or None
    if st["kind"] == "weigh_prompt":
        out = ops.prompt_attention(st["q"], st["k"], st["v"], st["cu"], st["scale"], cu_seqlens_k=st["cu_k"], window=window,
                                   weights=st["weights"])
        return out, st["weights"]
    if st["kind"] == "diff_prompt":
        return ops.diff_prompt_attention(st["q"], st["k"], st["v"], st["cu"], st["lam"], st["scale"],
                                         cu_seqlens_k=st["cu_k"], window=window)
    if "store" not in st:  # a program's own store, over its pages
        st["store"] = paged.PagedStore.over(st["pages"], st["D"], st["dt"])
    store, table, lens = st["store"], st["table"], st["lens"]
    if st["kind"] == "weigh_attend":
        return store.attend(st["q"], table, lens, st["scale"], window=window, weights=st["weights"]), st["weights"]
    if st["kind"] == "diff_attend":
        return store.diff_attend(st["q"], table, lens, st["lam"], st["scale"], window=window)
    lens, weights = store.evict(table, lens, st["weights"], st["keep"], recent=st["recent"], sinks=st["sinks"])
    return (lens, weights, *store.read(table, st["none"], st["cu"], st["tokens"]))


def _visible(c, lq, lk):
    """(query, key) pairs of one sequence."""
    w = c["window"] or lk
    # query i (of lq) ends at key i + lk - lq and sees min(that + 1, w) keys
    full = lk - lq + 1
    if w >= lk:
        return sum((full, full + lq - 1)) * lq // 2
    ramp = max(0, min(lq, w - full))  # queries that see fewer than w keys
    return ramp * (2 * full + ramp - 1) // 2 + (lq - ramp) * w


def work(case):
    c = case
    lens, Hkv, D = _lengths(c), c["Hkv"], c["D"]
    N, diff = sum(lens), c["kind"].startswith("diff")
    packed = 2 * (D // 2 + D // GROUP * 4)  # bytes of one token's K and V of one head
    if c["kind"] == "evict":
        kept = sum(min(n, c["keep"]) for n in lens)
        cut = sum(n for n in lens if n > c["keep"])
        # all weights read and written; a head's rows that have to move: the last ones, and what fills the places below
        # (in a cache whose weights know no order, that share of the places which is dropped)
        moved = sum(c["recent"] + (c["keep"] - c["recent"]) * (n - c["keep"]) / max(1, n - c["recent"]) for n in lens
                    if n > c["keep"])
        return {"bytes": Hkv * (8 * N + 2 * packed * moved + (packed + 4 * D) * kept), "flops": 2.0 * Hkv * cut}
    Hq, per = c["Hq"], 6 if diff else 4  # operations of a head, pair and dim (differential: V is twice as wide)
    if c["kind"].endswith("prompt"):
        pairs = sum(_visible(c, n, n + c["past"]) for n in lens)
        keys = sum(min(n + c["past"], n + (c["window"] or n + c["past"]) - 1) for n in lens)
        return {"bytes": 2 * D * (2 * N * Hq + 2 * keys * Hkv) + (0 if diff else 8 * keys * Hkv), "flops": 1.0 * per * D * Hq * pairs}
    m = c.get("new", 1)
    held = sum(min(n, n if not c["window"] else c["window"] + m - 1) for n in lens)
    pairs = sum(_visible(c, min(m, n), n) for n in lens)
    return {"bytes": held * Hkv * (packed + (0 if diff else 8)) + 4 * D * Hq * m * len(lens), "flops": 1.0 * per * D * Hq * pairs}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------
def _softmax_rows(logits, seen):
    """softmax over the keys that ``seen`` marks; a row that sees none is 0."""
    logits = torch.where(seen, logits, torch.full_like(logits, -1e300))
    e = torch.exp(logits - logits.max(-1, keepdim=True).values) * seen
    total = e.sum(-1, keepdim=True)
    return torch.where(total > 0, e / total.clamp(min=1e-300), torch.zeros_like(e))


def _sees(first, n, keys, window):
    """[n, keys]: query i stands at key ``first + i``."""
    at = first + torch.arange(n, device=DEV)
    key = torch.arange(keys, device=DEV)
    seen = key[None] <= at[:, None]
    return seen & (at[:, None] - key[None] < window) if window else seen


def _exact_cache(st, s, n):
    """K and V [Hkv, n, D] of sequence s from its pages, in 64 bits (rounded to the type, as the cache's values are)."""
    D, t = st["D"], st["dt"]
    U, G = D // 8, D // GROUP
    words = st["pages"][st["table"][s, :-(-n // PAGE)].long()].transpose(0, 1).contiguous()  # [H, P, W]
    H, P = words.shape[:2]
    kc, km, vc, vm = torch.split(words, [PAGE * U, PAGE * G, PAGE * U, PAGE * G], dim=-1)

    def nibbles(w):  # [..., U] words -> [..., D] codes, low nibble of each byte first
        b = w.contiguous().view(torch.uint8)
        return torch.stack([b % 16, torch.div(b, 16, rounding_mode="floor")], -1).flatten(-2).double()

    def halves(w):
        return w.contiguous().view(t).double()

    def value(code, scale, low):
        return (code * scale.repeat_interleave(GROUP, -1) + low.repeat_interleave(GROUP, -1)).to(t).double()

    meta = halves(km).view(H, P * PAGE, G, 2)
    k = value(nibbles(kc.reshape(H, P * PAGE, U)), meta[..., 0], meta[..., 1])
    # V blocks: [2 halves of a page, 4 blocks, U, 2 x 16 tokens, 4 tokens] -> tokens in order
    w = vc.reshape(H, P, 2, 4, U, 2, 4).permute(0, 1, 2, 5, 3, 6, 4).reshape(H, P * PAGE, U)
    m = halves(vm).view(H, P, 2, 4, G, 2, 2, 4).permute(0, 1, 2, 6, 3, 7, 4, 5).reshape(H, P * PAGE, G, 2)
    v = value(nibbles(w), m[..., 0], m[..., 1])
    return k[:, :n], v[:, :n]


def _exact_evict(st, lens):
    weights = st["weights"].cpu().numpy()
    keep, recent, sinks = st["keep"], st["recent"], st["sinks"]
    new, ks, vs = weights.astype(np.float64), [], []
    for s, n in enumerate(lens):
        k, v = _exact_cache(st, s, n)
        if n <= keep:
            ks.append(k.transpose(0, 1)), vs.append(v.transpose(0, 1))
            continue
        new[s] = 0
        kept = np.empty((k.shape[0], keep), dtype=np.int64)
        for h in range(k.shape[0]):
            score = weights[s, h, :n - recent].copy()
            score[:sinks] = np.inf
            best = set(np.lexsort((np.arange(n - recent), -score))[:keep - recent].tolist())
            late = sorted(i for i in best if i >= keep - recent)[::-1]
            kept[h] = [i if i in best else late.pop() for i in range(keep - recent)] + list(range(n - recent, n))
            new[s, h, :keep] = weights[s, h, kept[h]]
        at = torch.from_numpy(kept).to(DEV)[..., None].expand(-1, -1, k.shape[2])
        ks.append(k.gather(1, at).transpose(0, 1)), vs.append(v.gather(1, at).transpose(0, 1))
    return None, torch.from_numpy(new).to(DEV), torch.cat(ks), torch.cat(vs)


def exact(case, seed):
    c = case
    st = prepare(case, seed)
    lens, Hkv, D = _lengths(c), c["Hkv"], c["D"]
    if c["kind"] == "evict":
        return _exact_evict(st, lens)
    Hq, m, scale = c["Hq"], c.get("new", 1), st["scale"]
    r, diff, prompt = Hq // Hkv, c["kind"].startswith("diff"), c["kind"].endswith("prompt")
    wide = 2 if diff else 1
    out, k0, q0 = [], 0, 0
    gathered = None if diff else st["weights"].double()
    for s, n in enumerate(lens):
        if prompt:
            lq, keys = n, n + c["past"]
            q = st["q"][q0:q0 + n]
            k, v = (x[k0:k0 + keys].transpose(0, 1).double() for x in (st["k"], st["v"].reshape(-1, Hkv, D)))
        else:
            lq, keys = m, n
            q = st["q"][s].view(m, Hq, D)
            k, v = _exact_cache(st, s, n)
        q0, k0 = q0 + lq, k0 + keys
        seen = _sees(keys - lq, lq, keys, c["window"])
        o = torch.empty(lq, Hq // wide, wide * D, dtype=torch.float64, device=DEV)
        for i in range(Hq // wide):  # output heads
            g = i // r  # of the group of KV heads g * wide ..
            vv = torch.cat([v[g * wide + j] for j in range(wide)], -1)
            part = []
            for j in range(wide):
                p = _softmax_rows(q[:, i * wide + j].double() @ k[g * wide + j].t().contiguous() * scale, seen)
                if gathered is not None:
                    gathered[s, g, :keys] += p.sum(0)
                part.append(p @ vv)
            o[:, i] = part[0] - st["lam"][i].double() * part[1] if diff else part[0]
        out.append(o)
    o = torch.cat(out) if prompt else torch.stack(out)
    if not prompt and m == 1:
        o = o[:, 0]
    return o if gathered is None else (o, gathered)
