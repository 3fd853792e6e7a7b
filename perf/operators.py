"""The operators of serving many sequences of different lengths, measured through their public entry points.

Three kinds of call (``kind``):

* ``prompt``  ops.prompt_attention: causal attention over prompts packed one behind the other;
* ``append``  paged.PagedStore.append: new tokens of every sequence, rotated and quantized into 4-bit pages, with the
  step's queries rotated too; the appended tokens are read back (PagedStore.read) as the values the pages hold;
* ``attend``  paged.PagedStore.attend: one token (or a few drafted ones) per sequence over its 4-bit pages.

A page holds 64 tokens of every KV head.  One (page, head) is one run of 32-bit words,

    K codes [64 tokens][D/8]   K scales/zeros [64][D/32]   V codes [8 blocks][D/8][8 tokens]   V scales/zeros [8][D/32][s x 8, z x 8]

a word being 8 codes of one token (code i at bits 4i).  Token t of a page is token t%4 + 4*(t//16%2) of V block
t//32*4 + t%16//4.  A code c stands for c*s + z, rounded to the cache's type.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
DT = {"fp16": torch.float16, "bf16": torch.bfloat16}
PAGE, GROUP = 64, 32
# (query, KV) elements of the largest listed prompt, tokens of the largest append and of the largest cache: no drawn
# case is larger
MOST_PAIRS, MOST_NEW, MOST_HELD = 32 * 16384 * 16384, 4 * 8190, 8 * 32768


def listed():
    return [
        # one user's short question: bound by the launch and by latency
        dict(name="prompt_one_short", kind="prompt", seqs=1, longest=77, mix=0, past=0, window=0, Hq=32, Hkv=8, D=128,
             dtype="fp16"),
        # a step's prompts of different lengths, packed
        dict(name="prompt_packed", kind="prompt", seqs=16, longest=2000, mix=3, past=0, window=0, Hq=32, Hkv=8, D=128,
             dtype="bf16"),
        # a long document in one call: the matrix cores' work
        dict(name="prompt_long", kind="prompt", seqs=1, longest=16384, mix=0, past=0, window=0, Hq=32, Hkv=8, D=128,
             dtype="bf16"),
        # a chunk of each of four prompts behind its earlier keys, in a model with a sliding window
        dict(name="prompt_chunk_window", kind="prompt", seqs=4, longest=512, mix=0, past=6000, window=4096, Hq=32, Hkv=8,
             D=128, dtype="fp16"),
        # a decode step of a batch of 8: latency
        dict(name="append_step", kind="append", seqs=8, longest=1, mix=0, held=32768, Hq=32, Hkv=8, D=128, dtype="fp16"),
        # prompts of different lengths behind a shared beginning, bf16, head_dim 64
        dict(name="append_ragged", kind="append", seqs=24, longest=1500, mix=5, held=333, Hq=32, Hkv=8, D=64,
             dtype="bf16"),
        # the prefill of a batch
        dict(name="append_prefill", kind="append", seqs=4, longest=8190, mix=0, held=0, Hq=32, Hkv=8, D=128,
             dtype="bf16"),
        # one user, a short chat: latency
        dict(name="attend_one_short", kind="attend", seqs=1, longest=1000, mix=0, new=1, window=0, Hq=32, Hkv=8, D=128,
             dtype="fp16"),
        # a batch of 8 at 32k tokens: the cache's stream
        dict(name="attend_batch", kind="attend", seqs=8, longest=32768, mix=0, new=1, window=0, Hq=32, Hkv=8, D=128,
             dtype="fp16"),
        # a serving batch of very different lengths, bf16
        dict(name="attend_ragged", kind="attend", seqs=48, longest=16001, mix=7, new=1, window=0, Hq=32, Hkv=8, D=128,
             dtype="bf16"),
        # four drafted tokens per sequence checked at once
        dict(name="attend_drafts", kind="attend", seqs=16, longest=4099, mix=2, new=4, window=0, Hq=32, Hkv=8, D=64,
             dtype="fp16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["prompt", "append", "attend"])
    Hq, Hkv = rng.choice([(32, 8), (32, 8), (8, 8), (16, 2), (32, 4), (12, 4)])
    c = dict(kind=kind, mix=rng.choice([0, rng.randrange(1, 1000)]), Hq=Hq, Hkv=Hkv, D=rng.choice([64, 128]),
             dtype=rng.choice(["fp16", "bf16"]))
    if kind == "prompt":
        c["seqs"] = _log_int(rng, 1, 48)
        c["past"] = rng.choice([0, 0, _log_int(rng, 1, 8000)])
        c["longest"] = _log_int(rng, 1, 8200)
        while c["seqs"] * Hq * c["longest"] * (c["longest"] + c["past"]) > MOST_PAIRS:
            c["longest"] = c["longest"] * 3 // 4
        c["window"] = rng.choice([0, 0, _log_int(rng, 1, 8000)])
    elif kind == "append":
        c["seqs"] = _log_int(rng, 1, 200)
        c["longest"] = rng.choice([1, _log_int(rng, 1, MOST_NEW // c["seqs"])])
        c["held"] = rng.choice([0, _log_int(rng, 1, MOST_HELD // c["seqs"])])
    else:
        c["seqs"] = _log_int(rng, 1, 128)
        c["longest"] = _log_int(rng, 1, MOST_HELD // c["seqs"])
        c["new"] = min(rng.choice([1, 1, rng.randrange(1, 9)]), c["longest"])
        c["window"] = rng.choice([0, 0, _log_int(rng, 1, 8000)])
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


def _angles(positions, R):
    inv = 10000.0 ** (-torch.arange(0, R, 2, device=DEV, dtype=torch.float64) / R)
    a = torch.arange(positions, device=DEV, dtype=torch.float64)[:, None] * inv
    return a.cos().float(), a.sin().float()


def _int32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt, Hq, Hkv, D = DT[c["dtype"]], c["Hq"], c["Hkv"], c["D"]
    lens = _lengths(c)
    st = dict(c, dt=dt, scale=D ** -0.5)
    if c["kind"] == "prompt":
        N, S = sum(lens), len(lens)
        st["cu"], st["longest"] = _int32(_starts(lens)), max(lens)
        st["q"] = _normal(g, (N, Hq, D), dt)
        if not c["past"]:  # keys and values of one projection: strided views
            x = _normal(g, (N, 2 * Hkv, D), dt, 4)
            st["k"], st["v"] = x[:, :Hkv], x[:, Hkv:]
            st["cu_k"] = None
        else:
            st["k"] = _normal(g, (N + S * c["past"], Hkv, D), dt, 4)
            st["v"] = _normal(g, (N + S * c["past"], Hkv, D), dt)
            st["cu_k"] = _int32(_starts([n + c["past"] for n in lens]))
        return st
    if c["kind"] == "append":
        N = sum(lens)
        held = [c["held"]] * len(lens)
        if c["mix"]:
            r = random.Random(c["mix"] + 1)
            held = [r.randrange(c["held"] + 1) for _ in lens]
        pool, st["table"] = _tables(g, [a + b for a, b in zip(held, lens)])
        st["pages"] = torch.zeros(pool, Hkv, _page_words(D), dtype=torch.int32, device=DEV)
        st["held_lens"], st["tokens"] = _int32(held), N
        st["cu"] = _int32(_starts(lens))
        st["one_each"] = c["longest"] == 1
        st["cos"], st["sin"] = _angles(max(a + b for a, b in zip(held, lens)), D)
        st["q"] = _normal(g, (N, Hq, D), dt)
        x = _normal(g, (N, 2 * Hkv, D), dt, 4)
        st["k"], st["v"] = x[:, :Hkv], x[:, Hkv:]
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
    st["q"] = _normal(g, (len(lens), c["new"], Hq, D), dt)
    if c["new"] == 1:
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
    """Word offsets of K codes and K scales, then of V codes and half offsets of V scales, of page rows [n]."""
    U, G = D // 8, D // GROUP
    o, g = torch.arange(U, device=row.device), torch.arange(G, device=row.device)
    block, at = row // 32 * 4 + row % 16 // 4, row % 4 + row // 16 % 2 * 4
    row, block, at = (x[:, None] for x in (row, block, at))
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


def _rotate(x, cos, sin):
    x = x.float()
    R = cos.shape[-1]
    a, b = x[..., :R], x[..., R:2 * R]
    cos, sin = cos[:, None], sin[:, None]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * R:]], -1)


def _sequence_of(cu, n):
    i = torch.arange(n, device=cu.device)
    s = torch.searchsorted(cu[1:].contiguous(), i.to(cu.dtype), right=True)
    return s, i - cu[s]


def _attention(q, k, v, scale, hide):
    """softmax(q k^T scale) v over the last two dims, in fp32; ``hide`` broadcasts over the logits, rows of no key are 0."""
    s = torch.matmul(q, k.transpose(-1, -2)).mul_(scale).masked_fill_(hide, -math.inf)
    m = s.amax(-1, keepdim=True).clamp_(min=-3e38)
    s.sub_(m).exp_()
    return torch.matmul(s, v) / s.sum(-1, keepdim=True).clamp_(min=1e-38)


def _hidden(lq, lk, Lq, Lk, window):
    """[S, Lq, Lk]: key j is hidden from query i of a sequence of lq queries and lk keys."""
    i, j = torch.arange(Lq, device=lq.device)[None, :, None], torch.arange(Lk, device=lq.device)[None, None, :]
    last = i + (lk - lq)[:, None, None]
    hide = (j > last) | (j >= lk[:, None, None])
    return hide | (j <= last - window) if window else hide


def _plain_prompt(st):
    q, k, v, cu = st["q"], st["k"], st["v"], st["cu"]
    cu_k = cu if st["cu_k"] is None else st["cu_k"]
    Lq, Lk, Hkv, D = st["longest"], st["longest"] + st["past"], k.shape[1], k.shape[2]
    lq, lk = cu[1:] - cu[:-1], cu_k[1:] - cu_k[:-1]
    S, r = lq.shape[0], q.shape[1] // Hkv
    at = (cu[:-1, None] + torch.arange(Lq, device=cu.device)).clamp(max=q.shape[0] - 1)
    at_k = (cu_k[:-1, None] + torch.arange(Lk, device=cu.device)).clamp(max=k.shape[0] - 1)
    qp = q[at].float().view(S, Lq, Hkv, r, D).permute(0, 2, 3, 1, 4).reshape(S, Hkv, r * Lq, D)
    kp, vp = (x[at_k].float().permute(0, 2, 1, 3).contiguous() for x in (k, v))
    hide = _hidden(lq, lk, Lq, Lk, st["window"])[:, None].repeat(1, 1, r, 1)
    o = _attention(qp, kp, vp, st["scale"], hide).view(S, Hkv, r, Lq, D)
    s, i = _sequence_of(cu, q.shape[0])
    return o.permute(0, 3, 1, 2, 4)[s, i].reshape(q.shape).to(q.dtype)


def _plain_append(st):
    s, i = _sequence_of(st["cu"], st["tokens"])
    at = (st["held_lens"][s] + i).long()
    page, row = st["table"][s, at // PAGE].long(), at % PAGE
    cos, sin = st["cos"][at], st["sin"][at]
    t, D = st["dt"], st["D"]
    _put(st["pages"], page, row, _rotate(st["k"], cos, sin).to(t), st["v"])
    k, v = _get(st["pages"], page, row, D, t)
    return _rotate(st["q"], cos, sin).to(t), k.to(t), v.to(t)


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
    q = st["q"].view(S, st["new"], -1, D)
    m, Hq = q.shape[1:3]
    qp = q.float().view(S, m, Hkv, -1, D).permute(0, 2, 3, 1, 4).reshape(S, Hkv, -1, D)
    hide = _hidden(torch.full_like(lens, m), lens, m, T, st["window"])[:, None].repeat(1, 1, Hq // Hkv, 1)
    o = _attention(qp, k, v, st["scale"], hide).view(S, Hkv, -1, m, D)
    return o.permute(0, 3, 1, 2, 4).reshape(st["q"].shape).to(t)


# ---- one pass --------------------------------------------------------------------------------------------------
def run(state):
    st = state
    if not own:
        return {"prompt": _plain_prompt, "append": _plain_append, "attend": _plain_attend}[st["kind"]](st)
    from innerq_amd import ops, paged
    window = st.get("window") or None
    if st["kind"] == "prompt":
        return ops.prompt_attention(st["q"], st["k"], st["v"], st["cu"], st["scale"], cu_seqlens_k=st["cu_k"],
                                    window=window)
    if "store" not in st:  # a program's own store, over its pages
        st["store"] = paged.PagedStore.over(st["pages"], st["D"], st["dt"])
    if st["kind"] == "attend":
        return st["store"].attend(st["q"], st["table"], st["lens"], st["scale"], window=window)
    cu = None if st["one_each"] else st["cu"]
    q = st["store"].append(st["k"], st["v"], st["table"], st["held_lens"], cu, cos=st["cos"], sin=st["sin"], q=st["q"])
    k, v = st["store"].read(st["table"], st["held_lens"], cu, st["tokens"])
    return q, k, v


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
    lens, Hq, Hkv, D = _lengths(c), c["Hq"], c["Hkv"], c["D"]
    N = sum(lens)
    packed = 2 * Hkv * (D // 2 + D // GROUP * 4)  # bytes of one token's K and V
    if c["kind"] == "prompt":
        pairs = sum(_visible(c, n, n + c["past"]) for n in lens)
        keys = sum(min(n + c["past"], n + (c["window"] or n + c["past"]) - 1) for n in lens)
        return {"bytes": 2 * D * (2 * N * Hq + 2 * keys * Hkv), "flops": 4.0 * D * Hq * pairs}
    if c["kind"] == "append":
        moved = 2 * D * (2 * Hq + 4 * Hkv) + packed + 4 * D  # in, out, packed rows, cos and sin
        return {"bytes": N * moved, "flops": N * D * (3.0 * (Hq + Hkv) + 12 * Hkv)}
    m = c["new"]
    held = sum(min(n, n if not c["window"] else c["window"] + m - 1) for n in lens)
    pairs = sum(_visible(c, min(m, n), n) for n in lens)
    return {"bytes": held * packed + 4 * D * Hq * m * len(lens), "flops": 4.0 * D * Hq * pairs}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------
def _softmax_rows(logits, seen, v):
    """Rows of softmax(logits) v over the keys that ``seen`` marks; a row that sees none is 0."""
    logits = torch.where(seen, logits, torch.full_like(logits, -1e300))
    e = torch.exp(logits - logits.max(-1, keepdim=True).values) * seen
    total = e.sum(-1, keepdim=True)
    return torch.where(total > 0, (e @ v) / total.clamp(min=1e-300), torch.zeros_like(total))


def _sees(first, n, keys, window):
    """[n, keys]: query i stands at key ``first + i``."""
    at = first + torch.arange(n, device=DEV)
    key = torch.arange(keys, device=DEV)
    seen = key[None] <= at[:, None]
    return seen & (at[:, None] - key[None] < window) if window else seen


def _exact_group(x, t):
    """Codes, scales, minima of x [n, H, D] (doubles that the type t holds), by the definition."""
    near = lambda y: y.to(t).double()  # noqa: E731
    n, H, D = x.shape
    x = x.reshape(n, H, D // GROUP, GROUP)
    low, high = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
    step = near(near(high - low) / 15)
    level = torch.round(near(near(x - low) / torch.where(step > 0, step, torch.ones_like(step))).clamp(0, 15))
    return (level * step + low).reshape(n, H, D)


def _exact_rotation(x, angle_cos, angle_sin):
    half = angle_cos.shape[1]
    out = x.double().clone()
    c, s = angle_cos.double()[:, None], angle_sin.double()[:, None]
    first, second = x[..., :half].double(), x[..., half:2 * half].double()
    out[..., :half] = first * c - second * s
    out[..., half:2 * half] = second * c + first * s
    return out


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


def exact(case, seed):
    c = case
    st = prepare(case, seed)
    lens, Hq, Hkv, D = _lengths(c), c["Hq"], c["Hkv"], c["D"]
    r = Hq // Hkv
    if c["kind"] == "append":
        held = st["held_lens"].tolist()
        at = torch.cat([torch.arange(a, a + n) for a, n in zip(held, lens)]).to(DEV)
        cos, sin, t = st["cos"][at], st["sin"][at], st["dt"]
        q = _exact_rotation(st["q"], cos, sin)
        k = _exact_rotation(st["k"], cos, sin).to(t).double()
        return q, _exact_group(k, t), _exact_group(st["v"].double(), t)
    if c["kind"] == "prompt":
        out = torch.zeros(sum(lens), Hq, D, dtype=torch.float64, device=DEV)
        k0 = q0 = 0
        for n in lens:
            keys = n + c["past"]
            seen = _sees(c["past"], n, keys, c["window"])
            for h in range(Hq):
                q, k, v = (x.double() for x in (st["q"][q0:q0 + n, h], st["k"][k0:k0 + keys, h // r],
                                                st["v"][k0:k0 + keys, h // r]))
                out[q0:q0 + n, h] = _softmax_rows(q @ k.t().contiguous() * st["scale"], seen, v)
            q0, k0 = q0 + n, k0 + keys
        return out
    m = c["new"]
    q = st["q"].double().view(len(lens), m, Hkv, r, D)
    out = torch.zeros_like(q)
    for s, n in enumerate(lens):
        k, v = _exact_cache(st, s, n)
        seen = _sees(n - m, m, n, c["window"])
        for h in range(Hkv):
            logits = q[s, :, h].reshape(m * r, D) @ k[h].t().contiguous() * st["scale"]
            out[s, :, h] = _softmax_rows(logits, seen.repeat_interleave(r, 0), v[h]).view(m, r, D)
    return out.view(st["q"].shape)
