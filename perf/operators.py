"""Cases of the 4-bit paged KV cache operators (bfp200.kv4) and their plain forms.

  rope       rotary position embedding of a [tokens, heads, head dim] tensor, and its gradient (the inverse rotation)
  append     new keys and values rotated, quantized to 4-bit tiles and written to a paged cache, the queries rotated on
             the way; the written tokens come back as the values that the cache holds for them (kv4.read)
  read       cached tokens gathered from their pages and decoded
  attention  queries against the 4-bit cache: single tokens, a few tokens, prompts

Cache pool: uint8 [pages][KV heads][page][HD * 9 / 8]; the last two axes are one record per page and head:
  keys       [page/4][HD/8][4 positions][4 bytes]: nibble n of a word is dim 8 u + n of its position
  values     [page/8][HD/4][4 i][2 h][2 bytes]: position 8 o + 4 h + i, nibble n of its 2 bytes is dim 4 u + n
  key exponents [HD/16][page], value exponents [HD/16][page]: one byte B per 16-dim tile of a position
A nibble n with exponent byte B stands for (n - 8) * 2^(B - 21), 1 <= B <= 30.  Tiles are made by the framework's rule
with 4-bit mantissas: e = clip(floor(log2(max|v|)) + 1, -17, 12), m = clip(rint(v * 2^(3 - e)), -8, 7), B = e + 18.
"""
import os
import random
import sys

import numpy as np
import torch

own = False

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # one decode step's queries and keys (9 + 3 heads of 64): launch latency
        dict(name="rope_step", op="rope", t=1, heads=12, hd=64, rot=64, dtype="bf16", inter=False, inverse=False, npos=2048),
        # gradient of a long-context batch: half of each head rotated, interleaved pairs, 32-bit
        dict(name="rope_grad_16k", op="rope", t=16383, heads=40, hd=128, rot=64, dtype="f32", inter=True, inverse=True,
             npos=32768),
        # one decode step of 64 sequences: one new position each, scattered over the pool's pages
        dict(name="append_step_64", op="append", n=64, hq=9, hkv=3, hd=64, rot=64, dtype="bf16", inter=False, page=64,
             qmax=1, lmax=2047, lens=1),
        # prompts of 24 requests written in one call
        dict(name="append_prompts", op="append", n=24, hq=32, hkv=8, hd=128, rot=128, dtype="f16", inter=False, page=64,
             qmax=2048, lmax=4096, lens=2),
        # one sequence's cache handed to other code (KV 303: a 48-token prompt and 255 generated)
        dict(name="read_303", op="read", n=1, hq=9, hkv=3, hd=64, dtype="bf16", page=64, lmax=303, lens=3),
        # the whole cache of 16 long sequences
        dict(name="read_16x8k", op="read", n=16, hq=32, hkv=8, hd=128, dtype="f16", page=32, lmax=8192, lens=4),
        # single stream in the middle of a 256-token generation: latency
        dict(name="attn_1x176", op="attention", n=1, hq=9, hkv=3, hd=64, dtype="bf16", page=64, qmax=1, lmax=176, lens=5,
             causal=True, window=0, empty=False),
        # a serving step of 256 ragged sequences, one of them without any position yet
        dict(name="attn_256x2k", op="attention", n=256, hq=9, hkv=3, hd=64, dtype="bf16", page=64, qmax=1, lmax=2047,
             lens=6, causal=True, window=0, empty=True),
        # one very long stream: the long axis has to be split over the GPU
        dict(name="attn_1x128k", op="attention", n=1, hq=9, hkv=3, hd=64, dtype="f16", page=128, qmax=1, lmax=131071,
             lens=7, causal=True, window=0, empty=False),
        # a serving step of 64 long sequences with wide heads: cache bandwidth
        dict(name="attn_64x8k", op="attention", n=64, hq=32, hkv=8, hd=128, dtype="bf16", page=64, qmax=1, lmax=8191,
             lens=8, causal=True, window=0, empty=False),
        # short ragged prompts (up to 48 tokens) in 32 bits
        dict(name="prompts_33x48", op="attention", n=33, hq=9, hkv=3, hd=64, dtype="f32", page=16, qmax=48, lmax=48,
             lens=9, causal=True, window=0, empty=False),
        # one long prompt: the largest amount of arithmetic
        dict(name="prompt_8k", op="attention", n=1, hq=32, hkv=8, hd=128, dtype="bf16", page=64, qmax=8192, lmax=8192,
             lens=10, causal=True, window=0, empty=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["rope", "append", "read", "attention", "attention", "attention"])
    dtype = rng.choice(["bf16", "f16", "f32"])
    if op == "rope":
        hd = rng.choice([32, 64, 80, 96, 128, 256])
        heads = rng.choice([1, 3, 9, 12, 40])
        t = _log(rng, 1, min(16383, 16383 * 40 * 128 // (heads * hd)))
        return dict(op=op, t=t, heads=heads, hd=hd, rot=rng.choice([hd, hd // 2, hd // 4]), dtype=dtype,
                    inter=rng.random() < 0.5, inverse=rng.random() < 0.5, npos=rng.choice([2048, 8192, 32768]))
    hd = rng.choice([32, 64, 96, 128])
    hkv = rng.choice([1, 2, 3, 8])
    hq = hkv * rng.choice([1, 2, 3, 4, 5, 8])
    page = rng.choice([16, 32, 64, 128])
    lens = rng.randrange(1 << 20)
    if op == "append":
        n = _log(rng, 1, 64)
        qmax = _log(rng, 1, max(1, min(2048, 24 * 2048 // n)))
        return dict(op=op, n=n, hq=hq if hq <= 32 else hkv, hkv=hkv, hd=hd, rot=rng.choice([hd, hd // 2]), dtype=dtype,
                    inter=rng.random() < 0.5, page=page, qmax=qmax, lmax=max(qmax, _log(rng, 1, 4096)), lens=lens)
    if op == "read":
        n = _log(rng, 1, 64)
        return dict(op=op, n=n, hq=hq, hkv=hkv, hd=hd, dtype=dtype, page=page, lmax=_log(rng, 1, 16 * 8192 // max(n, 16)),
                    lens=lens)
    kind = rng.choice(["step", "few", "prompt"])
    n = _log(rng, 1, 256)
    cells = 64 * 8191 * 8 * 128 // 2 // (n * hkv * hd)          # cached values, half the largest listed case
    lmax = _log(rng, 1, max(1, min(131071, cells)))
    if kind == "step":
        qmax = 1
    else:
        room = max(1, (1 << 29) // (n * hq * lmax))               # padded scores of the plain form
        qmax = rng.randint(2, 16) if kind == "few" else _log(rng, 17, 4096)
        qmax = max(1, min(qmax, lmax, room))
    return dict(op=op, n=n, hq=hq, hkv=hkv, hd=hd, dtype=dtype, page=page, qmax=qmax, lmax=lmax, lens=lens,
                causal=rng.random() < 0.8, window=rng.choice([0, 0, 0, max(1, lmax // 3)]), empty=n > 1 and rng.random() < 0.3)


# ---- what a batch looks like: cached length and new tokens of each sequence ------------------------------------------

def _batch(case):
    """(lens, new): positions after the call, and how many of them are this call's tokens."""
    r = random.Random(case["lens"])
    lmax, n = case["lmax"], case["n"]
    lens = [lmax] + [r.randint(max(1, lmax // 8), lmax) for _ in range(n - 1)]
    qmax = case.get("qmax", 0)
    if case["op"] == "read":
        new = list(lens)
    else:
        new = [min(L, qmax if i == 0 else r.randint(max(1, qmax // 4), qmax)) for i, L in enumerate(lens)]
    if case.get("empty"):
        lens[-1], new[-1] = 0, 1
    return lens, new


def work(case):
    es = SIZE[case["dtype"]]
    if case["op"] == "rope":
        x = case["t"] * case["heads"] * case["hd"]
        rows = min(case["t"], case["npos"])
        return {"bytes": 2 * x * es + rows * case["rot"] * 4 + 4 * case["t"], "flops": 3 * case["t"] * case["heads"] * case["rot"]}
    lens, new = _batch(case)
    hq, hkv, hd = case["hq"], case["hkv"], case["hd"]
    t, cached = sum(new), hkv * hd * 9 // 8                           # bytes of one position's keys and values
    tables = 4 * (2 * len(lens) + 1 + sum(-(-L // case["page"]) for L in lens))
    if case["op"] == "append":
        b = 2 * t * hkv * hd * es + 2 * t * hq * hd * es + t * cached + t * case["rot"] * 4    # in, queries, cache, table
        return {"bytes": b + t * cached + 2 * t * hkv * hd * es + tables, "flops": 6 * t * (hq + 2 * hkv) * hd}
    if case["op"] == "read":
        return {"bytes": t * cached + 2 * t * hkv * hd * es + tables, "flops": 2 * t * hkv * hd}
    pairs = seen = 0
    for L, m in zip(lens, new):
        w = case["window"]
        q = np.arange(L - m, L)
        hi = np.minimum(q, L - 1) if case["causal"] else np.full(m, L - 1)
        lo = np.maximum(0, q - w + 1) if w else np.zeros(m, np.int64)
        k = np.where(q < 0, 0, np.maximum(0, hi - lo + 1))
        pairs += int(k.sum())
        if k.sum():
            seen += int(hi[k > 0].max() - lo[k > 0].min() + 1)
    return {"bytes": seen * cached + 2 * t * hq * hd * es + 4 * t * hq + tables, "flops": 4 * pairs * hq * hd}


# ---- inputs ------------------------------------------------------------------------------------------------------------

def _table(npos, rot, dev):
    """(cos, sin) of position * 10000^(-2 j / rot), 32-bit [npos, rot / 2, 2]."""
    f = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=dev) / rot)
    a = torch.arange(npos, dtype=torch.float64, device=dev)[:, None] * f
    return torch.stack([a.cos(), a.sin()], -1).float().contiguous()


def _acts(shape, gen, dtype):
    """Activations: normal, with a few channels several times larger than the rest."""
    x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    big = torch.rand(shape[-1], generator=gen, device="cuda") < 0.05
    return (x * torch.where(big, 6.0, 1.0)).to(DT[dtype])


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    s = dict(case=case)
    if case["op"] == "rope":
        # a user's x is a slice of a wider projection: tokens lie further apart than their heads need
        wide = _acts((case["t"], case["heads"] + 2, case["hd"]), gen, case["dtype"])
        s["x"] = wide[:, : case["heads"]]
        s["pos"] = torch.randint(0, case["npos"], (case["t"],), generator=gen, device=dev, dtype=torch.int32)
        s["table"] = _table(case["npos"], case["rot"], dev)
        return s
    lens, new = _batch(case)
    n, hkv, hd, page = case["n"], case["hkv"], case["hd"], case["page"]
    per = -(-case["lmax"] // page)
    used = [-(-L // page) for L in lens]
    total = sum(used) + 1
    order = torch.randperm(total, generator=gen, device=dev).to(torch.int32)
    first = np.concatenate([[0], np.cumsum(used)])
    at = torch.arange(per, device=dev)[None, :] + torch.tensor(first[:-1], device=dev)[:, None]
    live = torch.arange(per, device=dev)[None, :] < torch.tensor(used, device=dev)[:, None]
    s["bt"] = torch.where(live, order[at.clamp(max=total - 1)], torch.full_like(at, -1, dtype=torch.int32)).contiguous()
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    s["q_start"] = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device=dev)
    t = int(sum(new))
    s["tokens"] = t
    pool = torch.empty((total, hkv, page, hd * 9 // 8), dtype=torch.uint8, device=dev)
    rec = pool.view(total, hkv, page * hd * 9 // 8)
    for a in range(0, total, 2048):                    # cached keys and values of earlier calls
        m = min(2048, total - a)
        rec[a:a + m] = _pack(_acts((m, hkv, page, hd), gen, "f32"), _acts((m, hkv, page, hd), gen, "f32"))
    s["pool"] = pool
    if case["op"] == "append":
        qkv = _acts((t, case["hq"] + 2 * hkv, hd), gen, case["dtype"])          # one fused projection's output
        s["q"], s["k"], s["v"] = qkv[:, : case["hq"]], qkv[:, case["hq"]: case["hq"] + hkv], qkv[:, case["hq"] + hkv:]
        s["table"] = _table(per * page, case["rot"], dev)
    elif case["op"] == "attention":
        s["q"] = _acts((t, case["hq"], hd), gen, case["dtype"])
    return s


# ---- plain forms -------------------------------------------------------------------------------------------------------

def _rotate(x, cs, rot, inter, sign):
    """x float [tokens, heads, hd], cs [tokens, rot / 2, 2]."""
    c, sn = cs[:, None, :, 0], cs[:, None, :, 1] * sign
    head, tail = x[..., :rot], x[..., rot:]
    if inter:
        a, b = head[..., 0::2], head[..., 1::2]
        y = torch.stack([a * c - b * sn, a * sn + b * c], -1).flatten(-2)
    else:
        a, b = head[..., : rot // 2], head[..., rot // 2:]
        y = torch.cat([a * c - b * sn, a * sn + b * c], -1)
    return torch.cat([y, tail], -1)


def _pow2(e):
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _quantize(x):
    """float [..., hd] -> nibbles 0..15 (int32 [..., hd]) and exponent bytes (int32 [..., hd / 16])."""
    t = x.unflatten(-1, (-1, 16))
    top = t.abs().amax(-1)
    e = ((top.view(torch.int32) >> 23) - 126).clamp(-17, 12)
    m = torch.round(t * _pow2(3 - e)[..., None]).clamp(-8, 7)
    return (m.to(torch.int32) + 8).flatten(-2), e + 18


def _bytes(nib):
    return nib[..., 0::2] | (nib[..., 1::2] << 4)


def _pack(k, v):
    """Whole pages: float [..., page, hd] keys and values -> records [..., page * hd * 9 / 8]."""
    (kn, ke), (vn, ve) = _quantize(k), _quantize(v)
    page, hd = k.shape[-2:]
    kb = _bytes(kn).unflatten(-1, (hd // 8, 4)).unflatten(-3, (page // 4, 4)).transpose(-3, -2).flatten(-4)
    vb = _bytes(vn).unflatten(-1, (hd // 4, 2)).unflatten(-3, (page // 8, 2, 4))           # oct, h, i, unit, byte
    vb = vb.movedim(-2, -4).transpose(-3, -2).flatten(-5)                                   # oct, unit, i, h, byte
    return torch.cat([kb, vb, ke.transpose(-1, -2).flatten(-2), ve.transpose(-1, -2).flatten(-2)], -1).to(torch.uint8)


def _unpack(rec, page, hd):
    """Records [..., page * hd * 9 / 8] -> float keys and values [..., page, hd]."""
    half, ex = page * hd // 2, page * hd // 16
    two = lambda b: torch.stack([b & 15, b >> 4], -1).flatten(-2)
    kn = two(rec[..., :half].unflatten(-1, (page // 4, hd // 8, 4, 4)).transpose(-3, -2)).flatten(-2).flatten(-3, -2)
    vn = rec[..., half: 2 * half].unflatten(-1, (page // 8, hd // 4, 4, 2, 2)).transpose(-3, -2).movedim(-4, -2)
    vn = two(vn).flatten(-2).flatten(-4, -2)
    e = rec[..., 2 * half:].unflatten(-1, (2, hd // 16, page)).transpose(-1, -2)
    scale = _pow2(e.to(torch.int32) - 21).repeat_interleave(16, -1)
    return (kn.float() - 8) * scale[..., 0, :, :], (vn.float() - 8) * scale[..., 1, :, :]


def _tokens(s):
    """Sequence and position of each of the call's tokens."""
    t = torch.arange(s["tokens"], device=s["lens"].device)
    seq = torch.searchsorted(s["q_start"][1:].long(), t, right=True)
    new = (s["q_start"][1:] - s["q_start"][:-1]).long()
    return seq, s["lens"].long()[seq] - new[seq] + t - s["q_start"].long()[seq]


def _plain_rope(s):
    c = s["case"]
    y = _rotate(s["x"].float(), s["table"][s["pos"].long()], c["rot"], c["inter"], -1.0 if c["inverse"] else 1.0)
    return {"out": y.to(s["x"].dtype)}


def _plain_read(s):
    c = s["case"]
    page, hd, dt = c["page"], c["hd"], DT[c["dtype"]]
    seq, pos = _tokens(s)
    pages = s["bt"].long()[seq, pos // page]
    k, v = _unpack(s["pool"].flatten(-2), page, hd)
    return {"k": k[pages, :, pos % page].to(dt), "v": v[pages, :, pos % page].to(dt)}


def _plain_append(s):
    c = s["case"]
    page, hd, hkv, dt = c["page"], c["hd"], c["hkv"], DT[c["dtype"]]
    seq, pos = _tokens(s)
    cs = s["table"][pos]
    q = _rotate(s["q"].float(), cs, c["rot"], c["inter"], 1.0).to(dt)
    kn, ke = _quantize(_rotate(s["k"].float(), cs, c["rot"], c["inter"], 1.0))
    vn, ve = _quantize(s["v"].float())
    # byte addresses of the tokens' keys, values and exponents in their records
    rec = s["pool"].flatten(-2)
    dev = rec.device
    slot = (pos % page)[:, None]
    kb = torch.arange(hd // 2, device=dev)[None]
    ka = ((slot // 4) * (hd // 8) + kb // 4) * 16 + (slot % 4) * 4 + kb % 4
    va = page * hd // 2 + ((slot // 8) * (hd // 4) + kb // 2) * 16 + (slot % 4) * 4 + (slot // 4 % 2) * 2 + kb % 2
    ea = page * hd + torch.arange(hd // 16, device=dev)[None] * page + slot
    addr = torch.cat([ka, va, ea, ea + page * hd // 16], 1)[:, None]
    vals = torch.cat([_bytes(kn), _bytes(vn), ke, ve], -1).to(torch.uint8)
    page_of = s["bt"].long()[seq, pos // page][:, None, None]
    rec[page_of, torch.arange(hkv, device=dev)[None, :, None], addr] = vals
    scale = lambda e: _pow2(e - 21).repeat_interleave(16, -1)
    return {"q": q, "k": ((kn - 8) * scale(ke)).to(dt), "v": ((vn - 8) * scale(ve)).to(dt)}


def _plain_attention(s):
    c = s["case"]
    page, hd, hq, hkv, n, qmax, dt = c["page"], c["hd"], c["hq"], c["hkv"], c["n"], c["qmax"], DT[c["dtype"]]
    k, v = _unpack(s["pool"].flatten(-2)[s["bt"].clamp(min=0).long()], page, hd)            # [n, pages, hkv, page, hd]
    k, v = (x.transpose(1, 2).flatten(2, 3) for x in (k, v))                                # [n, hkv, keys, hd]
    keys = k.shape[2]
    new = (s["q_start"][1:] - s["q_start"][:-1]).long()
    j = torch.arange(qmax, device=k.device)
    row = (s["q_start"][:-1].long()[:, None] + j).clamp(max=s["tokens"] - 1)                # [n, qmax]
    g = hq // hkv
    q = s["q"].float()[row].unflatten(2, (hkv, g)).movedim(1, 3).flatten(2, 3)              # [n, hkv, g * qmax, hd]
    sc = (q @ k.transpose(-1, -2) * hd ** -0.5).unflatten(2, (g, qmax))
    qpos = (s["lens"].long() - new)[:, None] + j
    kpos = torch.arange(keys, device=k.device)
    see = (kpos[None, None] < s["lens"].long()[:, None, None]) & (qpos >= 0)[..., None]
    if c["causal"]:
        see = see & (kpos[None, None] <= qpos[..., None])
    if c["window"]:
        see = see & (kpos[None, None] > qpos[..., None] - c["window"])
    sc = torch.where(see[:, None, None], sc, torch.full((), -torch.inf, device=sc.device))
    top = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(top == -torch.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    o = (p.flatten(2, 3) @ v).unflatten(2, (g, qmax)) / torch.where(total == 0, torch.ones_like(total), total)
    lse = (top + torch.log(total))[..., 0]
    at = torch.arange(s["tokens"], device=k.device)
    seq = torch.searchsorted(s["q_start"][1:].long(), at, right=True)
    jj = at - s["q_start"].long()[seq]
    return {"out": o.movedim(3, 1).flatten(2, 3)[seq, jj].to(dt), "lse": lse.movedim(3, 1).flatten(2, 3)[seq, jj]}


# ---- one pass ----------------------------------------------------------------------------------------------------------

def _kv4():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tinyllm-fpga_b200")
    if at not in sys.path:
        sys.path.insert(1, at)
    from bfp200 import kv4
    return kv4


def run(s):
    c = s["case"]
    op = c["op"]
    if not own:
        return {"rope": _plain_rope, "append": _plain_append, "read": _plain_read, "attention": _plain_attention}[op](s)
    kv4 = sys.modules.get("bfp200.kv4") or _kv4()
    if op == "rope":
        return {"out": kv4.rope(s["x"], s["pos"], s["table"], interleaved=c["inter"], inverse=c["inverse"])}
    if op == "append":
        q = kv4.append(s["pool"], s["k"], s["v"], s["q_start"], s["lens"], s["bt"], q=s["q"], table=s["table"],
                       interleaved=c["inter"])
        k, v = kv4.read(s["pool"], s["q_start"], s["lens"], s["bt"], s["tokens"], dtype=DT[c["dtype"]])
        return {"q": q, "k": k, "v": v}
    if op == "read":
        k, v = kv4.read(s["pool"], s["q_start"], s["lens"], s["bt"], s["tokens"], dtype=DT[c["dtype"]])
        return {"k": k, "v": v}
    out, lse = kv4.attention(s["q"], s["pool"], s["q_start"], s["lens"], s["bt"], causal=c["causal"], window=c["window"],
                             return_lse=True)
    return {"out": out, "lse": lse}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------

def _held(pool, pages, pos, page, hd):
    """What the cache holds at `pos` of page table row `pages`, addressed value by value: float64 (k, v) [len, hkv, hd]."""
    rec = pool.flatten(-2)
    pg, sl = pages.long()[pos // page], pos % page
    d = torch.arange(hd, device=pool.device)
    out = []
    for what in (0, 1):
        if what == 0:
            byte = (sl[:, None] // 4) * 2 * hd + (d // 8) * 16 + (sl[:, None] % 4) * 4 + (d % 8) // 2
        else:
            byte = page * hd // 2 + (sl[:, None] // 8) * 4 * hd + (d // 4) * 16 + (sl[:, None] % 4) * 4 + \
                (sl[:, None] % 8 // 4) * 2 + (d % 4) // 2
        ex = page * hd + what * (hd // 16) * page + (d // 16) * page + sl[:, None]
        row = rec[pg]                                                    # [len, hkv, record]
        take = lambda a: torch.gather(row, 2, a[:, None].expand(-1, row.shape[1], -1)).double()
        b = take(byte)
        nib = torch.where((d % 2 == 1), torch.floor(b / 16), b - 16 * torch.floor(b / 16))
        out.append((nib - 8.0) * torch.exp2(take(ex) - 21.0))
    return out


def _angle(x, cs, rot, inter, sign):
    """Rotation as a product of complex numbers, 64-bit."""
    z = torch.view_as_complex(cs.double().contiguous())[:, None]
    z = z if sign > 0 else z.conj()
    y = x.double().clone()
    i = torch.arange(rot // 2, device=x.device)
    a, b = (2 * i, 2 * i + 1) if inter else (i, i + rot // 2)
    w = torch.complex(y[..., a], y[..., b]) * z
    y[..., a], y[..., b] = w.real, w.imag
    return y


def _rounded(x):
    """The values that a 4-bit cache holds for x (float64)."""
    t = x.unflatten(-1, (x.shape[-1] // 16, 16))
    top = t.abs().amax(-1, keepdim=True)
    e = (torch.frexp(top)[1].double()).clamp(-17, 12)
    e = torch.where(top == 0, torch.full_like(e, -17.0), e)
    step = torch.exp2(e - 3)
    return (torch.round(t / step).clamp(-8, 7) * step).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        return {"out": _angle(s["x"], s["table"][s["pos"].long()], case["rot"], case["inter"], -1 if case["inverse"] else 1)}
    lens, new = _batch(case)
    page, hd = case["page"], case["hd"]
    outs = []
    at = 0
    for b, (L, m) in enumerate(zip(lens, new)):
        pos = torch.arange(L - m, L, device="cuda")
        rows = slice(at, at + m)
        at += m
        if case["op"] == "append":
            cs = s["table"][pos]
            # a key within rounding of the middle of two steps has no one value: none are given for keys
            outs.append((_angle(s["q"][rows], cs, case["rot"], case["inter"], 1), None, _rounded(s["v"][rows].double())))
            continue
        if case["op"] == "read":
            ks, vs = zip(*[_held(s["pool"], s["bt"][b], p, page, hd) for p in pos.split(1024)])
            outs.append((torch.cat(ks), torch.cat(vs)))
            continue
        out = torch.zeros((m, case["hq"], hd), dtype=torch.float64, device="cuda")
        lse = torch.full((m, case["hq"]), -torch.inf, dtype=torch.float64, device="cuda")
        if L:
            both = [_held(s["pool"], s["bt"][b], p, page, hd) for p in torch.arange(L, device="cuda").split(1024)]
            k, v = torch.cat([x[0] for x in both]), torch.cat([x[1] for x in both])
            kp = torch.arange(L, device="cuda")
            dist = pos[:, None] - kp[None]
            bad = torch.zeros_like(dist, dtype=torch.bool)
            if case["causal"]:
                bad |= dist < 0
            if case["window"]:
                bad |= dist >= case["window"]
            bad |= pos[:, None] < 0
            for h in range(case["hq"]):
                kh = h * case["hkv"] // case["hq"]
                a = (s["q"][rows, h].double() @ k[:, kh].T) / hd ** 0.5
                a = a.masked_fill(bad, -torch.inf)
                l = torch.logsumexp(a, -1)
                w = torch.exp(a - torch.where(l == -torch.inf, torch.zeros_like(l), l)[:, None])
                out[:, h], lse[:, h] = w @ v[:, kh], l
        outs.append((out, lse))
    if case["op"] == "append":
        return {"q": torch.cat([o[0] for o in outs]), "k": None, "v": torch.cat([o[2] for o in outs])}
    a, b = torch.cat([o[0] for o in outs]), torch.cat([o[1] for o in outs])
    return {"k": a, "v": b} if case["op"] == "read" else {"out": a, "lse": b}
