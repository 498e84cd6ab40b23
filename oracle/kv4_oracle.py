"""64-bit restatement of the 4-bit paged KV cache operators (test
infrastructure): the number format, the record's bytes, the rotation and
attention, from their formulas in include/bfp200.h."""
import numpy as np


def quantize(v):
    """v [..., HD] -> (m int [-8, 7], e int [-17, 12] per tile of 16)."""
    t = np.asarray(v, np.float64).reshape(v.shape[:-1] + (-1, 16))
    a = np.abs(t)
    top = np.where(np.isnan(a), 0.0, a).max(-1)
    with np.errstate(all="ignore"):
        e = np.where(top > 0, np.frexp(np.minimum(top, 1e300))[1], -99)
        e = np.clip(np.where(np.isinf(top), 99, e), -17, 12)
        m = np.rint(np.where(np.isnan(t), 0.0, t) * 2.0 ** (3 - e[..., None]))
    return np.clip(m, -8, 7).astype(int).reshape(v.shape), e


def value(m, e):
    return m * 2.0 ** (np.repeat(e, 16, axis=-1) - 3)


def addresses(slot, page, HD):
    """(key byte, value byte, key exponent, value exponent) of the dims of the
    position at `slot` of a page; dim d is in the byte's high nibble if odd."""
    d = np.arange(HD)
    kb = slot // 4 * (HD // 8) * 16 + d // 8 * 16 + slot % 4 * 4 + d % 8 // 2
    vb = page * HD // 2 + slot // 8 * (HD // 4) * 16 + d // 4 * 16 + slot % 4 * 4 + slot % 8 // 4 * 2 + d % 4 // 2
    ke = page * HD + d // 16 * page + slot
    return kb, vb, ke, ke + page * HD // 16


def put(rec, slot, page, k, v):
    """Writes one position's float keys and values [HD] into a record (uint8)."""
    HD = k.shape[-1]
    for x, at, ex in zip((k, v), addresses(slot, page, HD)[:2], addresses(slot, page, HD)[2:]):
        m, e = quantize(x)
        n = (m + 8).astype(np.uint8)
        rec[at[0::2]] = n[0::2] | (n[1::2] << 4)
        rec[ex[0::16]] = e + 18


def put_pages(pool, k, v):
    """Whole pages: float keys and values [n, H, page, HD] into records pool [n, H, record] (uint8)."""
    page, HD = k.shape[2:]
    for x, which in ((k, 0), (v, 1)):
        m, e = quantize(x)
        n = (m + 8).astype(np.uint8)
        for slot in range(page):
            at, ex = addresses(slot, page, HD)[which], addresses(slot, page, HD)[2 + which]
            pool[..., at[0::2]] = n[:, :, slot, 0::2] | (n[:, :, slot, 1::2] << 4)
            pool[..., ex[0::16]] = e[:, :, slot] + 18


def get(rec, slot, page, HD):
    kb, vb, ke, ve = addresses(slot, page, HD)
    sh = np.where(np.arange(HD) % 2, 4, 0)
    return tuple(((rec[at] >> sh & 15).astype(np.float64) - 8) * 2.0 ** (rec[ex].astype(np.float64) - 21)
                 for at, ex in ((kb, ke), (vb, ve)))


def rotate32(x, cs, rot, inter, inverse=False):
    """Rotation of x [tokens, heads, HD] float32 by cs [tokens, rot / 2, 2]
    float32, every product and sum rounded to float32."""
    y = np.array(x, np.float32)
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    if inverse:
        s = -s
    i = np.arange(rot // 2)
    ia, ib = (2 * i, 2 * i + 1) if inter else (i, i + rot // 2)
    a, b = y[..., ia], y[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
    return y


def visible(length, n_q, causal, window):
    """[n_q, length] truth values."""
    qp = length - n_q + np.arange(n_q)[:, None]
    kp = np.arange(length)[None]
    see = (qp >= 0) & (kp < length)
    if causal:
        see = see & (kp <= qp)
    if window:
        see = see & (kp > qp - window)
    return see


def attention(q, k, v, see, scale):
    """q [n_q, HQ, HD], k, v [len, H, HD], see [n_q, len] -> out, lse, and
    per (query, head) the sum of |q k| scale of the largest score."""
    g = q.shape[1] // k.shape[1]
    out = np.zeros(q.shape)
    lse = np.full(q.shape[:2], -np.inf)
    mag = np.zeros(q.shape[:2])
    for h in range(q.shape[1]):
        kh, vh = k[:, h // g], v[:, h // g]
        with np.errstate(all="ignore"):
            s = np.where(see, q[:, h] @ kh.T * scale, -np.inf)
        for i in range(len(q)):
            if not see[i].any():
                continue
            top = s[i].max()
            w = np.where(see[i], np.exp(s[i] - top), 0.0)
            out[i, h] = w @ np.where(see[i][:, None], vh, 0.0) / w.sum()
            lse[i, h] = top + np.log(w.sum())
            mag[i, h] = (np.abs(q[i, h]) * np.abs(kh[see[i]])).sum(-1).max() * abs(scale)
    return out, lse, mag
