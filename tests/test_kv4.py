"""Host side of the 4-bit paged KV cache operators, no GPU: rotation tables,
the oracle's number format against the framework's tile rule, and the C entry
points' refusals (checked before any device is touched)."""
import ctypes as C
import math

import numpy as np
import pytest

from bfp200 import _lib, kv4, ops
from oracle import kv4_oracle as O


def test_frequencies_plain_match_rope_fp():
    """scaling "none" is rope_fp's theta (gen_smollm_blockfp_full.py:253)."""
    f, grow = kv4.rope_frequencies(64)
    assert grow == 1.0
    t = ops.rope_table(50, 64, 10000.0)
    a = np.arange(50)[:, None] * f
    assert np.abs(np.cos(a) - t[..., 0]).max() < 1e-13 and np.abs(np.sin(a) - t[..., 1]).max() < 1e-13


def test_scalings():
    f, _ = kv4.rope_frequencies(64)
    lin, g = kv4.rope_frequencies(64, scaling="linear", factor=4.0)
    assert np.allclose(lin, f / 4, rtol=1e-15) and g == 1.0
    ntk, g = kv4.rope_frequencies(64, scaling="ntk", factor=4.0)
    assert ntk[0] == f[0] and abs(ntk[-1] / (f[-1] / 4) - 1) < 1e-12 and g == 1.0
    assert (np.diff(ntk / f) < 0).all()
    b, g = kv4.rope_frequencies(64, scaling="bands", factor=4.0, original=2048)
    turns = 2048 * f / (2 * math.pi)
    assert np.array_equal(b[turns >= 32], f[turns >= 32]) and np.allclose(b[turns <= 1], f[turns <= 1] / 4, rtol=1e-15)
    mid = (turns > 1) & (turns < 32)
    ramp = (turns - 1) / 31
    assert mid.any() and np.allclose(b[mid], (f / 4 * (1 - ramp) + f * ramp)[mid], rtol=1e-15)
    assert g == pytest.approx(0.1 * math.log(4) + 1)
    for s in kv4.SCALINGS:                                    # a factor of 1 changes nothing
        assert np.allclose(kv4.rope_frequencies(32, scaling=s, factor=1.0)[0], kv4.rope_frequencies(32)[0], rtol=1e-15)
    assert kv4.rope_frequencies(0)[0].size == 0 and kv4.rope_frequencies(2, scaling="ntk", factor=2.0)[0].tolist() == [1.0]


def test_table_values():
    t = kv4.rope_table(300, 32, base=500.0, scaling="bands", factor=2.0, original=100, device="cpu")
    f, g = kv4.rope_frequencies(32, 500.0, "bands", 2.0, 100)
    assert t.shape == (300, 16, 2) and t.is_contiguous()
    for p in (0, 1, 299):
        for j in (0, 7, 15):
            assert float(t[p, j, 0]) == np.float32(math.cos(p * f[j]) * g) and float(t[p, j, 1]) == np.float32(math.sin(p * f[j]) * g)


@pytest.mark.parametrize("kw", [dict(rot_dim=3), dict(rot_dim=-2), dict(rot_dim=8, scaling="x"), dict(rot_dim=8, factor=0.5),
                                dict(rot_dim=8, factor=float("nan")), dict(rot_dim=8, base=1.0),
                                dict(rot_dim=8, scaling="bands", low=3.0, high=2.0), dict(rot_dim=8, scaling="bands", original=0)])
def test_frequency_refusals(kw):
    with pytest.raises(ValueError):
        kv4.rope_frequencies(**kw)


def test_format_follows_the_tile_rule():
    """The framework's tile_quantize with 4-bit mantissas: same exponent, and
    the mantissa of the same quotient on 2^3 instead of 2^15 steps."""
    from oracle import bfp_oracle as B
    rng = np.random.default_rng(0)
    v = rng.standard_normal(1600) * np.repeat(2.0 ** rng.integers(-15, 10, 100), 16)
    m, e = O.quantize(v)
    _, e16 = B.tile_quantize(v)
    assert np.array_equal(e, np.clip(e16, -17, 12))
    assert np.array_equal(m, np.clip(np.rint(v / 2.0 ** np.repeat(e, 16) * 8), -8, 7))
    err = np.abs(O.value(m, e) - v)
    assert (err <= 2.0 ** (np.repeat(e, 16) - 3)).all()       # half a step; a whole one where the top is cut at 7


def test_record_is_a_bijection():
    for page, HD in ((16, 32), (64, 64), (32, 96), (128, 128)):
        seen = np.zeros(page * HD * 9 // 8, int)
        for slot in range(page):
            kb, vb, ke, ve = O.addresses(slot, page, HD)
            for a in (kb, vb):
                np.add.at(seen, a, 1)
            for a in (ke, ve):
                np.add.at(seen, a[::16], 2)
        assert (seen == 2).all()                               # two nibbles a byte, or one exponent


def test_record_roundtrip():
    rng = np.random.default_rng(1)
    page, HD = 32, 96
    rec = np.zeros(page * HD * 9 // 8, np.uint8)
    k, v = rng.standard_normal((2, page, HD)) * 3
    for s in range(page):
        O.put(rec, s, page, k[s], v[s])
    for s in range(page):
        gk, gv = O.get(rec, s, page, HD)
        assert np.array_equal(gk, O.value(*O.quantize(k[s]))) and np.array_equal(gv, O.value(*O.quantize(v[s])))


def _batch(**kw):
    d = dict(pool=4096, bt=4096, qs=4096, lens=4096, n_pages=4, page=16, H=2, HD=64, n=1, cols=2, ld=2, T=2)
    d.update(kw)
    return tuple(d.values())


@pytest.mark.parametrize("kw,what", [(dict(HD=80), "HD"), (dict(page=24), "page"), (dict(H=0), "H_KV"), (dict(T=-1), "negative"),
                                     (dict(n=-1), "negative"), (dict(pool=4104), "aligned"), (dict(pool=0), "pool"),
                                     (dict(qs=0), "q_start"), (dict(bt=0), "block table"), (dict(cols=1 << 40), "2\\^30"),
                                     (dict(T=1 << 40), "too many")])
def test_batch_refusals(kw, what):
    b = _batch(**kw)
    L = _lib.lib()
    for rc in (L.bfp200_kv4_read_dev(kv4._READ.pack(*b, 4096, 4096, 0), None),
               L.bfp200_kv4_append_dev(kv4._APPEND.pack(*b, *[4096] * 4, *[64] * 8, 0, 0, 2, 0, 0, 0, 0), None),
               L.bfp200_kv4_attention_dev(kv4._ATTENTION.pack(*b, *[4096] * 4, 1 << 30, *[64] * 4, 4, 0, 1, 0, 0.125), None)):
        assert rc == _lib.EINVAL
        import re
        assert re.search(what, _lib.last_error()), _lib.last_error()


def test_other_refusals():
    L = _lib.lib()
    att = lambda ws=4096, nb=1 << 30, hq=4, dt=0, win=0, scale=0.125, q=4096: L.bfp200_kv4_attention_dev(
        kv4._ATTENTION.pack(*_batch(), q, 4096, 0, ws, nb, 64, 64, 64, 64, hq, dt, 1, win, scale), None)
    app = lambda table=4096, n_pos=64, rot=64, hq=4, dt=0, k=4096: L.bfp200_kv4_append_dev(
        kv4._APPEND.pack(*_batch(), k, 4096, 4096, 4096, *[64] * 8, table, 0, hq, n_pos, rot, dt, 0), None)
    rope = lambda x=4096, hd=64, rot=64, n_pos=8, dt=0, T=2, table=4096: L.bfp200_rope_dev(
        kv4._ROPE.pack(x, 4096, table, 4096, 64, 64, 64, 64, T, 2, hd, n_pos, rot, dt, 0, 0), None)
    for rc in (att(hq=3), att(hq=0), att(dt=3), att(win=-1), att(scale=math.nan), att(scale=math.inf), att(q=0), att(q=4097),
               att(ws=4100), app(rot=63), app(rot=66), app(rot=-2), app(n_pos=0), app(n_pos=31), app(dt=9), app(k=0), app(k=4098),
               app(table=4100), app(hq=-1), rope(x=0), rope(x=4097), rope(hd=0), rope(rot=65), rope(rot=66), rope(n_pos=0),
               rope(dt=-1), rope(T=-1), rope(table=0), rope(table=4100), L.bfp200_rope_dev(None, None),
               L.bfp200_kv4_append_dev(None, None), L.bfp200_kv4_read_dev(None, None), L.bfp200_kv4_attention_dev(None, None),
               L.bfp200_kv4_attention_workspace(None, None)):
        assert rc == _lib.EINVAL, _lib.last_error()
    # nothing to do: nothing is asked of a device
    assert rope(T=0) == _lib.OK
    assert L.bfp200_kv4_read_dev(kv4._READ.pack(*_batch(T=0, n=0), 0, 0, 0), None) == _lib.OK
    assert C.sizeof(C.c_longlong) * 31 == kv4._APPEND.size


def test_no_cpu_path():
    import torch
    from bfp200 import BfpError
    x = torch.zeros((1, 1, 64))
    with pytest.raises(BfpError):
        kv4.rope(x, torch.zeros(1, dtype=torch.int32), torch.zeros((4, 32, 2)))
