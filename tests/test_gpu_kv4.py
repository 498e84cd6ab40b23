"""The 4-bit paged KV cache operators on the GPU (bfp200.kv4) against their
64-bit restatement (oracle/kv4_oracle.py).  rope, append and read are held to
equality: each is single 32-bit operations of fixed order, then one rounding
to the output type or to 4 bits.

Attention's tolerance, for values up to V and scores whose products' absolute
values sum to at most M: scores are off by (HD + 8) 2^-23 M from their 32-bit
sums, the exponential by 2^-21, a weight by its rounding u (2^-11 where the
result is bfloat16, 2^-21 otherwise), sums over N positions by N 2^-24; a
relative error r of every weight moves the result by at most 2 r V.  The
result is then rounded to its type, whose smallest step is 2^-24 in
binary16."""
import numpy as np
import pytest

from oracle import kv4_oracle as O

pytestmark = pytest.mark.gpu

DTYPES = ["float32", "float16", "bfloat16"]
U_OUT = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
U_P = {"float32": 2.0 ** -21, "float16": 2.0 ** -21, "bfloat16": 2.0 ** -11}


def _dt(name):
    import torch
    return getattr(torch, name)


def _f64(t):
    return t.detach().double().cpu().numpy()


def _f32(t):
    return t.detach().float().cpu().numpy()


def _rounded(a, dtype):
    """float32 numpy -> the torch dtype and back, as float64."""
    import torch
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.float32)).to(_dt(dtype)).double().numpy()


def _i32(a):
    import torch
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def _rand(rng, shape, dtype, scale=1.0):
    import torch
    a = rng.standard_normal(shape) * scale
    if shape[-1] > 3:
        a[..., rng.integers(shape[-1])] *= 7.0                     # a channel larger than the rest
    return torch.from_numpy(a).to(_dt(dtype)).cuda()


class Case:
    """A batch with a filled cache: numpy k, v per sequence (what the cache
    holds) and the torch tensors."""

    def __init__(self, rng, lens, news, H, HD, page, spare_bytes=0xFF, extra_cols=1, scale=1.0):
        import torch
        from bfp200 import kv4
        self.H, self.HD, self.page = H, HD, page
        self.lens, self.news = list(lens), list(news)
        used = [-(-L // page) for L in self.lens]
        n_pages = sum(used) + 2
        order = rng.permutation(n_pages)
        cols = max(used + [0]) + extra_cols
        bt = np.full((len(self.lens), cols), -1)
        at = 0
        pool = np.full((n_pages, H, page * HD * 9 // 8), spare_bytes, np.uint8)   # bytes of no position: anything
        self.kv = []
        for s, L in enumerate(self.lens):
            bt[s, :used[s]] = order[at:at + used[s]]
            at += used[s]
            k, v = (rng.standard_normal((L, H, HD)) * scale for _ in range(2))
            for p in range(L):
                for h in range(H):
                    O.put(pool[bt[s, p // page], h], p % page, page, k[p, h], v[p, h])
            self.kv.append(tuple(O.value(*O.quantize(x)) for x in (k, v)) if L else (k, v))
        self.bt_np, self.pool_np = bt, pool
        self.bt, self.len_t, self.q_start = _i32(bt), _i32(self.lens), _i32(np.concatenate([[0], np.cumsum(self.news)]))
        self.pool = torch.from_numpy(pool.reshape(n_pages, H, page, HD * 9 // 8)).cuda()
        assert kv4.new_pool(n_pages, H, HD, page).shape == self.pool.shape
        self.tokens = int(sum(self.news))


def _check(case, q, dtype, out, lse, scale, causal, window):
    qn, on, ln = _f64(q), _f64(out), lse.double().cpu().numpy()
    t = 0
    for s, (L, n) in enumerate(zip(case.lens, case.news)):
        rows = slice(t, t + n)
        t += n
        if not n:
            continue
        k, v = case.kv[s]
        want, wl, mag = O.attention(qn[rows], k, v, O.visible(L, n, causal, window), scale)
        V = np.abs(v).max() if L else 0.0
        ds = (case.HD + 8) * 2.0 ** -23 * mag + 2.0 ** -21 + L * 2.0 ** -24
        tol = 2 * (ds + U_P[dtype])[..., None] * V
        tol = tol + U_OUT[dtype] * (np.abs(want) + tol) + (2.0 ** -25 if dtype == "float16" else 0.0)
        assert (np.abs(on[rows] - want) <= tol).all(), (s, np.abs(on[rows] - want).max(), tol.min())
        dead = np.isinf(wl)
        assert np.array_equal(dead, np.isinf(ln[rows])) and (ln[rows][dead] < 0).all() and (on[rows][dead] == 0).all()
        assert (np.abs(ln[rows][~dead] - wl[~dead]) <= ds[~dead] + 2.0 ** -22 * np.abs(wl[~dead])).all()


def _attend(case, q, dtype, scale=None, causal=True, window=0, **kw):
    from bfp200 import kv4
    out, lse = kv4.attention(q, case.pool, case.q_start, case.len_t, case.bt, scale=scale, causal=causal, window=window,
                             return_lse=True, **kw)
    _check(case, q, dtype, out, lse, case.HD ** -0.5 if scale is None else scale, causal, window)
    return out, lse


# ---- rope ----------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,H,HD,rot", [(1, 12, 64, 64), (7, 3, 128, 64), (33, 5, 80, 40), (3, 1, 6, 2), (130, 2, 96, 24),
                                        (5, 2, 33, 30), (4, 9, 64, 0), (257, 40, 256, 128), (0, 3, 64, 64), (2, 0, 64, 64)])
@pytest.mark.parametrize("inter", [False, True])
def test_rope(T, H, HD, rot, inter, dtype):
    import torch
    from bfp200 import kv4
    rng = np.random.default_rng(T * 1000 + HD + rot)
    x = _rand(rng, (T, H, HD), dtype)
    pos = rng.integers(0, 500, T)
    table = kv4.rope_table(500, rot) if rot else torch.empty((500, 0, 2), device="cuda")
    cs = table.cpu().numpy()[pos]
    for inverse in (False, True):
        got = kv4.rope(x, _i32(pos), table, interleaved=inter, inverse=inverse)
        assert got.dtype == x.dtype and got.shape == x.shape
        assert np.array_equal(_f64(got), _rounded(O.rotate32(_f32(x), cs, rot, inter, inverse), dtype))


@pytest.mark.parametrize("dtype", DTYPES)
def test_rope_strides_alignment_and_in_place(dtype):
    import torch
    from bfp200 import kv4
    rng = np.random.default_rng(5)
    table = kv4.rope_table(64, 64)
    pos = rng.integers(0, 64, 9)
    cs = table.cpu().numpy()[pos]
    wide = _rand(rng, (9, 8, 64), dtype)
    flat = _rand(rng, (1, 1, 9 * 4 * 64 + 1), dtype)[0, 0]
    forms = [wide[:, 2:5], wide.transpose(0, 1).contiguous().transpose(0, 1), flat[1:].view(9, 4, 64), wide[:, ::3],
             flat[:9 * 4 * 64 - 3 * 64].as_strided((9, 3, 64), (3 * 64 + 1, 64, 1)), wide[:1].expand(9, 8, 64)]
    for x in forms:
        for inter in (False, True):
            want = _rounded(O.rotate32(_f32(x), cs, 64, inter), dtype)
            assert np.array_equal(_f64(kv4.rope(x, _i32(pos), table, interleaved=inter)), want)
    out = torch.full((9, 8, 64), 3.0, dtype=wide.dtype, device="cuda")
    want = _rounded(O.rotate32(_f32(wide[:, 1:4]), cs, 64, False), dtype)
    kv4.rope(wide[:, 1:4], _i32(pos), table, out=out[:, 5:8])
    assert np.array_equal(_f64(out[:, 5:8]), want) and (out[:, :5] == 3).all()
    kv4.rope(wide[:, 1:4], _i32(pos), table, out=wide[:, 1:4])
    assert np.array_equal(_f64(wide[:, 1:4]), want)


def test_rope_positions_outside_the_table_take_its_ends():
    import torch
    from bfp200 import kv4
    x = _rand(np.random.default_rng(0), (4, 2, 64), "float32")
    table = kv4.rope_table(16, 64)
    got = kv4.rope(x, _i32([-5, 0, 15, 2 ** 31 - 1]), table)
    assert torch.equal(got, kv4.rope(x, _i32([0, 0, 15, 15]), table))


@pytest.mark.parametrize("inter", [False, True])
def test_rope_inverse_is_the_gradient(inter):
    """d <rope(x), g> / dx against differences; rope is linear, so a
    difference over a step of 1 has only rounding errors: 96 dims of products
    rounded to 32 bits, each value below 40."""
    from bfp200 import kv4
    rng = np.random.default_rng(8)
    x, g = _rand(rng, (3, 2, 96), "float32"), _rand(rng, (3, 2, 96), "float32")
    table, pos = kv4.rope_table(100, 48), _i32([3, 99, 41])
    grad = _f64(kv4.rope(g, pos, table, interleaved=inter, inverse=True))
    base = _f64(kv4.rope(x, pos, table, interleaved=inter))
    for _ in range(24):
        i = tuple(rng.integers(n) for n in x.shape)
        y = x.clone()
        y[i] += 1.0
        step = float(y[i]) - float(x[i])
        diff = ((_f64(kv4.rope(y, pos, table, interleaved=inter)) - base) * _f64(g)).sum()
        assert abs(diff - grad[i] * step) <= 4 * 40 * 40 * 2.0 ** -23
    back = kv4.rope(kv4.rope(x, pos, table, interleaved=inter), pos, table, interleaved=inter, inverse=True)
    assert np.abs(_f64(back) - _f64(x)).max() <= 8 * 40 * 2.0 ** -23


# ---- append and read -------------------------------------------------------------------------------------------------------

def _append_check(rng, dtype, lens, news, HQ, H, HD, page, rot, inter, k, v, q, positions=None, table_len=None):
    """Appends to a pool of known bytes and compares every byte of it."""
    import torch
    from bfp200 import kv4
    case = Case(rng, lens, news, H, HD, page, spare_bytes=0xA5)
    cap = case.bt_np.shape[1] * page
    table = kv4.rope_table(table_len or cap, rot) if rot else None
    seq = np.repeat(np.arange(len(lens)), news)
    pos = np.concatenate([np.arange(L - n, L) for L, n in zip(lens, news)]).astype(int)
    rp = pos if positions is None else positions
    kr, qr, vr = _f32(k), None if q is None else _f32(q), _f32(v)
    if rot:
        cs = table.cpu().numpy()[np.clip(rp, 0, table.shape[0] - 1)]
        kr = O.rotate32(kr, cs, rot, inter)
        qr = None if q is None else O.rotate32(qr, cs, rot, inter)
    want = case.pool_np.copy()
    for t in range(len(pos)):
        if pos[t] < 0 or pos[t] // page >= case.bt_np.shape[1]:
            continue
        pg = case.bt_np[seq[t], pos[t] // page]
        for h in range(H):
            if pg >= 0:
                O.put(want[pg, h], pos[t] % page, page, kr[t, h], vr[t, h])
    got = kv4.append(case.pool, k, v, case.q_start, case.len_t, case.bt, q=q, table=table, interleaved=inter,
                     positions=None if positions is None else _i32(positions))
    assert np.array_equal(case.pool.cpu().numpy().reshape(want.shape), want)
    if q is None:
        assert got is None
    else:
        assert np.array_equal(_f64(got), _rounded(qr, dtype))
    # and back, as the values that the bytes stand for
    ok = pos >= 0
    for rd in DTYPES:
        rk, rv = kv4.read(case.pool, case.q_start, case.len_t, case.bt, case.tokens, dtype=_dt(rd))
        for x, y in ((rk, kr), (rv, vr)):
            wantv = O.value(*O.quantize(y)) if len(y) else y
            assert np.array_equal(_f64(x)[ok], wantv[ok])
            assert (_f64(x)[~ok] == 0).all()
    return case


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("HD,rot", [(32, 32), (64, 64), (64, 32), (96, 96), (96, 24), (128, 128), (128, 6), (64, 0)])
@pytest.mark.parametrize("inter", [False, True])
def test_append(HD, rot, inter, dtype):
    rng = np.random.default_rng(HD + rot)
    lens, news = [37, 1, 130, 5, 16], [37, 1, 3, 0, 9]
    T, H, HQ = sum(news), 3, 9
    qkv = _rand(rng, (T, HQ + 2 * H, HD), dtype)
    _append_check(rng, dtype, lens, news, HQ, H, HD, 16, rot, inter, qkv[:, HQ:HQ + H], qkv[:, HQ + H:], qkv[:, :HQ])


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_append_pages_heads_and_positions(page):
    rng = np.random.default_rng(page)
    lens, news = [300, 0, 255, 257], [3, 0, 255, 1]
    T = sum(news)
    k, v = _rand(rng, (T, 1, 64), "bfloat16"), _rand(rng, (T, 1, 64), "bfloat16")
    q = _rand(rng, (T, 7, 64), "bfloat16")
    _append_check(rng, "bfloat16", lens, news, 7, 1, 64, page, 64, False, k, v, q, positions=rng.integers(-3, 900, T),
                  table_len=800)
    _append_check(rng, "bfloat16", lens, news, 0, 1, 64, page, 64, False, k, v, None)


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_unaligned_and_broadcast(dtype):
    rng = np.random.default_rng(3)
    flat = _rand(rng, (1, 1, 5 * 6 * 64 + 3), dtype)[0, 0]
    x = flat[3:].view(5, 6, 64)
    _append_check(rng, dtype, [5], [5], 2, 2, 64, 16, 64, False, x[:, :2], x[:, 2:4], x[:, 4:])
    one = _rand(rng, (5, 1, 64), dtype)
    _append_check(rng, dtype, [9], [5], 2, 3, 64, 16, 64, True, one.expand(5, 3, 64), one.expand(5, 3, 64), one.expand(5, 2, 64))


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_extreme_values(dtype):
    """Zeros, values below and above the exponent window, infinities and NaN:
    a tile keeps its finite elements' rounding, infinities saturate, NaN is 0."""
    import torch
    rng = np.random.default_rng(4)
    k = _rand(rng, (8, 2, 64), dtype)
    v = _rand(rng, (8, 2, 64), dtype)
    k[0] = 0
    k[1, 0, :16] = 1e-7
    k[2] *= 3000.0
    k[3, 0, 5] = float("inf")
    k[3, 1, 17] = float("-inf")
    k[4, 0, 20] = float("nan")
    k[5, 1] = float("nan")
    v[6] = torch.finfo(v.dtype).max
    v[7] = -torch.finfo(v.dtype).tiny
    v[5, 0, 3] = 8.0
    v[5, 0, 4] = -7.999
    _append_check(rng, dtype, [8], [8], 0, 2, 64, 16, 0, False, k, v, None)


def test_append_skips_what_has_no_place():
    """More tokens than positions, table entries outside the pool, lengths past
    the table: nothing is written for those, every other byte is right."""
    import torch
    from bfp200 import kv4
    rng = np.random.default_rng(6)
    k, v = _rand(rng, (6, 1, 32), "float32"), _rand(rng, (6, 1, 32), "float32")
    pool = torch.full((3, 1, 16, 36), 0x5A, dtype=torch.uint8, device="cuda")
    before = pool.clone()
    for lens, bt, q_start in [([2], [[7]], [0, 6]), ([2], [[-1]], [0, 6]), ([6 + 16], [[0]], [0, 6]), ([-4], [[0]], [0, 6]),
                              ([3], [[0]], [9, 12]), ([2 ** 31 - 1], [[0]], [0, 6])]:
        kv4.append(pool, k, v, _i32(q_start), _i32(lens), _i32(bt))
        assert torch.equal(pool, before)
        rk, rv = kv4.read(pool, _i32(q_start), _i32(lens), _i32(bt), 6)
        assert not rk.any() and not rv.any()
    kv4.append(pool, k, v, _i32([0, 6]), _i32([4]), _i32([[1]]))           # tokens 0 and 1 lie before the sequence
    assert torch.equal(pool[[0, 2]], before[[0, 2]])
    rk, _ = kv4.read(pool, _i32([0, 6]), _i32([4]), _i32([[1]]), 6, dtype=torch.float32)
    assert not rk[:2].any() and np.array_equal(_f64(rk[2:]), O.value(*O.quantize(_f64(k[2:]))))


def test_append_queries_in_place():
    import torch
    from bfp200 import kv4
    rng = np.random.default_rng(12)
    case = Case(rng, [40], [40], 2, 64, 32)
    k, v, q = (_rand(rng, (40, h, 64), "float16") for h in (2, 2, 4))
    table = kv4.rope_table(128, 64)
    want = kv4.append(case.pool, k, v, case.q_start, case.len_t, case.bt, q=q, table=table)
    again = kv4.append(case.pool, k, v, case.q_start, case.len_t, case.bt, q=q, table=table, q_out=q)
    assert again is q and torch.equal(q, want)


# ---- attention --------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("HD", [32, 64, 96, 128])
@pytest.mark.parametrize("group", [1, 3, 5, 8, 11])
def test_attention_single_tokens(HD, group, dtype):
    rng = np.random.default_rng(HD * 100 + group)
    lens = [1, 0, 15, 16, 17, 31, 32, 33, 64, 100, 257, 300]
    case = Case(rng, lens, [1] * len(lens), 2, HD, 16)
    _attend(case, _rand(rng, (case.tokens, 2 * group, HD), dtype), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 1), (True, 40), (False, 7)])
def test_attention_ragged_prompts_and_masks(page, causal, window, dtype):
    """Prompts, chunks behind a cached prefix, single tokens, a sequence
    without tokens, one without positions and one with fewer positions than
    tokens (its first rows see nothing)."""
    rng = np.random.default_rng(page + window)
    lens, news = [50, 129, 70, 33, 0, 3, 64, 300], [50, 20, 1, 0, 1, 5, 64, 2]
    case = Case(rng, lens, news, 2, 64, page)
    _attend(case, _rand(rng, (case.tokens, 6, 64), dtype), dtype, causal=causal, window=window)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("HD", [32, 64, 96, 128])
@pytest.mark.parametrize("group", [1, 2, 3, 8])
def test_attention_prompts(HD, group, dtype):
    rng = np.random.default_rng(HD + group)
    case = Case(rng, [150, 97, 260], [150, 97, 130], 1, HD, 32)
    _attend(case, _rand(rng, (case.tokens, group, HD), dtype), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [1, 3, 9])
def test_attention_long_axis_is_split(dtype, new):
    rng = np.random.default_rng(new)
    case = Case(rng, [5000], [new], 1, 64, 64)
    _attend(case, _rand(rng, (new, 3, 64), dtype), dtype)
    _attend(case, _rand(rng, (new, 3, 64), dtype), dtype, window=3001)


@pytest.mark.parametrize("HD,page", [(64, 64), (128, 16)])
def test_attention_many_prompt_items(HD, page):
    """More items than CTAs, of one and of two tiles of 128 rows in turn, cut
    anywhere, with causal tiles of different lengths."""
    import torch
    rng = np.random.default_rng(HD)
    n, H, G = 48, 5, 3
    lens, news = rng.integers(100, 600, n), rng.integers(40, 100, n)
    used = [-(-int(L) // page) for L in lens]
    pool = np.full((sum(used), H, page * HD * 9 // 8), 0xFF, np.uint8)
    k, v = rng.standard_normal((2, sum(used), H, page, HD))
    O.put_pages(pool, k, v)
    case = Case.__new__(Case)
    case.lens, case.news, case.HD, case.page = [int(x) for x in lens], [int(x) for x in news], HD, page
    bt = np.full((n, max(used)), -1)
    first = np.concatenate([[0], np.cumsum(used)])
    case.kv = []
    for s in range(n):
        bt[s, :used[s]] = np.arange(first[s], first[s + 1])
        flat = lambda x: O.value(*O.quantize(x[first[s]:first[s + 1]].transpose(0, 2, 1, 3).reshape(-1, H, HD)[:lens[s]]))
        case.kv.append((flat(k), flat(v)))
    case.bt, case.len_t, case.q_start = _i32(bt), _i32(lens), _i32(np.concatenate([[0], np.cumsum(news)]))
    case.pool = torch.from_numpy(pool.reshape(-1, H, page, HD * 9 // 8)).cuda()
    q = _rand(rng, (int(news.sum()), H * G, HD), "bfloat16")
    _attend(case, q, "bfloat16")
    _attend(case, q, "bfloat16", window=150)


def test_attention_many_sequences():
    rng = np.random.default_rng(77)
    lens = rng.integers(0, 90, 700)
    case = Case(rng, lens, rng.integers(0, 3, 700), 1, 32, 16)
    _attend(case, _rand(rng, (case.tokens, 2, 32), "bfloat16"), "bfloat16")


@pytest.mark.parametrize("scale", [0.0, -0.3, 3.0])
def test_attention_scales(scale):
    rng = np.random.default_rng(1)
    case = Case(rng, [90, 40], [2, 40], 2, 64, 16)
    _attend(case, _rand(rng, (42, 4, 64), "float32"), "float32", scale=scale)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_over_the_exponent_window(dtype):
    """Cached values from the smallest quantum to the largest: every one is
    exact in the operands."""
    for scale in (2e-6, 1e-3, 700.0):
        rng = np.random.default_rng(2)
        case = Case(rng, [70], [70], 1, 64, 16, scale=scale)
        q = _rand(rng, (70, 2, 64), dtype, scale=min(1.0 / scale, 1.0))
        _attend(case, q, dtype)


@pytest.mark.parametrize("spare", [0x00, 0x7F, 0xFF])
@pytest.mark.parametrize("HD", [64, 96])
def test_attention_ignores_bytes_of_no_position(spare, HD):
    """Whatever lies past a sequence's end, in pages before a window and in
    pages of nobody (as exponents: infinities and NaN) changes nothing."""
    import torch
    from bfp200 import kv4
    rng = np.random.default_rng(9)
    lens, news = [37, 200, 161], [37, 1, 100]
    case = Case(rng, lens, news, 2, HD, 16, spare_bytes=spare)
    q = _rand(rng, (case.tokens, 6, HD), "bfloat16")
    _attend(case, q, "bfloat16")
    want, lw = _attend(case, q, "bfloat16", window=20)
    bt = case.bt.clone()
    bt[0, 3:], bt[1, 13:], bt[2, 11:] = 0, 0, 0                       # unused entries: any page of the pool
    bt[1, :11] = -1                                                   # freed behind the window
    out, lse = kv4.attention(q, case.pool, case.q_start, case.len_t, bt, window=20, return_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, lw)


def test_attention_pages_outside_the_pool_read_as_zeros():
    import torch
    from bfp200 import kv4
    rng = np.random.default_rng(10)
    case = Case(rng, [64], [1], 1, 64, 16)
    bt = case.bt.clone()
    bt[0, 1], bt[0, 2] = -1, 10 ** 6
    k, v = case.kv[0]
    k[16:48] = 0
    v[16:48] = 0
    q = _rand(rng, (1, 3, 64), "float32")
    out, lse = kv4.attention(q, case.pool, case.q_start, case.len_t, bt, return_lse=True)
    _check(case, q, "float32", out, lse, 64 ** -0.5, True, 0)


@pytest.mark.parametrize("new", [1, 70])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_attention_a_bad_query_stays_alone(bad, new):
    import torch
    from bfp200 import kv4
    rng = np.random.default_rng(13)
    case = Case(rng, [90, 90], [new, new], 1, 64, 16)
    for dtype in DTYPES:
        q = _rand(rng, (2 * new, 3, 64), dtype)
        want = kv4.attention(q, case.pool, case.q_start, case.len_t, case.bt)
        q[0, 1, 7] = bad
        got = kv4.attention(q, case.pool, case.q_start, case.len_t, case.bt)
        assert torch.isnan(got[0, 1]).all()
        got[0, 1] = want[0, 1]
        assert torch.equal(got, want)


def test_attention_strided_and_unaligned():
    import torch
    rng = np.random.default_rng(14)
    for new in (1, 60):
        case = Case(rng, [60, 200], [new, new], 2, 64, 32)
        for dtype in DTYPES:
            wide = _rand(rng, (2 * new, 9, 64), dtype)
            flat = _rand(rng, (1, 1, 2 * new * 4 * 64 + 1), dtype)[0, 0]
            out = torch.full((2 * new, 10, 64), 5.0, dtype=wide.dtype, device="cuda")
            for q in (wide[:, 3:7], wide[:, ::2][:, :4], flat[1:].view(2 * new, 4, 64), wide[:, :1].expand(2 * new, 4, 64)):
                _attend(case, q, dtype, out=out[:, 2:6])
                assert (out[:, :2] == 5).all() and (out[:, 6:] == 5).all()
            odd = torch.full((2 * new * 4 * 64 + 1,), 5.0, dtype=wide.dtype, device="cuda")
            _attend(case, wide[:, 3:7], dtype, out=odd[1:].view(2 * new, 4, 64))


def test_attention_repeats_and_joins():
    """Same inputs, same bits; and two halves of the keys join by their
    log-sum-exp to the whole (each side within its rounding)."""
    import torch
    from bfp200 import kv4
    rng = np.random.default_rng(15)
    case = Case(rng, [4096], [1], 3, 64, 64)
    q = _rand(rng, (1, 9, 64), "float32")
    a, la = _attend(case, q, "float32")
    for _ in range(3):
        b, lb = kv4.attention(q, case.pool, case.q_start, case.len_t, case.bt, return_lse=True)
        assert torch.equal(a, b) and torch.equal(la, lb)
    half = case.bt[:, 32:].contiguous()
    o1, l1 = kv4.attention(q, case.pool, case.q_start, _i32([2048]), case.bt, return_lse=True)
    o2, l2 = kv4.attention(q, case.pool, case.q_start, _i32([2048]), half, return_lse=True)
    w = torch.softmax(torch.stack([l1, l2]).double(), 0)[..., None]
    assert ((w[0] * o1 + w[1] * o2) - a).abs().max() <= 2.0 ** -17


def test_attention_empty_calls():
    import torch
    from bfp200 import kv4
    pool = kv4.new_pool(0, 2, 64)
    q = torch.empty((0, 4, 64), device="cuda")
    out, lse = kv4.attention(q, pool, _i32([0]), _i32([]), _i32(np.zeros((0, 0))), return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    q = torch.ones((2, 4, 64), device="cuda")
    out, lse = kv4.attention(q, pool, _i32([0, 1, 2]), _i32([0, 0]), _i32(np.zeros((2, 0))), return_lse=True)
    assert not out.any() and torch.isinf(lse).all()
    out, lse = kv4.attention(q, pool, _i32([0, 1, 2]), _i32([5, 0]), _i32([[0], [0]]), return_lse=True)  # no such page
    assert not out.any() and abs(float(lse[0, 0]) - np.log(5)) < 1e-6 and torch.isinf(lse[1]).all()


def test_pool_beyond_32_bit_offsets():
    """A pool of more than 2^32 bytes, used at its far end."""
    import torch
    from bfp200 import kv4
    rng = np.random.default_rng(16)
    page, H, HD = 256, 8, 128
    n_pages = (1 << 32) // (H * page * HD * 9 // 8) + 40
    pool = kv4.new_pool(n_pages, H, HD, page)
    L = 300
    k, v, q = (_rand(rng, (L, h, HD), "bfloat16") for h in (H, H, H))
    bt, lens, qs = _i32([[n_pages - 1, n_pages - 2]]), _i32([L]), _i32([0, L])
    kv4.append(pool, k, v, qs, lens, bt)
    rk, rv = kv4.read(pool, qs, lens, bt, L, dtype=torch.float32)
    kn, vn = O.value(*O.quantize(_f64(k))), O.value(*O.quantize(_f64(v)))
    assert np.array_equal(_f64(rk), kn) and np.array_equal(_f64(rv), vn)
    out, lse = kv4.attention(q[-2:], pool, _i32([0, 2]), lens, bt, return_lse=True)
    case = Case.__new__(Case)
    case.lens, case.news, case.kv, case.HD = [L], [2], [(kn, vn)], HD
    _check(case, q[-2:], "bfloat16", out, lse, HD ** -0.5, True, 0)


# ---- streams, graphs, refusals ------------------------------------------------------------------------------------------------

def test_streams_and_graph_capture():
    """A decode step captured once and replayed with lengths updated on the
    device; and two streams at once."""
    import torch
    from bfp200 import kv4
    rng = np.random.default_rng(17)
    H, HQ, HD, page, n = 2, 6, 64, 16, 5
    case = Case(rng, [10, 40, 3, 77, 16], [1] * n, H, HD, page, extra_cols=4)
    for s in range(n):                                       # pages for the growth
        for c in range(case.bt_np.shape[1]):
            if case.bt_np[s, c] < 0:
                case.bt_np[s, c] = 0
    pool = torch.zeros((n * case.bt_np.shape[1], H, page, HD * 9 // 8), dtype=torch.uint8, device="cuda")
    bt = _i32(np.arange(n * case.bt_np.shape[1]).reshape(n, -1))
    lens = _i32([9, 39, 2, 76, 15])
    qs = _i32(range(n + 1))
    table = kv4.rope_table(bt.shape[1] * page, HD)
    k, v, q = (torch.zeros((n, h, HD), device="cuda") for h in (H, H, HQ))
    steps = [[_rand(rng, (n, h, HD), "float32") for h in (H, H, HQ)] for _ in range(6)]

    def step(pool, lens):
        lens += 1
        qr = kv4.append(pool, k, v, qs, lens, bt, q=q, table=table)
        return kv4.attention(qr, pool, qs, lens, bt)

    eager_pool, eager_lens, want = pool.clone(), lens.clone(), []
    for x in steps:
        for dst, src in zip((k, v, q), x):
            dst.copy_(src)
        want.append(step(eager_pool, eager_lens))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    start = lens.clone()
    with torch.cuda.stream(side):
        step(pool, lens)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(pool, lens)
    lens.copy_(start)
    for x, w in zip(steps, want):
        for dst, src in zip((k, v, q), x):
            dst.copy_(src)
        g.replay()
        assert torch.equal(out, w)
    assert torch.equal(lens, eager_lens)
    # two streams: each has its own workspace
    a = Case(rng, [3000], [1], 1, 64, 64)
    qa = [_rand(rng, (1, 4, 64), "bfloat16") for _ in range(8)]
    want = [kv4.attention(x, a.pool, a.q_start, a.len_t, a.bt) for x in qa]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for i, x in enumerate(qa):
        with torch.cuda.stream(streams[i % 4]):
            got.append(kv4.attention(x, a.pool, a.q_start, a.len_t, a.bt))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_refusals():
    import torch
    from bfp200 import BfpError, _lib, kv4
    q = torch.zeros((2, 4, 64), device="cuda")
    kv = torch.zeros((2, 2, 64), device="cuda")
    pool = torch.zeros((4, 2, 16, 72), dtype=torch.uint8, device="cuda")
    qs, lens, bt = _i32([0, 2]), _i32([2]), _i32([[0, 1]])
    table = kv4.rope_table(64, 64)
    att = lambda *a, **k: lambda: kv4.attention(*a, **k)
    app = lambda *a, **k: lambda: kv4.append(*a, **k)
    rop = lambda *a, **k: lambda: kv4.rope(*a, **k)
    calls = [
        att(q.double(), pool, qs, lens, bt), att(q.cpu(), pool, qs, lens, bt), att(q[0], pool, qs, lens, bt),
        att(q[:, :3], pool, qs, lens, bt), att(q[..., :32], pool, qs, lens, bt), att(q.transpose(1, 2), pool, qs, lens, bt),
        att(q, pool.float(), qs, lens, bt), att(q, pool[:, :, :12].contiguous(), qs, lens, bt), att(q, pool[:, :, ::2], qs, lens, bt),
        att(q, pool, qs.long(), lens, bt), att(q, pool, qs[:1], lens, bt), att(q, pool, qs, lens, bt[0]),
        att(q, pool, qs, lens, bt.cpu()), att(q, pool, qs, lens, bt, window=-1), att(q, pool, qs, lens, bt, scale=float("nan")),
        att(q, pool, qs, lens, bt, scale=float("inf")), att(q, pool, qs, lens, bt, out=q.half()), att(q, pool, qs, lens, bt, out=q[:1]),
        att(torch.zeros((2, 0, 64), device="cuda"), pool, qs, lens, bt),
        app(pool, kv, kv.half(), qs, lens, bt), app(pool, kv, kv[:1], qs, lens, bt), app(pool, kv[:, :1], kv[:, :1], qs, lens, bt),
        app(pool, kv, kv, qs, lens, bt, q=q.half()), app(pool, kv, kv, qs, lens, bt, q_out=q),
        app(pool, kv, kv, qs, lens, bt, positions=lens), app(pool, kv, kv, qs, lens, bt, table=table[:20]),
        app(pool, kv, kv, qs, lens, bt, table=table.double()), app(pool, kv, kv, qs, lens, bt, table=kv4.rope_table(64, 128)),
        app(pool, kv, kv, qs, lens, bt, table=table, positions=lens),
        rop(q, _i32([1]), table), rop(q, torch.zeros(2, device="cuda"), table), rop(q, _i32([0, 1]), kv4.rope_table(8, 66)),
        rop(q, _i32([0, 1]), table.cpu()), rop(q, _i32([0, 1]), table, out=q.half()),
        lambda: kv4.read(pool, qs, lens, bt, 2, dtype=torch.float64), lambda: kv4.read(pool[:, :0], qs, lens, bt, 2),
    ]
    for i, c in enumerate(calls):
        with pytest.raises(BfpError) as e:
            c()
        assert e.value.code == _lib.EINVAL, i
    for c in (lambda: kv4.new_pool(4, 2, 80), lambda: kv4.new_pool(4, 2, 64, page=24), lambda: kv4.rope_table(0, 64)):
        with pytest.raises(ValueError):
            c()
    torch.cuda.synchronize()
    assert kv4.attention(q, pool, qs, lens, bt).shape == q.shape
