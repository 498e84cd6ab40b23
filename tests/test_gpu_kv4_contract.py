"""What bfp200.kv4 does with calls at the edges of its contract, on the GPU:
empty calls, lengths past the table, rows of no sequence, calls without
sequences.  Outputs are filled with NaN beforehand, so that a row that nobody
writes shows.  Attention is held to the tolerance that tests/test_gpu_kv4.py
derives."""
import contextlib

import numpy as np
import pytest

from oracle import kv4_oracle as O
from test_gpu_kv4 import Case, DTYPES, U_OUT, U_P, _dt, _f32, _f64, _i32, _rand, _rounded

pytestmark = pytest.mark.gpu


@contextlib.contextmanager
def _empty_is_nan():
    """Fresh memory from torch's allocator holds NaN (bytes: 255)."""
    import torch
    torch.use_deterministic_algorithms(True)
    try:
        assert torch.utils.deterministic.fill_uninitialized_memory
        assert torch.empty((3,), device="cuda").isnan().all()
        yield
    finally:
        torch.use_deterministic_algorithms(False)


def _visible(pos, n_keys, causal, window):
    """[len(pos), n_keys]: what tokens at positions `pos` see of positions 0 .. n_keys - 1."""
    p, k = np.asarray(pos)[:, None], np.arange(n_keys)[None]
    see = (p >= 0) & (k >= 0)
    if causal:
        see = see & (k <= p)
    if window:
        see = see & (k > p - window)
    return see


def _check_rows(q, k, v, see, out, lse, dtype):
    """Rows of one sequence against the formula."""
    HD = q.shape[-1]
    want, wl, mag = O.attention(_f64(q), k, v, see, HD ** -0.5)
    on, ln = _f64(out), _f64(lse)
    V = np.abs(v).max() if len(v) else 0.0
    ds = (HD + 8) * 2.0 ** -23 * mag + 2.0 ** -21 + len(k) * 2.0 ** -24
    tol = 2 * (ds + U_P[dtype])[..., None] * V
    tol = tol + U_OUT[dtype] * (np.abs(want) + tol) + (2.0 ** -25 if dtype == "float16" else 0.0)
    assert (np.abs(on - want) <= tol).all(), np.abs(on - want).max()
    dead = np.isinf(wl)
    assert np.array_equal(dead, np.isinf(ln)) and (ln[dead] < 0).all() and (on[dead] == 0).all()
    assert (np.abs(ln[~dead] - wl[~dead]) <= ds[~dead] + 2.0 ** -22 * np.abs(wl[~dead])).all()


# (HD, query heads a KV head, tokens a sequence): single tokens and few rows on
# one kernel; more than 32 rows a sequence at heads of 128, or 256 at heads of
# 64, on the prompts' kernel where the type has 16 bits
FORMS = [(64, 3, 1), (64, 8, 4), (128, 8, 12), (64, 8, 40)]


@pytest.mark.parametrize("n_seq", [0, 2])
def test_attention_after_an_empty_call(n_seq):
    """A call without tokens asks for no workspace; the next call still gets its own."""
    import torch
    from bfp200 import kv4
    rng = np.random.default_rng(0)
    case = Case(rng, [700], [1], 1, 64, 16)
    kv4._workspace_bytes.clear()
    q = torch.empty((0, 3, 64), device="cuda")
    bt = torch.zeros((n_seq, 60), dtype=torch.int32, device="cuda")
    out, lse = kv4.attention(q, case.pool, _i32([0] * (n_seq + 1)), _i32([500] * n_seq), bt, return_lse=True)
    assert out.shape == (0, 3, 64) and lse.shape == (0, 3)
    q = _rand(rng, (1, 3, 64), "float32")
    out, lse = kv4.attention(q, case.pool, case.q_start, case.len_t, case.bt, return_lse=True)
    _check_rows(q, *case.kv[0], _visible([699], 700, True, 0), out, lse, "float32")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 9), (False, 0), (False, 9)])
@pytest.mark.parametrize("HD,group,new", FORMS)
def test_attention_lengths_past_the_table(HD, group, new, causal, window, dtype):
    """Tokens keep their positions lens - q_start[s + 1] + t where the table is
    shorter than lens: they see what the table holds of them, as append places
    them.  The sequences end 2 positions past the table, within the call's
    tokens past it, and far past it."""
    from bfp200 import kv4
    rng = np.random.default_rng(HD + new)
    cap = 64
    over = [cap + 2, cap + new, cap, cap + 300, 2 ** 31 - 1]
    case = Case(rng, [cap] * len(over), [new] * len(over), 2, HD, 16, extra_cols=0)
    q = _rand(rng, (case.tokens, 2 * group, HD), dtype)
    out, lse = kv4.attention(q, case.pool, case.q_start, _i32(over), case.bt, causal=causal, window=window, return_lse=True)
    for s, L in enumerate(over):
        rows = slice(s * new, (s + 1) * new)
        see = _visible(L - new + np.arange(new), cap, causal, window)
        _check_rows(q[rows], *case.kv[s], see, out[rows], lse[rows], dtype)


@pytest.mark.parametrize("HD,group,new", FORMS)
def test_append_and_attention_agree_past_the_table(HD, group, new):
    """What append writes of a call that runs past its table, attention sees
    under the mask of the positions that append gave the tokens."""
    import torch
    from bfp200 import kv4
    rng = np.random.default_rng(3)
    new, cap = new + 1, 16
    L = cap + new - 1                                        # the first token still has a place
    k, v, q = (_rand(rng, (new, h, HD), "bfloat16") for h in (1, 1, group))
    pool = torch.full((1, 1, 16, HD * 9 // 8), 0xFF, dtype=torch.uint8, device="cuda")
    args = (pool, _i32([0, new]), _i32([L]), _i32([[0]]))
    kf, vf = (rng.standard_normal((cap, 1, HD)) for _ in range(2))
    rec = pool.cpu().numpy()[0].reshape(1, -1).copy()
    for p in range(cap):
        O.put(rec[0], p, 16, kf[p, 0], vf[p, 0])
    pool.copy_(torch.from_numpy(rec.reshape(tuple(pool.shape))))
    kv4.append(pool, k, v, *args[1:])
    kf[cap - 1], vf[cap - 1] = _f64(k)[0], _f64(v)[0]
    out, lse = kv4.attention(q, *args, return_lse=True)
    _check_rows(q, O.value(*O.quantize(kf)), O.value(*O.quantize(vf)), _visible(L - new + np.arange(new), cap, True, 0), out, lse, "bfloat16")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("HD,group,new", FORMS)
def test_attention_rows_of_no_sequence(HD, group, new, dtype):
    """Rows before q_start[0] and from q_start[n_seq] on give zeros and
    -infinity, in outputs with any strides, and change nothing elsewhere."""
    import torch
    from bfp200 import kv4
    rng = np.random.default_rng(HD * new)
    n, lead, tail = 3, 5, 70
    case = Case(rng, [100] * n, [new] * n, 2, HD, 32)
    T, HQ = lead + n * new + tail, 2 * group
    q = _rand(rng, (T, HQ, HD), dtype)
    qs = case.q_start + lead
    wide = torch.full((T, HQ + 2, HD), float("nan"), dtype=_dt(dtype), device="cuda")
    with _empty_is_nan():
        for out in (None, wide[:, 1:-1]):
            got, lse = kv4.attention(q, case.pool, qs, case.len_t, case.bt, out=out, return_lse=True)
            for s in range(n):
                rows = slice(lead + s * new, lead + (s + 1) * new)
                _check_rows(q[rows], *case.kv[s], _visible(100 - new + np.arange(new), 100, True, 0), got[rows], lse[rows], dtype)
            for rows in (slice(0, lead), slice(lead + n * new, T)):
                assert (got[rows] == 0).all() and (lse[rows] == -torch.inf).all()
        assert wide[:, 0].isnan().all() and wide[:, -1].isnan().all()
        # every row of no sequence: sequences without tokens
        got, lse = kv4.attention(q, case.pool, _i32([T] * (n + 1)), case.len_t, case.bt, return_lse=True)
        assert (got == 0).all() and (lse == -torch.inf).all()
        got, lse = kv4.attention(q, case.pool, _i32([0] * (n + 1)), case.len_t, case.bt, return_lse=True)
        assert (got == 0).all() and (lse == -torch.inf).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [0, 40])
@pytest.mark.parametrize("T", [1, 300])
def test_calls_without_sequences(T, cols, dtype):
    """Tokens of no sequence at all: zeros from read and attention, nothing
    written by append, whose queries are turned by their `positions`, without
    them by position 0."""
    import torch
    from bfp200 import kv4
    rng = np.random.default_rng(T)
    pool = torch.full((2, 2, 16, 72), 0x5A, dtype=torch.uint8, device="cuda")
    before = pool.clone()
    b = (_i32([0]), _i32([]), torch.zeros((0, cols), dtype=torch.int32, device="cuda"))
    k, v, q = (_rand(rng, (T, h, 64), dtype) for h in (2, 2, 6))
    table = kv4.rope_table(640, 64)
    pos = rng.integers(0, 640, T)
    cs = table.cpu().numpy()
    with _empty_is_nan():
        for rd in DTYPES:
            rk, rv = kv4.read(pool, *b, T, dtype=_dt(rd))
            assert (rk == 0).all() and (rv == 0).all()
        out, lse = kv4.attention(q, pool, *b, return_lse=True)
        assert (out == 0).all() and (lse == -torch.inf).all()
        assert torch.equal(kv4.append(pool, k, v, *b, q=q), q)
        got = kv4.append(pool, k, v, *b, q=q, table=table)
        assert np.array_equal(_f64(got), _rounded(O.rotate32(_f32(q), cs[np.zeros(T, int)], 64, False), dtype))
        got = kv4.append(pool, k, v, *b, q=q, table=table, positions=_i32(pos))
        assert np.array_equal(_f64(got), _rounded(O.rotate32(_f32(q), cs[pos], 64, False), dtype))
        assert kv4.append(pool, k, v, *b) is None
    assert torch.equal(pool, before)


def _raw_attention(fn, case, q, out, lse, ws):
    """A C entry point that takes bfp200_kv4_attention_args, causal, on the default stream."""
    import torch
    from bfp200 import _lib, kv4
    args = kv4._ATTENTION.pack(*kv4._batch(case.pool, case.q_start, case.len_t, case.bt, q.shape[0])[1], q.data_ptr(), out.data_ptr(),
                               lse.data_ptr(), ws.data_ptr(), ws.numel(), *q.stride()[:2], *out.stride()[:2], q.shape[1],
                               kv4._DTYPES[q.dtype], 1, 0, q.shape[2] ** -0.5)
    return getattr(_lib.lib(), fn)(args, torch.cuda.current_stream().cuda_stream)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("HD,lens,new", [(128, [90, 50], 30), (64, [3000], 300), (128, [2000] * 40, 64)])
def test_a_wait_that_runs_out_is_reported_to_its_caller(HD, lens, new, dtype):
    """Whole items, one item cut over many CTAs, and more items than CTAs: every
    row is NaN, the status says so, rows of no sequence keep their zeros, the
    next call with the same workspace is right, and a Decoder hears nothing of
    it."""
    import torch
    from bfp200 import BfpConfig, Decoder, _lib, kv4, synth
    rng = np.random.default_rng(HD)
    H, group, lead = 2, 8, 3
    case = Case(rng, lens[:1], [new], H, HD, 64)              # (one filled sequence, read by all)
    case.bt, case.len_t = case.bt.expand(len(lens), -1), _i32(lens)
    case.q_start = _i32(lead + new * np.arange(len(lens) + 1))
    T = lead + new * len(lens)
    q = _rand(rng, (T, H * group, HD), dtype)
    want, wl = kv4.attention(q, case.pool, case.q_start, case.len_t, case.bt, return_lse=True, check_done=True)
    assert not want.isnan().any()
    ws = torch.full((64 << 20,), 0xFF, dtype=torch.uint8, device="cuda")
    status = lambda: _lib.lib().bfp200_kv4_attention_status(ws.data_ptr(), torch.cuda.current_stream().cuda_stream)
    for _ in range(2):
        out, lse = torch.zeros_like(q), torch.zeros((T, H * group), device="cuda")
        assert _raw_attention("bfp200_kv4_wait_probe", case, q, out, lse, ws) == _lib.OK
        assert status() == _lib.ETIMEOUT and "timed out" in _lib.last_error()
        assert out[lead:].isnan().all() and lse[lead:].isnan().all()
        assert (out[:lead] == 0).all() and (lse[:lead] == -torch.inf).all()
        assert _raw_attention("bfp200_kv4_attention_dev", case, q, out, lse, ws) == _lib.OK
        assert status() == _lib.OK
        assert torch.equal(out, want) and torch.equal(lse, wl)
    assert _raw_attention("bfp200_kv4_wait_probe", case, q, out, lse, ws) == _lib.OK
    cfg = BfpConfig(D=64, H_Q=1, H_KV=1, HD=64, FFN=128, NL=2, VOCAB=64, MAX_CTX=16, max_seqs=1)
    with Decoder(cfg) as dec:
        dec.load_image(synth.synthetic_image(cfg, 5))
        assert len(dec.generate([[1, 2, 3]], 2)[0]) == 5
    assert status() == _lib.ETIMEOUT


def test_the_status_of_calls_without_waits():
    import torch
    from bfp200 import _lib, kv4
    rng = np.random.default_rng(1)
    L, stream = _lib.lib(), torch.cuda.current_stream().cuda_stream
    assert L.bfp200_kv4_attention_status(None, stream) == _lib.OK
    assert L.bfp200_kv4_attention_status(4, stream) == _lib.EINVAL
    case = Case(rng, [700], [1], 1, 64, 16)
    ws = torch.full((64 << 20,), 0xFF, dtype=torch.uint8, device="cuda")
    for dtype in DTYPES:
        q = _rand(rng, (1, 3, 64), dtype)
        out, lse = torch.zeros_like(q), torch.zeros((1, 3), device="cuda")
        assert _raw_attention("bfp200_kv4_wait_probe", case, q, out, lse, ws) == _lib.EINVAL
        ws.fill_(0xFF)
        assert _raw_attention("bfp200_kv4_attention_dev", case, q, out, lse, ws) == _lib.OK
        assert L.bfp200_kv4_attention_status(ws.data_ptr(), stream) == _lib.OK
        kv4.attention(q, case.pool, case.q_start, case.len_t, case.bt, check_done=True)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31, 2 ** 63 - 1])
@pytest.mark.parametrize("HD,group,new", FORMS)
def test_attention_windows_wider_than_any_position(HD, group, new, window, dtype):
    """As without a window, also for tokens before their sequence and far past its table."""
    import torch
    from bfp200 import kv4
    rng = np.random.default_rng(HD)
    case = Case(rng, [112, 112, 112], [new] * 3, 2, HD, 16, extra_cols=0)      # whole pages: the last length claims them all
    lens = _i32([new // 2, 112, 10 ** 9])
    q = _rand(rng, (3 * new, 2 * group, HD), dtype)
    for causal in (True, False):
        want = kv4.attention(q, case.pool, case.q_start, lens, case.bt, causal=causal, return_lse=True)
        got = kv4.attention(q, case.pool, case.q_start, lens, case.bt, causal=causal, window=window, return_lse=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("inter,inverse", [(False, False), (True, False), (False, True)])
def test_rope_hands_its_gradient_on(inter, inverse, dtype):
    """A tensor that requires a gradient gets it, the inverse turn of the
    output's, from a gradient with any strides; the second derivative is the
    turn again."""
    import torch
    from bfp200 import kv4
    rng = np.random.default_rng(2)
    table, pos = kv4.rope_table(100, 48), _i32([3, 99, 41])
    turn = lambda x, inv: kv4.rope(x, pos, table, interleaved=inter, inverse=inv)
    x = _rand(rng, (3, 2, 96), dtype).requires_grad_()
    g = _rand(rng, (3, 2, 96), dtype)
    y = turn(x, inverse)
    assert y.requires_grad and torch.equal(y.detach(), turn(x.detach(), inverse))
    for grad in (g, g.transpose(0, 1).contiguous().transpose(0, 1), g.transpose(1, 2).contiguous().transpose(1, 2), g[:1, :1, :1].expand(3, 2, 96)):
        got, = torch.autograd.grad(y, x, grad, retain_graph=True)
        assert torch.equal(got, turn(grad.contiguous(), not inverse))
    y.sum().backward()
    assert torch.equal(x.grad, turn(torch.ones_like(g), not inverse))
    h = g.clone().requires_grad_()
    first, = torch.autograd.grad(turn(x, inverse), x, h, create_graph=True)
    second, = torch.autograd.grad(first, h, g)
    assert torch.equal(second, turn(g, inverse))
    with torch.no_grad():
        assert not turn(x, inverse).requires_grad


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("n,HD,group,window", [(300, 128, 4, 0), (700, 128, 4, 20), (300, 32, 12, 0)])
def test_attention_prompts_of_many_sequences(n, HD, group, window, dtype):
    """The prompts' kernel over more than 256 sequences, whose schedule is kept
    in chunks of several: among them sequences without tokens, without
    positions and with fewer positions than tokens."""
    from bfp200 import kv4
    rng = np.random.default_rng(n + window)
    lens, news = rng.integers(0, 60, n), rng.integers(0, 26 if HD > 64 else 64, n)
    news[rng.integers(0, n, n // 10)] = 0
    lens[rng.integers(0, n, n // 10)] = 0
    case = Case(rng, lens, news, 1, HD, 16)
    assert case.tokens * group > (32 if HD > 64 else 256) * n     # enough rows a sequence for that kernel
    q = _rand(rng, (case.tokens, group, HD), dtype)
    out, lse = kv4.attention(q, case.pool, case.q_start, case.len_t, case.bt, window=window, return_lse=True)
    t = 0
    for s in range(n):
        L, m = int(lens[s]), int(news[s])
        rows = slice(t, t + m)
        t += m
        if m:
            _check_rows(q[rows], *case.kv[s], _visible(L - m + np.arange(m), L, True, window), out[rows], lse[rows], dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_of_lowest_and_highest_mantissas(dtype):
    """Words whose nibbles are all 0 (mantissa -8, a sum below -2^31) or all 15."""
    import torch
    from bfp200 import kv4
    pool = kv4.new_pool(1, 1, 64, 16)
    k = torch.full((2, 1, 64), -1.99, device="cuda", dtype=_dt(dtype))
    k[1] = 1.99
    args = (pool, _i32([0, 2]), _i32([2]), _i32([[0]]))
    kv4.append(args[0], k, k, *args[1:])
    rk, rv = kv4.read(*args, 2, dtype=torch.float32)
    assert (rk[0] == -2.0).all() and (rk[1] == 1.75).all() and torch.equal(rk, rv)


def test_check_done_waits_for_calls_without_a_workspace():
    import torch
    from bfp200 import kv4
    case = Case(np.random.default_rng(0), [20], [1], 1, 64, 16)
    q = torch.ones((1, 3, 64), device="cuda")
    for t in (1, 0):
        qs = _i32([0, t])
        torch.cuda.synchronize()
        torch.cuda._sleep(100_000_000)                       # some 50 ms
        kv4.attention(q[:t], case.pool, qs, case.len_t, case.bt)
        assert not torch.cuda.current_stream().query()
        kv4.attention(q[:t], case.pool, qs, case.len_t, case.bt, check_done=True)
        assert torch.cuda.current_stream().query()
