"""A paged KV cache held in 4 bits, and the rotary positions that feed it.

    pool = kv4.new_pool(n_pages, H_KV, HD, page=64)              # uint8, on the current GPU
    table = kv4.rope_table(n_pos, HD, scaling="bands", factor=4)  # (cos, sin), 32-bit
    q = kv4.append(pool, k, v, q_start, lens, block_table, q=q, table=table)
    out = kv4.attention(q, pool, q_start, lens, block_table)

Unlike ``bfp200.ops`` these take and return torch tensors on the GPU and run
on torch's current stream, asynchronously; they keep nothing between calls
(workspaces come from torch's allocator) and can be captured into a graph.
Activations are float32, float16 or bfloat16 ``[tokens, heads, HD]`` with a
contiguous last axis and any other strides (a slice of a fused projection
needs no copy).  The C entry points are ``bfp200_rope_dev`` and
``bfp200_kv4_*_dev`` of include/bfp200.h, which also defines the bytes of the
cache: BFP tiles of 16 head dims, 4-bit mantissas, one exponent byte.

Rotation passes gradients on; append, read and attention have no backward pass,
and what they return carries no gradient.

A batch is three int32 tensors: ``lens[s]`` positions of sequence s, held in
pages ``block_table[s, 0..]``; ``q_start[s] .. q_start[s + 1]`` its rows among
this call's tokens, which are its last positions.  They are read on the
device, so a serving loop updates them there without a synchronization.
"""
from __future__ import annotations

import struct

import numpy as np
import torch

from . import _lib
from ._lib import EINVAL, BfpError, check

PAGES = (16, 32, 64, 128, 256)
HEAD_DIMS = (32, 64, 96, 128)
SCALINGS = ("none", "linear", "ntk", "bands")

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_ROPE = struct.Struct("@16q")
_APPEND = struct.Struct("@31q")
_READ = struct.Struct("@15q")
_ATTENTION = struct.Struct("@25qd")
_workspace_bytes = {}           # (device, HD) -> bytes


def _bad(what):
    raise BfpError(EINVAL, what)


def rope_frequencies(rot_dim, base=10000.0, scaling="none", factor=1.0, original=2048, low=1.0, high=32.0):
    """Angle per position of each of the rot_dim / 2 pairs (float64), and the
    factor that cos and sin are multiplied by.

    none    base^(-2 j / rot_dim)
    linear  the same over `factor`: positions interpolated
    ntk     base * factor^(rot_dim / (rot_dim - 2)): the slowest pair is
            interpolated, the fastest left alone
    bands   pairs that turn at least `high` times within `original` positions
            are left alone, those under `low` turns are interpolated, and a
            linear ramp lies between; cos and sin grow by 0.1 ln(factor) + 1
    """
    if rot_dim < 0 or rot_dim % 2:
        raise ValueError("rot_dim must be even")
    if scaling not in SCALINGS:
        raise ValueError(f"scaling must be one of {SCALINGS}")
    if not factor >= 1.0 or not base > 1.0:
        raise ValueError("factor must be at least 1 and base above 1")
    j = np.arange(0, rot_dim, 2, dtype=np.float64)
    if scaling == "ntk":
        if rot_dim > 2:
            base = base * factor ** (rot_dim / (rot_dim - 2.0))
        return base ** (-j / max(rot_dim, 1)), 1.0
    f = base ** (-j / max(rot_dim, 1))
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "bands":
        if not 0 < low < high or original < 1:
            raise ValueError("bands needs 0 < low < high and original >= 1")
        keep = np.clip((original * f / (2 * np.pi) - low) / (high - low), 0.0, 1.0)
        return f / factor * (1.0 - keep) + f * keep, 0.1 * np.log(factor) + 1.0
    return f, 1.0


def rope_table(n_pos, rot_dim, base=10000.0, scaling="none", factor=1.0, original=2048, low=1.0, high=32.0, device=None):
    """(cos, sin) of every position and pair, float32 [n_pos, rot_dim / 2, 2]
    on the GPU; built in 64 bits on the host (rope_fp's angles, :253-254, where
    scaling is "none")."""
    if n_pos < 1:
        raise ValueError("n_pos must be at least 1")
    f, grow = rope_frequencies(rot_dim, base, scaling, factor, original, low, high)
    a = np.arange(n_pos, dtype=np.float64)[:, None] * f
    t = np.stack([np.cos(a) * grow, np.sin(a) * grow], -1).astype(np.float32)
    return torch.from_numpy(np.ascontiguousarray(t)).to(device or torch.device("cuda"))


def new_pool(n_pages, H_KV, HD, page=64, device=None):
    """An empty pool: uint8 [n_pages, H_KV, page, HD * 9 / 8] (the last two
    axes are one record).  Positions are written by append before they are
    read, so nothing is cleared."""
    if HD not in HEAD_DIMS or page not in PAGES or n_pages < 0 or H_KV < 1:
        raise ValueError(f"HD must be one of {HEAD_DIMS} and page one of {PAGES}")
    return torch.empty((n_pages, H_KV, page, HD * 9 // 8), dtype=torch.uint8, device=device or torch.device("cuda"))


def _fn(name):
    """A C entry point of the library, looked up once."""
    f = _fns.get(name)
    if f is None:
        f = _fns[name] = getattr(_lib.lib(), name)
    return f


_fns = {}
_current_device = getattr(torch._C, "_cuda_getDevice", None) or (lambda: torch.cuda.current_device())
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


def _run(fn, arg, index):
    """Calls a C entry point on torch's current stream of GPU `index`."""
    if _current_device() == index:
        rc = fn(arg, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(arg, _raw_stream(index))
    if rc:
        check(rc)


def _workspace(packed, index):
    n = _lib.C.c_size_t()
    f = _fn("bfp200_kv4_attention_workspace")
    if _current_device() == index:
        check(f(packed, n))
    else:
        with torch.cuda.device(index):
            check(f(packed, n))
    return n.value


def _acts(x, name):
    """An activation tensor's GPU, dtype code, shape and outer strides."""
    code = _DTYPES.get(x.dtype)
    if code is None or x.dim() != 3 or not x.is_cuda:
        _bad(f"{name} must be a [tokens, heads, HD] float32, float16 or bfloat16 tensor on the GPU")
    t, h, d = x.shape
    st, sh, sd = x.stride()
    if sd != 1 and d > 1 and t and h:
        _bad(f"{name}'s last axis must be contiguous")
    return x.get_device(), code, t, h, d, st, sh


def _like(x, name, dev, code, t, h, d):
    """Outer strides of a tensor that has to fit another one."""
    v = _acts(x, name)
    if v[0] != dev:
        _bad(f"{name} is on another device")
    if v[1] != code:
        _bad(f"{name} must have the same dtype as the other tensors")
    if v[2] != t or v[3] != h or v[4] != d:
        _bad(f"{name} has shape {tuple(x.shape)}, which does not fit the other arguments")
    return v[5], v[6]


def _positions(x, dev, tokens):
    if x.dtype != torch.int32 or x.dim() != 1 or x.get_device() != dev or x.shape[0] != tokens \
            or (tokens > 1 and x.stride(0) != 1):
        _bad("positions must be a contiguous int32 tensor on the same GPU with one entry per token")
    return x.data_ptr()


def _batch(pool, q_start, lens, block_table, tokens):
    """The GPU and the 12 words of bfp200_kv4_batch."""
    if pool.dtype != torch.uint8 or pool.dim() != 4 or not pool.is_cuda or not pool.is_contiguous():
        _bad("pool must be a contiguous uint8 [pages, H_KV, page, HD * 9 / 8] tensor on the GPU")
    dev = pool.get_device()
    n_pages, h, page, rec = pool.shape
    if lens.dtype != torch.int32 or q_start.dtype != torch.int32 or block_table.dtype != torch.int32 \
            or lens.dim() != 1 or q_start.dim() != 1 or block_table.dim() != 2:
        _bad("lens [n], q_start [n + 1] and block_table [n, pages] must be int32")
    n, width = block_table.shape
    ld, step = block_table.stride()
    if lens.shape[0] != n or q_start.shape[0] != n + 1:
        _bad("lens [n], q_start [n + 1] and block_table [n, pages] must fit each other")
    if lens.get_device() != dev or q_start.get_device() != dev or block_table.get_device() != dev:
        _bad("lens, q_start and block_table must be on the pool's device")
    if (n > 1 and lens.stride(0) != 1) or q_start.stride(0) != 1 or (width > 1 and step != 1):
        _bad("lens, q_start and block_table's rows must be contiguous")
    if rec % 9:
        _bad("the pool's last axis must be HD * 9 / 8")
    return dev, (pool.data_ptr(), block_table.data_ptr(), q_start.data_ptr(), lens.data_ptr(), n_pages, page, h,
                 rec * 8 // 9, n, width, ld, tokens)


def _table(table, dev):
    if table.dtype != torch.float32 or table.dim() != 3 or table.shape[2] != 2 or table.get_device() != dev \
            or not table.is_contiguous():
        _bad("table must be a contiguous float32 [n_pos, rot / 2, 2] tensor on the same GPU")
    return table.data_ptr(), table.shape[0], table.shape[1] * 2


def rope(x, positions, table, interleaved=False, inverse=False, out=None):
    """x [tokens, heads, HD] with the first rot = 2 * table.shape[1] dims of
    every head turned by its token's angles: pairs (j, j + rot / 2), or (2 j,
    2 j + 1) if interleaved; the other dims are copied.  inverse turns back,
    which is the gradient of the forward turn: an x that requires a gradient
    gets it so.  out may be x; a result in out carries no gradient."""
    if out is None and x.requires_grad and torch.is_grad_enabled():
        return _Rope.apply(x, positions, table, interleaved, inverse)
    dev, code, t, h, d, xt, xh = _acts(x, "x")
    if out is None:
        out = x.new_empty((t, h, d))
        ot, oh = h * d, d
    else:
        ot, oh = _like(out, "out", dev, code, t, h, d)
    pp = _positions(positions, dev, t)
    tp, n_pos, rot = _table(table, dev)
    _run(_fn("bfp200_rope_dev"), _ROPE.pack(x.data_ptr(), out.data_ptr(), tp, pp, xt, xh, ot, oh, t, h, d, n_pos, rot, code,
                                            interleaved, inverse), dev)
    return out


class _Rope(torch.autograd.Function):
    """rope of an x that requires a gradient."""

    @staticmethod
    def forward(ctx, x, positions, table, interleaved, inverse):
        ctx.save_for_backward(positions, table)
        ctx.form = interleaved, inverse
        return rope(x, positions, table, interleaved, inverse)

    @staticmethod
    def backward(ctx, g):
        positions, table = ctx.saved_tensors
        interleaved, inverse = ctx.form
        g = g if g.stride(-1) == 1 else g.contiguous()
        return rope(g, positions, table, interleaved, not inverse), None, None, None, None


def append(pool, k, v, q_start, lens, block_table, q=None, table=None, interleaved=False, positions=None, q_out=None):
    """Writes this call's keys and values [tokens, H_KV, HD] to the cache, at
    their sequences' last positions (lens counts them already).  With a table,
    keys and the queries q [tokens, H_Q, HD] are rotated on the way, by their
    cache positions or by `positions` [tokens].  Returns the rotated queries
    (q_out if given, which may be q), or None without q."""
    dev, code, t, h, d, kt, kh = _acts(k, "k")
    vt, vh = _like(v, "v", dev, code, t, h, d)
    where, b = _batch(pool, q_start, lens, block_table, t)
    if where != dev or b[6] != h or b[7] != d:
        _bad("k and v do not fit the pool's heads, HD or device")
    hq = qt = qh = ot = oh = qp = op = tp = n_pos = rot = pp = 0
    if q is not None:
        hq = q.shape[1] if q.dim() == 3 else 0
        qt, qh = _like(q, "q", dev, code, t, hq, d)
        if q_out is None:
            q_out = q.new_empty((t, hq, d))
            ot, oh = hq * d, d
        else:
            ot, oh = _like(q_out, "q_out", dev, code, t, hq, d)
        qp, op = q.data_ptr(), q_out.data_ptr()
    elif q_out is not None:
        _bad("q_out needs q")
    if table is not None:
        tp, n_pos, rot = _table(table, dev)
        if positions is not None:
            pp = _positions(positions, dev, t)
    elif positions is not None:
        _bad("positions need a table")
    _run(_fn("bfp200_kv4_append_dev"), _APPEND.pack(*b, k.data_ptr(), v.data_ptr(), qp, op, kt, kh, vt, vh, qt, qh, ot, oh, tp,
                                                    pp, hq, n_pos, rot, code, interleaved), dev)
    return q_out


def read(pool, q_start, lens, block_table, tokens, dtype=torch.bfloat16):
    """(k, v) [tokens, H_KV, HD]: what the cache holds for the last q_start[s +
    1] - q_start[s] positions of every sequence (all of them with q_start =
    cumsum of lens).  Exact in every dtype."""
    code = _DTYPES.get(dtype)
    if code is None:
        _bad("dtype must be float32, float16 or bfloat16")
    if tokens < 0:
        _bad("tokens must not be negative")
    dev, b = _batch(pool, q_start, lens, block_table, tokens)
    k = pool.new_empty((tokens, b[6], b[7]), dtype=dtype)
    v = pool.new_empty((tokens, b[6], b[7]), dtype=dtype)
    _run(_fn("bfp200_kv4_read_dev"), _READ.pack(*b, k.data_ptr(), v.data_ptr(), code), dev)
    return k, v


def attention(q, pool, q_start, lens, block_table, scale=None, causal=True, window=0, out=None, return_lse=False,
              check_done=False):
    """Softmax attention of q [tokens, H_Q, HD] over the cached positions of
    the tokens' sequences; H_Q a multiple of H_KV, query head i reads KV head
    i // (H_Q / H_KV).  A token at position p sees the positions k < lens[s]
    with k <= p (causal) and k > p - window (window > 0).  scale defaults to
    HD^-1/2.  Returns out, and with return_lse the log-sum-exp of the scaled
    scores (float32 [tokens, H_Q]) to join it with attention over other keys;
    a token that sees nothing gets zeros and -inf.

    The kernel of prompts has bounded waits; rows that one leaves undone are
    NaN.  check_done waits for the call and raises BfpError (ETIMEOUT) then."""
    dev, code, t, hq, d, qt, qh = _acts(q, "q")
    where, b = _batch(pool, q_start, lens, block_table, t)
    if where != dev or b[7] != d:
        _bad("q does not fit the pool's HD or device")
    if out is None:
        out = q.new_empty((t, hq, d))
        ot, oh = hq * d, d
    else:
        ot, oh = _like(out, "out", dev, code, t, hq, d)
    lse = q.new_empty((t, hq), dtype=torch.float32) if return_lse else None
    small = b[5] * b[9] <= 256                  # a cache that short may need none: asked for each time
    need = 0 if not t or not b[8] else None if small else _workspace_bytes.get((dev, d))
    if need is None:                            # (an empty call needs none, which says nothing of the next one)
        need = _workspace(_ATTENTION.pack(*b, 0, 0, 0, 0, 0, 0, 0, 0, 0, hq, code, 0, 0, 0.0), dev)
        if not small:
            _workspace_bytes[(dev, d)] = need
    ws = q.new_empty((need,), dtype=torch.uint8) if need else None
    _run(_fn("bfp200_kv4_attention_dev"),
         _ATTENTION.pack(*b, q.data_ptr(), out.data_ptr(), lse.data_ptr() if return_lse else 0, ws.data_ptr() if need else 0, need, qt, qh, ot, oh,
                         hq, code, causal, window, d ** -0.5 if scale is None else scale), dev)
    if check_done:
        _run(_fn("bfp200_kv4_attention_status"), ws.data_ptr() if need else None, dev)
    return (out, lse) if return_lse else out
