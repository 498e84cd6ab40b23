"""Edges of the contract of bfp200.kv4 and bfp200.paged that need no GPU."""
import pytest


def _paged():
    """A PagedDecoder without a model, for what generate checks first."""
    import numpy as np
    from bfp200 import paged
    dec = object.__new__(paged.PagedDecoder)
    dec.page, dec.free, dec.table, dec.device = 16, [3, 2, 1, 0], np.zeros((64, 32, 2), np.float32), "cpu"
    return dec


@pytest.mark.parametrize("prompts", [[[]], [[1, 2], []], [[], [1, 2]]])
def test_paged_generate_refuses_empty_prompts(prompts):
    """An empty prompt has no token to go on from (it took the sequence before it's)."""
    dec = _paged()
    with pytest.raises(ValueError, match="at least one id"):
        dec.generate(prompts, 3)
    assert dec.free == [3, 2, 1, 0]


def test_paged_generate_of_no_prompts():
    assert _paged().generate([], 3) == []


def _batch(**kw):
    d = dict(pool=4096, bt=4096, qs=4096, lens=4096, n_pages=4, page=16, H=2, HD=64, n=1, cols=2, ld=2, T=2)
    d.update(kw)
    return tuple(d.values())


def _calls(batch):
    """read, append, attention and its workspace with these words of the batch."""
    from bfp200 import _lib, kv4
    L = _lib.lib()
    att = kv4._ATTENTION.pack(*batch, *[4096] * 4, 1 << 30, *[64] * 4, 4, 0, 1, 0, 0.125)
    return (L.bfp200_kv4_read_dev(kv4._READ.pack(*batch, 4096, 4096, 0), None),
            L.bfp200_kv4_append_dev(kv4._APPEND.pack(*batch, *[4096] * 4, *[64] * 8, 0, 0, 2, 0, 0, 0, 0), None),
            L.bfp200_kv4_attention_dev(att, None), L.bfp200_kv4_attention_workspace(att, _lib.C.c_size_t()))


@pytest.mark.parametrize("which", ["bt", "qs", "lens"])
@pytest.mark.parametrize("off", [1, 2, 3])
def test_misaligned_batch_arrays_are_refused(which, off):
    """The kernels read them as 32-bit words, which at other addresses would be a fault of the GPU."""
    from bfp200 import _lib
    assert _calls(_batch(**{which: 4096 + off})) == (_lib.EINVAL,) * 4
    assert "aligned" in _lib.last_error()


@pytest.mark.parametrize("off", [1, 2, 3])
def test_misaligned_positions_are_refused(off):
    from bfp200 import _lib, kv4
    L = _lib.lib()
    for rc in (L.bfp200_rope_dev(kv4._ROPE.pack(4096, 4096, 4096, 4096 + off, 64, 64, 64, 64, 2, 2, 64, 8, 64, 0, 0, 0), None),
               L.bfp200_kv4_append_dev(kv4._APPEND.pack(*_batch(), *[4096] * 4, *[64] * 8, 4096, 4096 + off, 2, 64, 64, 0, 0), None)):
        assert rc == _lib.EINVAL and "aligned" in _lib.last_error()


@pytest.mark.parametrize("cols,page", [(1 << 60, 16), ((1 << 60) + 5, 16), (1 << 55, 256), ((1 << 63) - 1, 256), ((1 << 26) + 1, 16)])
def test_tables_of_too_many_positions_are_refused(cols, page):
    """Also where max_pages * page passes 64 bits."""
    from bfp200 import _lib
    assert _calls(_batch(cols=cols, page=page, pool=4096)) == (_lib.EINVAL,) * 4
    assert "2^30 positions" in _lib.last_error()


def test_no_exception_leaves_a_c_entry_point():
    """Each one is a function-try-block: an error message that finds no memory becomes a code."""
    import os
    import re
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tinyllm-fpga_b200", "csrc")
    heads = []
    for name in ("kv4.cu", "kv4_attn.cu", "kv4_prompt.cu"):
        with open(os.path.join(csrc, name)) as f:
            heads += re.findall(r'^extern "C" int (\w+)\([^)]*\) *(\w*)', f.read(), re.M)
    assert len(heads) >= 7 and [h for h, word in heads if word != "try"] == []


@pytest.mark.parametrize("T,hq,H", [(1 << 20, 1 << 16, 1), (1 << 15, 1 << 16, 1), (1 << 28, 1 << 16, 1 << 10)])
def test_attention_refuses_more_rows_than_it_counts(T, hq, H):
    """The kernels count a KV head's rows, tokens times query heads, in 32 bits."""
    from bfp200 import _lib, kv4
    args = kv4._ATTENTION.pack(*_batch(T=T, H=H), *[4096] * 4, 1 << 40, *[64] * 4, hq, 0, 1, 0, 0.125)
    for rc in (_lib.lib().bfp200_kv4_attention_dev(args, None), _lib.lib().bfp200_kv4_attention_workspace(args, _lib.C.c_size_t())):
        assert rc == _lib.EINVAL and "rows" in _lib.last_error()


def test_attention_workspace_checks_the_heads_as_attention_does():
    from bfp200 import _lib, kv4
    for hq in (0, 3, -2, (1 << 16) + 2, 1 << 33):
        args = kv4._ATTENTION.pack(*_batch(), *[4096] * 4, 1 << 40, *[64] * 4, hq, 0, 1, 0, 0.125)
        assert _lib.lib().bfp200_kv4_attention_dev(args, None) == _lib.EINVAL
        assert _lib.lib().bfp200_kv4_attention_workspace(args, _lib.C.c_size_t()) == _lib.EINVAL
