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
