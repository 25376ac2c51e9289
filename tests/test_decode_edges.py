"""Edges of the decoding operators and of the decoder's bookkeeping, against the same numpy restatement in 64 bits. Every result is an
integer, so every comparison is exact."""
import numpy as np
import pytest

import test_decode_ops as ops

gpu = pytest.mark.gpu


# ------------------------------------------------------------------------------------- tables that do not rise

def _falling(seed, top):
    """A table of large entries whose last one, that of a row's largest score, is `top`: what stands at a score that no key of the row has
    is as much as 2^30 times the sum."""
    lut = np.random.default_rng(seed).integers(1 << 20, 1 << 30, 256)
    lut[255] = top
    return lut


@gpu
@pytest.mark.parametrize("one", [127, 910, 911, 32767])
@pytest.mark.parametrize("heads_q", [1, 4, 5, 8, 9, 16])
@pytest.mark.parametrize("seed", range(4))
def test_attention_tables_whose_unseen_entries_are_large(monkeypatch, seed, heads_q, one):
    """One visible key and a few, with every form of the tiles (up to 4, 8 and 16 rows, narrow and wide digits)."""
    monkeypatch.setitem(ops.LUTS, "falling", _falling(seed, 1 + seed))
    ops.attention_case([1, 1, 1, 1], [1] * 4, heads_q, 1, 32, seed=seed, lut="falling", one=one)
    ops.attention_case([3, 70, 2], [1] * 3, heads_q, 1, 64, seed=seed, lut="falling", one=one)
    ops.attention_case([64, 1], [1] * 2, heads_q, 1, 128, seed=seed, lut="falling", one=one, window=1)
    ops.attention_case([2400], [1], heads_q, 1, 32, seed=seed, lut="falling", one=one, window=2300)


@gpu
@pytest.mark.parametrize("one", [1, 127, 128, 32639, 32640])
@pytest.mark.parametrize("window", [0, 1, 2100])
def test_attention_of_many_rows_with_tables_whose_unseen_entries_are_large(monkeypatch, window, one):
    monkeypatch.setitem(ops.LUTS, "falling", _falling(window, 3))
    for case in ops.MANY:
        ops.attention_case(*case, 32, seed=one, lut="falling", one=one, window=window)
