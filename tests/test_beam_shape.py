"""Slices of a beam selection, by the workspace that it asks for (host only)."""
import ctypes

import pytest

from ft_b200 import lib

MERGE_BYTES = 176 << 10      # of shared memory for the listed logits of a request, 4 each


def slices(batch, beams, vocab, best, dtype):
    a = lib.BeamSelectArgs()
    a.dtype, a.batch, a.beams, a.vocab, a.best = dtype, batch, beams, vocab, best
    size = lib.load().ft_beam_select_workspace(ctypes.byref(a))
    assert size > 0 and size % (batch * beams * 8 * (best + 1)) == 0
    return size // (batch * beams * 8 * (best + 1))


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("batch", [1, 2, 3, 7])
def test_every_call_has_slices_that_its_merge_holds(batch, dtype):
    for beams in range(1, 65):
        for step in range(160):
            vocab = int(1.147 ** step) + step * (beams % 7)
            assert 4 * beams * slices(batch, beams, min(vocab, 1 << 30), 64, dtype) * 64 <= MERGE_BYTES, (beams, vocab)


def test_a_call_of_many_uneven_slices():
    assert 4 * 59 * slices(1, 59, 353898340, 64, 2) * 64 <= MERGE_BYTES
