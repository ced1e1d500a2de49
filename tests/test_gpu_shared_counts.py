"""Counts of shared blocks over resizes: a reorder in which every row is its own parent counts again."""
import numpy as np
import pytest

from test_gpu_tables import Tables

pytestmark = pytest.mark.gpu


def counts(t, per):
    t.check_reorder(np.arange(t.n), per)  # (against the model)
    return t.m.reorder(np.arange(t.n), per)[0].tolist()


@pytest.mark.parametrize("stride", [8, 3000])
def test_a_row_that_was_cut_into_the_shared_blocks(gkv, cuda, stride):
    t = Tables(gkv, 8, stride, 200)
    assert t.check_resize([80, 0, 0, 0, 60, 0, 0, 0])
    t.check_reorder([0, 0, 0, 0, 4, 4, 4, 4], 4)
    assert counts(t, 4) == [5, 3]
    assert t.check_resize([80, 80, 20, 90, 61, 62, 63, 64])
    assert counts(t, 4) == [1, 3]
    assert t.check_resize([80, 80, 80, 90, 61, 62, 63, 64])
    assert counts(t, 4) == [1, 3]  # (as long as before, in other blocks)


def test_an_empty_row_shares_nothing(gkv, cuda):
    t = Tables(gkv, 4, 8, 64)
    assert t.check_resize([80, 0, 0, 0])
    t.check_reorder([0, 0, -1, 0], 4)
    assert counts(t, 4) == [0]
    t.check_reorder([0, 1, 0, 3], 4)
    assert counts(t, 4) == [5]
