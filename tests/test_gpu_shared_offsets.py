"""Group offsets of the shared decode that are none: flagged, whichever of them it is, and nothing outside the batch
is touched; offsets that are right are not flagged."""
import numpy as np
import pytest
import torch

from keptcase import BF16, BLOCK
from sharedcase import Shared, dev

pytestmark = pytest.mark.gpu


def flags(gkv, B, cu, fmt=BF16):
    """Error bits of a call over B equal sequences whose groups share two blocks."""
    s = Shared(np.full(B, 50), [B], [2], 1, fmt)
    s.c.table[:] = s.c.table[:1]
    cu = np.asarray(cu, np.int32)
    n = len(cu) - 1
    view = s.c.device(gkv)
    q, out = torch.randn(B, 8 * 64, device="cuda"), torch.full((B + 2, 8 * 64), 7.0, device="cuda")
    need = gkv.shared_workspace_bytes(B, n, 8, 1, 2, 32)
    ws = torch.zeros(need + 4096, dtype=torch.uint8, device="cuda")
    ws[need:] = 0x55
    gkv.shared_decode(q, 8, dev(cu), dev(np.full(n, 2, np.int32)), dev(s.c.lens), 50, view, out[1:B + 1], 2, 32,
                      workspace=ws[:need], dev_err=s.c.err)
    torch.cuda.synchronize()
    assert (out[0] == 7).all() and (out[B + 1] == 7).all() and (ws[need:] == 0x55).all()
    return int(s.c.err.item())


@pytest.mark.parametrize("fmt", [BF16, BLOCK])
@pytest.mark.parametrize("cu", [[0, 3, 1, 3], [3, 0], [0, 4], [0, 1, 2, 9], [-1, 3], [-2**31, 0, 3], [0, 2**31 - 1],
                                [2**31 - 1, -2**31], [0, -1, 3], [1, 3, 2], [0, 0, 3, 2]])
def test_offsets_that_are_none(gkv, cuda, fmt, cu):
    assert flags(gkv, 3, cu, fmt) & 2


@pytest.mark.parametrize("fmt", [BF16, BLOCK])
@pytest.mark.parametrize("cu", [[0, 3], [1, 2], [0, 0, 0, 3], [3, 3, 3], [0, 1, 2, 3], [0, 3, 3]])
def test_offsets_that_are_right(gkv, cuda, fmt, cu):
    assert flags(gkv, 3, cu, fmt) == 0


@pytest.mark.parametrize("B,n", [(1, 500), (2, 129), (70, 1000), (300, 300)])
def test_one_of_many(gkv, cuda, B, n):
    good = np.minimum(np.arange(n + 1), B)
    assert flags(gkv, B, good) == 0
    for i in (0, 1, n // 2, n - 1, n):
        bad = good.copy()
        bad[i] = -1 if i else B + 1
        assert flags(gkv, B, bad) & 2, i
