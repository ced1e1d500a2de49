"""The workspace of the shared decode: what is enough for a batch is enough for every smaller one, however it is
grouped."""
import numpy as np
import pytest
import torch

from keptcase import BF16, BLOCK
from sharedcase import Shared, dev, shared_bound, within


@pytest.mark.parametrize("Hq,Hkv", [(64, 8), (8, 1), (6, 3), (7, 7)])
@pytest.mark.parametrize("shared,own", [(0, 0), (1, 1), (128, 1000), (4000, 100), (5, 100000), (4000, 100000)])
def test_room_for_all_is_room_for_fewer(gkv, Hq, Hkv, shared, own):
    need = lambda B, n: gkv.shared_workspace_bytes(B, n, Hq, Hkv, shared, own)  # noqa: E731
    sizes = [1, 2, 3, 5, 9, 16, 31, 64, 100, 256, 257, 300, 511, 512, 513, 1000, 2047, 2048, 2049, 5000, 8192]
    most = 0
    for B in sizes:
        grouped = [need(B, n) for n in sorted({0, 1, 2, B // 8, B // 2, B, 2 * B})]
        assert min(grouped) >= most, B
        most = max(grouped)


def test_bounds_that_grow(gkv):
    for B in (1, 7, 300):
        for low, high in (((3, 10), (3, 5000)), ((3, 10), (900, 10)), ((0, 0), (1, 1))):
            assert gkv.shared_workspace_bytes(B, 2, 64, 8, *low) <= gkv.shared_workspace_bytes(B, 2, 64, 8, *high)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,bf16", [(BF16, True), (BF16, False), (BLOCK, True), (BLOCK, False)])
@pytest.mark.parametrize("most,now", [((300, 1), [256]), ((300, 1), [4]), ((300, 300), [300]), ((64, 1), [8, 8, 8, 8]),
                                      ((24, 1), [1])])
def test_a_smaller_batch_in_a_larger_ones_workspace(gkv, cuda, fmt, bf16, most, now):
    rng = np.random.default_rng(sum(now))
    blocks, Hq, Hkv = 128, 8, 1
    s = Shared(blocks * 16 + rng.integers(1, 40, sum(now)), now, [blocks] * len(now), Hkv, fmt)
    n = gkv.shared_workspace_bytes(most[0], most[1], Hq, Hkv, blocks, 40)
    ws = torch.full((n + 4096,), 0xFF, dtype=torch.uint8, device="cuda")
    q = rng.standard_normal((s.B, Hq, 64)).astype(np.float32)
    out = torch.zeros(s.B, Hq * 64, dtype=torch.bfloat16 if bf16 else torch.float32, device="cuda")
    view = s.c.device(gkv)
    gkv.shared_decode(dev(q.reshape(s.B, -1)), Hq, dev(s.cu), dev(s.shared), dev(s.c.lens), int(s.c.lens.max()), view, out,
                      blocks, 40, workspace=ws[:n], dev_err=s.c.err)
    want, pav, qk, qm = s.expect(q, None)
    within(out.float().cpu().numpy().reshape(want.shape), want, shared_bound(want, pav, qk, qm, fmt, bf16))
    assert int(s.c.err.item()) == 0 and (ws[n:] == 0xFF).all()
