"""Calls whose host bounds are smaller than the lengths, or far larger."""
import numpy as np
import pytest
import torch

from keptcase import D

pytestmark = pytest.mark.gpu


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


@pytest.mark.parametrize("Hq,Hkv", [(8, 1), (4, 2), (3, 3)])
@pytest.mark.parametrize("rows,bound", [([40, 3], 39), ([1, 600], 500), ([2, 0, 2], 1), ([64, 65], 64), ([300, 301], 300)])
def test_prefill_flags_prompts_longer_than_the_bound(gkv, cuda, Hq, Hkv, rows, bound):
    """... and gives the rows within the bound as ever."""
    n = sum(rows)
    g = torch.Generator(device="cuda").manual_seed(2)
    q = torch.randn(n, Hq * D, generator=g, device="cuda")
    k, v = (torch.randn(n, Hkv * D, generator=g, device="cuda").bfloat16() for _ in "kv")
    cu = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    view, outs = gkv.CacheView(n_kv_heads=Hkv), []
    for m, want in ((max(rows), 0), (bound, gkv.DEVERR_LENGTH)):
        out, err = torch.zeros(n, Hq * D, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
        gkv.kept_prefill(dev(cu), m, q, Hq, view, out, k=k, v=v, dev_err=err)
        assert int(err.item()) == want
        gkv.kept_prefill(dev(cu), m, q, Hq, view, out, k=k, v=v)  # (without a place for flags)
        outs.append(out)
    # (one group of waves and two round the weights against other references: 2^-11 of each
    # and of their sum, on both sides; 2^-16 for the fp32 sums)
    tol = float(v.float().abs().max()) * (2.0 ** -9 + 2.0 ** -16)
    for b, m in enumerate(rows):
        r = slice(cu[b], cu[b] + min(m, bound))
        assert torch.allclose(outs[0][r], outs[1][r], rtol=0, atol=tol)
