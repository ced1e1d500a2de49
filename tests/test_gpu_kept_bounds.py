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


def test_prefill_under_a_bound_of_more_workgroups_than_a_grid_row(gkv, cuda):
    """300 prompts of a few rows, the bound 131072 rows: ten million workgroups, nearly all empty."""
    B, Hkv = 300, 8
    rng = np.random.default_rng(3)
    rows = rng.integers(0, 4, B)
    n = int(rows.sum())
    g = torch.Generator(device="cuda").manual_seed(3)
    q = torch.randn(n, 8 * Hkv * D, generator=g, device="cuda")
    k, v = (torch.randn(n, Hkv * D, generator=g, device="cuda").bfloat16() for _ in "kv")
    cu = dev(np.concatenate([[0], np.cumsum(rows)]).astype(np.int32))
    outs = []
    for m in (4, 131072):
        out, err = torch.zeros(n, 8 * Hkv * D, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
        gkv.kept_prefill(cu, m, q, 8 * Hkv, gkv.CacheView(n_kv_heads=Hkv), out, k=k, v=v, dev_err=err)
        assert int(err.item()) == 0
        outs.append(out)
    assert torch.equal(*outs) and outs[0].abs().sum(1).min() > 0


@pytest.mark.parametrize("views,pairs", [(32, 600001), (3, 9000000)])
def test_copies_of_more_blocks_than_a_launch_takes(gkv, cuda, views, pairs):
    """Ids outside the cache but for the first, the middle and the last pair."""
    nb = 8
    g = torch.Generator(device="cuda").manual_seed(4)
    caches = [[torch.randint(0, 256, (nb, m), dtype=torch.uint8, device="cuda", generator=g) for m in (1024, 1024, 8)]
              for _ in range(views)]
    src = torch.full((pairs,), -1, dtype=torch.int32, device="cuda")
    dst = torch.zeros(pairs, dtype=torch.int32, device="cuda")
    for i, (s, d) in zip((0, pairs // 2, pairs - 1), ((1, 2), (3, 4), (7, 6))):
        src[i], dst[i] = s, d
    want = [[x.clone() for x in c] for c in caches]
    for c in want:
        for x in c:
            x[[2, 4, 6]] = x[[1, 3, 7]]
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    arr = gkv.cache_views([gkv.CacheView(c[0].data_ptr(), c[1].data_ptr(), None, 0, nb, 1, 0, c[2].data_ptr(),
                                         gkv.KV_FP8_BLOCK) for c in caches])
    gkv.copy_blocks(arr, src, dst, dev_err=err)
    assert int(err.item()) == gkv.DEVERR_BLOCK_ID
    assert all(torch.equal(x, y) for c, w in zip(caches, want) for x, y in zip(c, w))
