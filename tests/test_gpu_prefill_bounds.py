"""A prefill under a host bound far above the prompts' lengths: a grid of more threads than a launch
counts along one axis."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_prefill_under_a_bound_of_more_workgroups_than_a_grid_row(gkv, cuda):
    """300 prompts of a few rows, the bound 131072 rows: ten million workgroups, nearly all empty."""
    B, Hkv, D = 300, 8, 64
    rows = np.random.default_rng(3).integers(0, 4, B)
    n = int(rows.sum())
    g = torch.Generator(device="cuda").manual_seed(3)
    q = torch.randn(n, 8 * Hkv * D, generator=g, device="cuda")
    k, v = (torch.randn(n, Hkv * D, generator=g, device="cuda").bfloat16() for _ in "kv")
    cu = torch.from_numpy(np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)).cuda()
    sinks = torch.zeros(8 * Hkv, device="cuda")
    outs = []
    for m in (4, 131072):
        out = torch.zeros(n, 8 * Hkv * D, device="cuda")
        gkv.prefill_attention(cu, m, q, k, v, sinks, out, Hkv, window=128)
        outs.append(out)
    assert torch.equal(*outs) and outs[0].abs().sum(1).min() > 0
