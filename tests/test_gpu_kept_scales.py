"""Block scales that are NaN: what sees the block gives NaN (the prefill flags it), nothing else does.
Scales at the end of the prefill's range for V, 2^26."""
import numpy as np
import pytest
import torch

from keptcase import BLOCK, D, Cache, Layout

pytestmark = pytest.mark.gpu


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


NANS = [np.float32(np.nan), -np.float32(np.nan)]


@pytest.mark.parametrize("which", [0, 1])  # K's scale, V's
@pytest.mark.parametrize("nan", NANS)
@pytest.mark.parametrize("block", [0, 5, 18])
@pytest.mark.parametrize("kept,window", [(0, 0), (16, 240)])
@pytest.mark.parametrize("max_len", [300, 20000])
def test_decode_keeps_a_scale_that_is_nan(gkv, cuda, which, nan, block, kept, window, max_len):
    lay = Layout(kept, window, False)
    c = Cache([300, 300, 300], 2, lay, BLOCK)
    c.s[c.table[1, block], 1, which] = nan
    view = c.device(gkv)
    q = torch.randn(3, 4 * D, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    ws = torch.zeros(max(16, gkv.kept_workspace_bytes(3, 2, max_len, kept, window)), dtype=torch.uint8, device="cuda")
    out = torch.zeros(3, 4, D, device="cuda")
    gkv.kept_decode(q, 4, dev(np.array([300] * 3, np.int32)), max_len, view, out.view(3, -1), kept=kept, window=window,
                    workspace=ws, dev_err=c.err)
    bad = torch.zeros(3, 4, dtype=torch.bool)
    bad[1, 2:] = bool(lay.sees(299, np.arange(16 * block, min(300, 16 * block + 16))).any())
    assert torch.equal(torch.isnan(out).all(-1).cpu(), bad) and torch.equal(torch.isnan(out).any(-1).cpu(), bad)


@pytest.mark.parametrize("nan", NANS + [np.float32(np.inf)])
@pytest.mark.parametrize("block", [0, 5, 18])
@pytest.mark.parametrize("kept,window", [(0, 0), (16, 240)])
@pytest.mark.parametrize("max_len", [60, 20000])
def test_prefill_keeps_and_flags_a_k_scale_that_is_not_finite(gkv, cuda, nan, block, kept, window, max_len):
    lay = Layout(kept, window, False)
    c = Cache([304, 304], 2, lay, BLOCK)
    c.s[c.table[1, block], 1, 0] = nan
    view = c.device(gkv)
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn(120, 4 * D, generator=g, device="cuda")
    k, v = (torch.randn(120, 2 * D, generator=g, device="cuda").bfloat16() for _ in "kv")
    out = torch.zeros(120, 4, D, device="cuda")
    gkv.kept_prefill(dev(np.array([0, 60, 120], np.int32)), max_len, q, 4, view, out.view(120, -1),
                     start_pos=dev(np.array([304, 304], np.int32)), k=k, v=v, kept=kept, window=window, dev_err=c.err)
    bad = torch.zeros(120, 4, dtype=torch.bool)
    for i in range(60):
        bad[60 + i, 2:] = bool(lay.sees(304 + i, np.arange(16 * block, 16 * block + 16)).any())
    assert torch.equal(torch.isnan(out).all(-1).cpu(), bad) and torch.equal(torch.isnan(out).any(-1).cpu(), bad)
    assert int(c.err.item()) == (gkv.DEVERR_RANGE if bad.any() else 0)


@pytest.mark.parametrize("scale,flag", [(2.0 ** 17, False), (149000.0, False), (2.0 ** 18, True), (150000.0, True),
                                        (2.0 ** 60, True), (3e30, True)])
@pytest.mark.parametrize("max_len", [4, 20000])
def test_prefill_flags_block_scales_beyond_its_range(gkv, cuda, scale, flag, max_len):
    """V of 448 scale and of 1 scale, all weights equal: exact within fp16's rounding of v 2^-10 up to 2^26
    (65520, halfway to 2^16, is the first that rounds past the largest), an infinity beyond."""
    c = Cache([16], 1, Layout(0, 0, False), BLOCK)
    blk = c.table[0, 0]
    c.k[blk], c.s[blk, 0] = 0, (1, scale)
    c.v[blk] = 0x38                                        # 1.0
    c.v[blk, 0, :64] = 0x7E                                # 448: 16 tokens of dims 0, 16, 32, 48
    view = c.device(gkv)
    q, kv = torch.ones(2, D, device="cuda"), torch.zeros(2, D, dtype=torch.bfloat16, device="cuda")
    out = torch.zeros(2, D, device="cuda")
    gkv.kept_prefill(dev(np.array([0, 2], np.int32)), max_len, q, 1, view, out, start_pos=dev(np.array([16], np.int32)),
                     k=kv, v=kv, dev_err=c.err)
    assert int(c.err.item()) == (gkv.DEVERR_RANGE if flag else 0)
    if not flag:
        want = np.full(D, scale)
        want[::16] *= 448
        for i in range(2):
            assert (np.abs(out[i].cpu().numpy() - want * 16 / (17 + i)) <= want * (2.0 ** -11 + 2.0 ** -10)).all()
    else:
        assert torch.isinf(out[:, ::16]).all()
