"""Decode over tables with ids outside the pool among good ones: the tokens of such a block count
for nothing, whatever stands in the pool's first block, and the call is flagged."""
import numpy as np
import pytest
import torch

from keptcase import BF16, BLOCK, BT, D, Cache, Layout, attend, decode_bound

pytestmark = pytest.mark.gpu


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def leave_first_block(c):
    """Moves what stands in the pool's block 0 elsewhere; NaN there instead."""
    free = next(i for i in range(1, c.nb) if not (c.table == i).any())
    for x in (c.k, c.v) + (() if c.s is None else (c.s,)):
        x[free] = x[0]
    c.table[c.table == 0] = free
    c.k[0] = c.v[0] = 0x7FC0 if c.fmt == BF16 else 0x7F
    if c.s is not None:
        c.s[0] = np.nan


@pytest.mark.parametrize("bad", [-2**31, 2**31 - 1, -1])
@pytest.mark.parametrize("kept,window,ring", [(0, 0, False), (16, 64, True), (16, 64, False)])
@pytest.mark.parametrize("max_len", [100, 20000])
def test_any_id_outside_the_pool_is_flagged(gkv, cuda, bad, kept, window, ring, max_len):
    """Of a block that is seen, by the decode and the prefill; of one that nothing sees it is not."""
    lay = Layout(kept, window, ring)
    for lose, flag in ((5, gkv.DEVERR_BLOCK_ID), (1 if window and not ring else None, 0)):
        c = Cache([96], 1, lay, BLOCK)
        if lose is not None:
            c.table[0, lay.entry(lose)] = bad
        view = c.device(gkv)
        q = torch.ones(3, D, device="cuda")
        ws = torch.zeros(max(16, gkv.kept_workspace_bytes(1, 1, max_len, kept, window)), dtype=torch.uint8, device="cuda")
        out, kv = torch.zeros(3, D, device="cuda"), torch.zeros(3, D, dtype=torch.bfloat16, device="cuda")
        gkv.kept_decode(q[:1], 1, dev(np.array([96], np.int32)), max_len, view, out[:1], kept=kept, window=window,
                        workspace=ws, dev_err=c.err)
        assert int(c.err.item()) == flag
        c.err.zero_()
        gkv.kept_prefill(dev(np.array([0, 3], np.int32)), max_len, q, 1, view, out, start_pos=dev(np.array([96], np.int32)),
                         k=kv, v=kv, kept=kept, window=window, dev_err=c.err)
        assert int(c.err.item()) == flag


@pytest.mark.parametrize("fmt", [BF16, BLOCK])
@pytest.mark.parametrize("kept,window,ring", [(0, 0, False), (16, 64, False), (32, 64, True), (0, 1600, True),
                                              (48, 1616, False)])
@pytest.mark.parametrize("max_len", [2000, 20000])  # (the second: ranges, in full layers)
@pytest.mark.parametrize("which", ["even", "odd", "first", "last", "both", "kept", "all but one"])
@pytest.mark.parametrize("bf16", [False, True])
def test_decode_masks_missing_blocks(gkv, cuda, fmt, kept, window, ring, max_len, which, bf16):
    lay = Layout(kept, window, ring)
    lens = [700, 1, 33, 1999, 160, 0, 129]
    c = Cache(lens, 2, lay, fmt, seed=kept + window)
    last = np.asarray(lens) - 1
    c.poison(last, last)
    leave_first_block(c)
    gone = [np.zeros(n, bool) for n in lens]
    for b, n in enumerate(lens):
        seen = [j for j in range(-(-n // BT)) if lay.sees(n - 1, np.arange(j * BT, min(n, j * BT + BT))).any()]
        win = [j for j in seen if j >= kept // BT] if window else seen  # the window's blocks
        lose = {"even": seen[2:8:2] + seen[-4::2], "odd": seen[1:8:2], "first": win[:1], "last": seen[-1:],
                "both": seen[4:6] + win[-2:], "kept": seen[:1], "all but one": [j for j in seen if j != seen[len(seen) // 2]]}
        for i, j in enumerate(lose[which]):
            c.table[b, lay.entry(j)] = [-1, c.nb, 2**31 - 1, -2**31 + 1][i % 4]
            gone[b][j * BT:j * BT + BT] = True
    view = c.device(gkv)
    Hq = 6
    rng = np.random.default_rng(1)
    q = rng.standard_normal((len(lens), Hq, D)).astype(np.float32)
    sinks = rng.standard_normal(Hq).astype(np.float32) if bf16 else None
    ws = torch.full((max(16, gkv.kept_workspace_bytes(len(lens), 2, max_len, kept, window)),), 255, dtype=torch.uint8,
                    device="cuda")
    out = torch.full((len(lens), Hq * D), float("nan"), dtype=torch.bfloat16 if bf16 else torch.float32, device="cuda")
    gkv.kept_decode(dev(q.reshape(len(lens), -1)), Hq, dev(np.asarray(lens, np.int32)), max_len, view, out,
                    sinks=None if sinks is None else dev(sinks), kept=kept, window=window, workspace=ws, dev_err=c.err)
    assert int(c.err.item()) == gkv.DEVERR_BLOCK_ID
    got = out.float().cpu().numpy().reshape(len(lens), Hq, D).astype(np.float64)
    for b, n in enumerate(lens):
        k, v = (np.nan_to_num(x) for x in c.kv[b])
        ok = (lay.sees(n - 1, np.arange(n)) & ~gone[b])[None]
        want, pav, qk = attend(q[b:b + 1].astype(np.float64), k, v, ok, sinks)
        bound = decode_bound(want, pav, qk, fmt, bf16)[0]
        err = np.abs(got[b] - want[0])
        assert (err <= bound).all(), (b, n, float((err / bound).max()))
