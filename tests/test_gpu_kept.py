"""gkv_kept_append, gkv_kept_decode, gkv_kept_prefill and gkv_copy_blocks on the GPU, against
their definitions in 64 bits (tolerances derived in keptcase.py); appends and copies bit for
bit."""
import numpy as np
import pytest
import torch

from keptcase import (BF16, BLOCK, BT, D, PLACES, Cache, Layout, attend, block_scale, decode_bound,
                      e4m3, e4m3_values, prefill_bound)
from oracle import kv_oracle as O

pytestmark = pytest.mark.gpu


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def rotated(qkv, Hq, Hkv, cos, sin, pos):
    """The oracle's rotated query and key rows (fp32) and the bf16 K and V."""
    q, k, kb, vb = O.kv_append(np.ascontiguousarray(qkv), Hq, Hkv, cos, sin, np.asarray(pos, np.int32))
    n = qkv.shape[0]
    return q.reshape(n, Hq, D), np.asarray(k).reshape(n, Hkv, D), kb.reshape(n, Hkv, D), vb.reshape(n, Hkv, D)


def same(name, x, y):
    if x is not None:
        bad = np.argwhere(x.view(np.uint8) != y.view(np.uint8))
        assert len(bad) == 0, f"{name}: {len(bad)} bytes differ, first at {bad[:3].tolist()}"


# ---- append ---------------------------------------------------------------------


def expect_append(c, n_rows, krot, v, fmt):
    """The pool after the append of n_rows[b] rows behind c.lens[b] tokens."""
    k, vv = c.k.copy(), c.v.copy()
    s = None if c.s is None else c.s.copy()
    row = 0
    for b in range(c.B):
        lo, L = int(c.lens[b]), int(c.lens[b]) + n_rows[b]
        for j in range(lo // BT, -(-L // BT)):
            later = range(j + 1, -(-L // BT))
            if c.lay.ring and c.lay.entry(j) in [c.lay.entry(i) for i in later]:
                continue
            phys = c.table[b, c.lay.entry(j)]
            t0, t1 = max(lo, j * BT), min(L, j * BT + BT)
            if t0 >= t1:
                continue
            old = t0 - j * BT
            for i, (pool, x) in enumerate(((k, krot), (vv, v))):
                x = x[row + t0 - lo:row + t1 - lo].transpose(1, 0, 2)   # [Hkv, n, 64]
                blk = pool[phys][:, PLACES[fmt][i]]                     # [Hkv, 16, 64]
                if not old:
                    blk[:] = 0
                if fmt == BF16:
                    blk[:, old:old + t1 - t0] = O.to_bf16(np.ascontiguousarray(x))
                else:
                    fin = np.where(np.isfinite(x), np.abs(x), 0)
                    sn = block_scale(fin.max((1, 2)))
                    if old:
                        sn = np.maximum(sn, s[phys, :, i])
                        r = np.where(sn > 0, s[phys, :, i] / np.where(sn > 0, sn, 1), 0)
                        blk[:, :old] = np.where((sn != s[phys, :, i])[:, None, None],
                                                e4m3(e4m3_values(blk[:, :old]) * r[:, None, None].astype(np.float32)),
                                                blk[:, :old])
                    with np.errstate(all="ignore"):
                        y = x * (1 / np.where(sn > 0, sn, 1))[:, None, None].astype(np.float32)
                    blk[:, old:old + t1 - t0] = e4m3(np.clip(y, -448, 448))
                    s[phys, :, i] = sn
                pool[phys][:, PLACES[fmt][i]] = blk
        row += n_rows[b]
    return k, vv, s


def run_append(gkv, lens, n_rows, Hq, Hkv, lay, fmt, seed=0, pack=False, tweak=None, stride_pad=0):
    c = Cache(lens, Hkv, lay, fmt, seed=seed)
    rng = np.random.default_rng(seed + 1)
    n = int(sum(n_rows))
    qkv = (rng.standard_normal((n, (Hq + 2 * Hkv) * D)) * 2.0 ** rng.integers(-3, 6, (n, 1))).astype(np.float32)
    if tweak:
        tweak(qkv)
    pos = np.concatenate([np.arange(a, a + m) for a, m in zip(lens, n_rows)] + [np.zeros(0, int)])
    cos, sin = O.rope_table(int(max(a + m for a, m in zip(lens, n_rows))) + 1)
    _, krot, kb, vb = rotated(qkv, Hq, Hkv, cos, sin, pos)
    view = c.device(gkv)
    kp = vp = None
    if pack:
        kp, vp = (torch.zeros(n, Hkv, D, dtype=torch.int16, device="cuda") for _ in "kv")
    x = torch.zeros(n, qkv.shape[1] + stride_pad, device="cuda")
    x[:, :qkv.shape[1]] = dev(qkv)
    one = all(m == 1 for m in n_rows)
    cu = None if one else dev(np.concatenate([[0], np.cumsum(n_rows)]).astype(np.int32))
    gkv.kept_append(x, Hq, dev(cos), dev(sin), dev((np.asarray(lens) + n_rows).astype(np.int32)), view,
                    kept=lay.kept, window=lay.window, cu_seqlens=cu, max_rows=max(n_rows), k_pack=kp,
                    v_pack=vp, dev_err=c.err)
    v = qkv[:, (Hq + Hkv) * D:].reshape(n, Hkv, D)
    got, want = c.pulled(), expect_append(c, n_rows, krot, v, fmt)
    assert int(c.err.item()) == 0
    for name, x, y in zip("kvs", got, want):
        if fmt == BLOCK and name != "s":  # (a NaN has two codes)
            x, y = (np.where(z & 0x7f == 0x7f, np.uint8(0x7f), z) for z in (x, y))
        same(name, x, y)
    if pack:
        assert np.array_equal(kp.cpu().numpy().view(np.uint16), kb)
        assert np.array_equal(vp.cpu().numpy().view(np.uint16), vb)


@pytest.mark.parametrize("fmt", [BF16, BLOCK])
@pytest.mark.parametrize("kept,window,ring", [(0, 0, False), (16, 32, True), (0, 16, True), (48, 64, False)])
@pytest.mark.parametrize("lens,rows", [([0], [1]), ([5, 15, 16, 0, 33], [1, 1, 1, 1, 1]),
                                       ([0, 0, 7, 16, 40], [1, 17, 30, 200, 16])])
def test_append_is_exact(gkv, cuda, fmt, kept, window, ring, lens, rows):
    run_append(gkv, lens, rows, 8, 2, Layout(kept, window, ring), fmt, seed=len(rows) + kept)


@pytest.mark.parametrize("fmt", [BF16, BLOCK])
@pytest.mark.parametrize("Hq,Hkv", [(64, 8), (6, 3), (7, 7), (11, 11), (8, 1)])
def test_append_head_counts_and_packed_rows(gkv, cuda, fmt, Hq, Hkv):
    run_append(gkv, [0, 3, 50], [40, 1, 19], Hq, Hkv, Layout(0, 0, False), fmt, seed=Hq, pack=True,
               stride_pad=4)


def test_append_values_at_the_borders(gkv, cuda):
    """All zeros, the scale's borders, tiny values, infinities and NaN (K rows at position 0,
    where the rotation leaves them as they are but for x * 0)."""
    def tweak(q):
        q[0] = 0
        q[1, :] = 448.0
        q[2, :] = np.nextafter(np.float32(448), np.float32(500))
        q[3, :] = 1e-42
        q[4, -64:] = np.inf
        q[5, -64:] = np.nan
        q[6, -3] = -np.inf
        q[7, :] = 3e38
    run_append(gkv, [0] * 8, [1] * 8, 2, 1, Layout(0, 0, False), BLOCK, tweak=tweak)


def test_append_one_by_one_is_the_block_at_once_but_for_the_older_codes(gkv, cuda):
    """16 tokens of growing size: the scale grows with them, and each code is at most one
    more rounding (half a step of e4m3, or of its subnormals) off."""
    rng = np.random.default_rng(3)
    qkv = (rng.standard_normal((16, 4 * D)) * 2.0 ** np.arange(16)[:, None] / 64).astype(np.float32)
    cos, sin = O.rope_table(16)
    _, krot, _, _ = rotated(qkv, 2, 1, cos, sin, np.arange(16))
    c = Cache([0], 1, Layout(0, 0, False), BLOCK)
    view = c.device(gkv)
    for t in range(16):
        gkv.kept_append(dev(qkv[t:t + 1]), 2, dev(cos), dev(sin), dev(np.array([t + 1], np.int32)),
                        view, dev_err=c.err)
    k, v, s = c.pulled()
    blk = c.table[0, 0]
    for i, (pool, x) in enumerate(((k, krot), (v, qkv[:, 3 * D:].reshape(16, 1, D)))):
        sc = s[blk, 0, i]
        assert sc == block_scale(np.abs(x).max())
        got = e4m3_values(pool[blk, 0][PLACES[BLOCK][i]]).astype(np.float64) * sc
        err = np.abs(got - x[:, 0])
        # half a step each time: of the value (2^-4 of it), or of the subnormals (2^-10 of s)
        assert (err <= np.maximum(np.abs(x[:, 0]) * 2.0 ** -4, 2.0 ** -10 * sc) * 2).all()


def test_append_bad_pages_and_idle_rows(gkv, cuda):
    """Ids outside the pool and rows past the table are flagged and not stored; a length of 0
    is an idle place; more rows than max_rows are flagged."""
    lay = Layout(0, 0, False)
    c = Cache([20, 20, 0], 2, lay, BLOCK)
    c.table[0, 1] = c.nb
    view = c.device(gkv)
    cos, sin = O.rope_table(64)
    rng = np.random.default_rng(0)
    qkv = dev(rng.standard_normal((3, 8 * D)).astype(np.float32))
    before = c.pulled()
    gkv.kept_append(qkv, 4, dev(cos), dev(sin), dev(np.array([21, 0, 0], np.int32)), view, dev_err=c.err)
    assert int(c.err.item()) == gkv.DEVERR_BLOCK_ID
    for name, x, y in zip("kvs", before, c.pulled()):
        same(name, x, y)
    c.err.zero_()
    cap = c.table.shape[1] * BT
    cos, sin = O.rope_table(cap)
    gkv.kept_append(qkv, 4, dev(cos), dev(sin), dev(np.array([cap + 1, 0, 0], np.int32)), view,
                    dev_err=c.err)
    assert int(c.err.item()) == gkv.DEVERR_LENGTH
    for name, x, y in zip("kvs", before, c.pulled()):
        same(name, x, y)
    c.err.zero_()
    gkv.kept_append(qkv, 4, dev(cos), dev(sin), dev(np.array([0, 3, 0], np.int32)), view, max_rows=2,
                    cu_seqlens=dev(np.array([0, 0, 3, 3], np.int32)), dev_err=c.err)
    assert int(c.err.item()) == gkv.DEVERR_LENGTH


# ---- decode ---------------------------------------------------------------------


def run_decode(gkv, lens, Hq, Hkv, lay, fmt, sinks=True, bf16=False, seed=0, rope=True, max_len=None,
               spread=False, view_of=None, ws_pad=0):
    c = Cache(lens, Hkv, lay, fmt, seed=seed, spread=spread)
    last = np.asarray(lens) - 1
    c.poison(last, last)
    rng = np.random.default_rng(seed + 2)
    B = len(lens)
    width = (Hq + 2 * Hkv) * D
    qkv = rng.standard_normal((B, width)).astype(np.float32)
    sk = rng.standard_normal(Hq).astype(np.float32) if sinks else None
    max_len = max_len or max(max(lens), 1)
    cos, sin = O.rope_table(max_len)
    q = qkv[:, :Hq * D].reshape(B, Hq, D)
    if rope:
        q = rotated(qkv, Hq, Hkv, cos, sin, np.maximum(last, 0))[0]
    view = c.device(gkv)
    ws_n = gkv.kept_workspace_bytes(B, Hkv, max_len, lay.kept, lay.window)
    ws = torch.full((ws_n,), 255, dtype=torch.uint8, device="cuda") if ws_n else None
    out = torch.full((B, Hq * D + 8), float("nan"), dtype=torch.bfloat16 if bf16 else torch.float32, device="cuda")
    gkv.kept_decode(dev(qkv), Hq, dev(np.asarray(lens, np.int32)), max_len, view, out,
                    sinks=None if sk is None else dev(sk), kept=lay.kept, window=lay.window,
                    cos_tab=dev(cos) if rope else None, sin_tab=dev(sin) if rope else None, workspace=ws,
                    dev_err=c.err)
    assert int(c.err.item()) == 0
    got = out.float().cpu().numpy()
    assert np.isnan(got[:, Hq * D:]).all()
    got = got[:, :Hq * D].reshape(B, Hq, D).astype(np.float64)
    for b in range(B):
        k, v = c.kv[b]
        ok = lay.sees(lens[b] - 1, np.arange(lens[b]))[None]
        want, pav, qk = attend(q[b:b + 1].astype(np.float64), k, v, ok, sk)
        if lens[b] == 0:
            assert (got[b] == 0).all()
            continue
        bound = decode_bound(want, pav, qk, fmt, bf16)[0]
        err = np.abs(got[b] - want[0])
        assert (err <= bound).all(), (b, lens[b], float((err / bound).max()))


LENS = [[1], [0, 1, 15, 16, 17], [33, 250, 0, 64, 31, 129], [700, 3]]


@pytest.mark.parametrize("fmt", [BF16, BLOCK])
@pytest.mark.parametrize("kept,window,ring", [(0, 0, False), (16, 32, True), (0, 16, True),
                                              (48, 64, False), (32, 128, True)])
@pytest.mark.parametrize("lens", LENS)
def test_decode(gkv, cuda, fmt, kept, window, ring, lens):
    run_decode(gkv, lens, 16, 2, Layout(kept, window, ring), fmt, seed=kept + len(lens),
               sinks=len(lens) % 2 == 0, bf16=len(lens) == 5, spread=len(lens) == 6)


@pytest.mark.parametrize("fmt", [BF16, BLOCK])
@pytest.mark.parametrize("Hq,Hkv", [(64, 8), (6, 3), (7, 7), (40, 8), (8, 1), (5, 5), (24, 4)])
@pytest.mark.parametrize("kept,window,ring", [(0, 0, False), (16, 48, True)])
def test_decode_head_counts(gkv, cuda, fmt, Hq, Hkv, kept, window, ring):
    run_decode(gkv, [40, 0, 900, 17], Hq, Hkv, Layout(kept, window, ring), fmt, seed=Hq, sinks=Hq % 2 == 0)


@pytest.mark.parametrize("fmt", [BF16, BLOCK])
def test_decode_many_short_sequences_through_the_ranges(gkv, cuda, fmt):
    """Far more sequences than ranges' steps, many of them empty, and one long."""
    rng = np.random.default_rng(5)
    lens = list(rng.integers(0, 40, 300)) + [600]
    run_decode(gkv, [int(x) for x in lens], 2, 1, Layout(0, 0, False), fmt, max_len=20000)


@pytest.mark.parametrize("fmt", [BF16, BLOCK])
def test_decode_one_long_sequence_in_many_pieces(gkv, cuda, fmt):
    run_decode(gkv, [9001], 4, 1, Layout(0, 0, False), fmt, sinks=False)


def test_decode_wide_window_and_query_already_rotated(gkv, cuda):
    run_decode(gkv, [6000, 2049], 8, 1, Layout(64, 4096, True), BLOCK, rope=False)


def test_decode_extremes(gkv, cuda):
    """Sinks of -inf and far above every score, a query of zeros, large and tiny queries."""
    lay = Layout(16, 32, True)
    for fmt in (BF16, BLOCK):
        c = Cache([100, 100, 100], 1, lay, fmt, seed=4)
        c.poison([99] * 3, [99] * 3)
        rng = np.random.default_rng(1)
        qkv = rng.standard_normal((3, 6 * D)).astype(np.float32)
        qkv[0] = 0
        qkv[1] *= 1e-30
        qkv[2] *= 30
        sk = np.array([-np.inf, 60.0, -60.0, 0.0], np.float32)
        out = torch.zeros(3, 4 * D, device="cuda")
        gkv.kept_decode(dev(qkv), 4, dev(np.array([100] * 3, np.int32)), 100, c.device(gkv), out,
                        sinks=dev(sk), kept=16, window=32, dev_err=c.err)
        got = out.cpu().numpy().reshape(3, 4, D).astype(np.float64)
        for b in range(3):
            q = qkv[b, :4 * D].reshape(1, 4, D).astype(np.float64)
            want, pav, qk = attend(q, *c.kv[b], lay.sees(99, np.arange(100))[None], sk)
            bound = decode_bound(want, pav, qk, fmt, False) + 2.0 ** -126
            assert (np.abs(got[b] - want[0]) <= bound[0]).all()


def test_decode_bad_pages_and_long_lengths(gkv, cuda):
    """A bad block id masks its block and is flagged; all bad and no sink: zeros; a length past
    the bound is flagged."""
    for window in (0, 32):
        lay = Layout(0, window, False)
        c = Cache([64, 700], 1, lay, BLOCK, seed=2)
        c.table[0, :] = [c.nb + 9, -1] * (c.table.shape[1] // 2) + [-1] * (c.table.shape[1] % 2)
        view = c.device(gkv)
        q = dev(np.random.default_rng(0).standard_normal((2, 2 * D)).astype(np.float32))
        out = torch.full((2, 2 * D), 7.0, device="cuda")
        ws = torch.zeros(max(1, gkv.kept_workspace_bytes(2, 1, 700, 0, window)), dtype=torch.uint8, device="cuda")
        gkv.kept_decode(q, 2, dev(np.array([64, 700], np.int32)), 700, view, out, window=window,
                        workspace=ws, dev_err=c.err)
        assert int(c.err.item()) == gkv.DEVERR_BLOCK_ID
        assert (out[0] == 0).all() and torch.isfinite(out[1]).all()
        c.err.zero_()
        gkv.kept_decode(q, 2, dev(np.array([0, 701], np.int32)), 700, view, out, window=window,
                        workspace=ws, dev_err=c.err)
        assert int(c.err.item()) == gkv.DEVERR_LENGTH


# ---- prefill --------------------------------------------------------------------


def run_prefill(gkv, starts, rows, Hq, Hkv, lay, fmt, sinks=True, bf16=False, seed=0, cached=True,
                from_cache=False, spread=False, scale=1.0, max_len=None):
    c = Cache(np.asarray(starts) + (rows if from_cache else 0), Hkv, lay, fmt, seed=seed, spread=spread,
              scale=scale)
    last = np.asarray(starts) + rows - 1
    c.poison(starts, last)
    rng = np.random.default_rng(seed + 3)
    n = int(sum(rows))
    qkv = rng.standard_normal((n, (Hq + 2 * Hkv) * D)).astype(np.float32)
    pos = np.concatenate([np.arange(a, a + m) for a, m in zip(starts, rows)])
    cos, sin = O.rope_table(int(pos.max()) + 1)
    q, _, kb, vb = rotated(qkv, Hq, Hkv, cos, sin, pos)
    sk = rng.standard_normal(Hq).astype(np.float32) if sinks else None
    view = c.device(gkv)
    if not cached:
        view = gkv.CacheView(n_kv_heads=Hkv)
    out = torch.full((n, Hq * D), float("nan"), dtype=torch.bfloat16 if bf16 else torch.float32, device="cuda")
    cu = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    gkv.kept_prefill(dev(cu), max_len or max(rows), dev(qkv), Hq, view, out,
                     start_pos=dev(np.asarray(starts, np.int32)) if cached else None,
                     k=None if from_cache else dev(kb.view(np.int16)),
                     v=None if from_cache else dev(vb.view(np.int16)),
                     sinks=None if sk is None else dev(sk), kept=lay.kept, window=lay.window,
                     cos_tab=dev(cos), sin_tab=dev(sin), dev_err=c.err)
    assert int(c.err.item()) == 0
    got = out.float().cpu().numpy().reshape(n, Hq, D).astype(np.float64)
    kf, vf = O.from_bf16(kb).astype(np.float64), O.from_bf16(vb).astype(np.float64)
    for b in range(len(rows)):
        r = slice(cu[b], cu[b + 1])
        k, v = c.kv[b]
        if not from_cache:
            k, v = np.concatenate([k, kf[r]]), np.concatenate([v, vf[r]])
        t = np.arange(len(k))
        ok = np.stack([lay.sees(p, t) for p in range(starts[b], starts[b] + rows[b])])
        want, pav, qk = attend(q[r].astype(np.float64), k, v, ok, sk)
        bound = prefill_bound(want, pav, qk, len(k), np.nanmax(np.abs(v)), bf16)
        err = np.abs(got[r] - want)
        assert (err <= bound).all(), (b, float((err / bound).max()))


@pytest.mark.parametrize("kept,window", [(16, 32), (0, 16), (64, 128), (96, 16), (0, 0)])
@pytest.mark.parametrize("Hq,Hkv", [(16, 2), (3, 3), (4, 2), (3, 1)])
def test_prefill_of_prompts(gkv, cuda, kept, window, Hq, Hkv):
    run_prefill(gkv, [0, 0, 0], [1, 77, 300], Hq, Hkv, Layout(kept, window, False), BF16, cached=False,
                sinks=Hq % 2 == 0, bf16=Hq == 16)


@pytest.mark.parametrize("fmt", [BF16, BLOCK])
@pytest.mark.parametrize("kept,window,ring", [(0, 0, False), (16, 32, True), (0, 16, True), (96, 48, True),
                                              (48, 64, False), (32, 256, True)])
@pytest.mark.parametrize("Hq,Hkv", [(16, 2), (3, 3), (4, 2), (4, 1)])
def test_prefill_of_chunks(gkv, cuda, fmt, kept, window, ring, Hq, Hkv):
    run_prefill(gkv, [0, 16, 208, 336, 48], [5, 33, 70, 16, 130], Hq, Hkv, Layout(kept, window, ring), fmt,
                sinks=Hq % 2 == 0, seed=kept, bf16=Hq == 3)


@pytest.mark.parametrize("fmt", [BF16, BLOCK])
def test_prefill_with_every_key_in_the_cache(gkv, cuda, fmt):
    run_prefill(gkv, [0, 96], [40, 70], 8, 1, Layout(0, 0, False), fmt, from_cache=True)


def test_prefill_flags_bad_pages_and_starts(gkv, cuda):
    lay = Layout(0, 0, False)
    c = Cache([32], 1, lay, BLOCK)
    c.table[0, 1] = -1
    view = c.device(gkv)
    qkv = torch.zeros(8, 4 * D, device="cuda")
    kv = torch.zeros(8, D, dtype=torch.int16, device="cuda")
    out = torch.zeros(8, 2 * D, device="cuda")
    cu = dev(np.array([0, 8], np.int32))
    gkv.kept_prefill(cu, 8, qkv, 2, view, out, start_pos=dev(np.array([32], np.int32)), k=kv, v=kv, dev_err=c.err)
    assert int(c.err.item()) == gkv.DEVERR_BLOCK_ID
    c.err.zero_()
    gkv.kept_prefill(cu, 8, qkv, 2, view, out, start_pos=dev(np.array([7], np.int32)), k=kv, v=kv, dev_err=c.err)
    assert int(c.err.item()) & gkv.DEVERR_ALIGN


# ---- copies ---------------------------------------------------------------------


@pytest.mark.parametrize("fmt,Hkv", [(0, 8), (0, 1), (1, 3), (2, 5), (3, 8), (3, 1), (3, 3)])
@pytest.mark.parametrize("layers,pairs", [(1, 1), (3, 7), (35, 4), (2, 600)])
def test_copy_blocks(gkv, cuda, fmt, Hkv, layers, pairs):
    nb = 2 * pairs + 3
    sizes = {0: (2048, 2048, 0), 1: (2048, 1024, 64), 2: (1024, 1024, 128), 3: (1024, 1024, 8)}[fmt]
    g = torch.Generator(device="cuda").manual_seed(1)
    pools = [[torch.randint(0, 256, (nb, Hkv * n), dtype=torch.uint8, device="cuda", generator=g) if n else None
              for n in sizes] for _ in range(layers)]
    perm = torch.randperm(nb, device="cuda", generator=g).to(torch.int32)
    src, dst = perm[:pairs].contiguous(), perm[pairs:2 * pairs].contiguous()
    src[0] = -1 if pairs > 3 else src[0]
    dst[-1] = nb if pairs > 3 else dst[-1]
    want = []
    good = ((src >= 0) & (dst < nb)).nonzero()[:, 0]
    for p in pools:
        w = [None if x is None else x.clone() for x in p]
        for x in w:
            if x is not None:
                x[dst[good].long()] = x[src[good].long()]
        want.append(w)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    views = gkv.cache_views([gkv.CacheView(p[0].data_ptr(), p[1].data_ptr(), None, 0, nb, Hkv, 0,
                                           None if p[2] is None else p[2].data_ptr(), fmt) for p in pools])
    gkv.copy_blocks(views, src, dst, dev_err=err)
    assert int(err.item()) == (gkv.DEVERR_BLOCK_ID if pairs > 3 else 0)
    for p, w in zip(pools, want):
        for x, y in zip(p, w):
            assert x is None or torch.equal(x, y)
