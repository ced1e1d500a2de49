"""gkv_shared_decode on the GPU against its definition in 64 bits (tolerances derived in
sharedcase.py)."""
import numpy as np
import pytest
import torch

from keptcase import BF16, BLOCK, BT, D
from oracle import kv_oracle as O
from sharedcase import Shared, dev, shared_bound, within

pytestmark = pytest.mark.gpu


def check(gkv, lens, sizes, shared, Hq, Hkv, fmt, bf16, sinks="some", seed=0, seen=None, err=0, prepare=None, spread=False,
          scale=1.0, poison=True, **kw):
    s = Shared(lens, sizes, shared, Hkv, fmt, seed=seed, spread=spread, scale=scale)
    if prepare:
        prepare(s)
    rng = np.random.default_rng(seed + 7)
    sk = rng.standard_normal(Hq).astype(np.float32) * 2 if isinstance(sinks, str) else sinks
    got, q, *_ = s.run(gkv, Hq, sk, bf16, **kw)
    out, pav, qk, qm = s.expect(q, sk, seen)
    within(got, out, shared_bound(out, pav, qk, qm, fmt, bf16), f"{fmt} {bf16}")
    assert int(s.c.err.item()) == err
    return got


FORMS = [(BF16, True), (BF16, False), (BLOCK, True), (BLOCK, False)]


@pytest.mark.parametrize("fmt,bf16", FORMS)
def test_the_smallest(gkv, cuda, fmt, bf16):
    check(gkv, [16, 17], [2], [1], 8, 1, fmt, bf16)
    check(gkv, [1], [1], [0], 8, 1, fmt, bf16)
    check(gkv, [33, 48, 50], [3], [2], 2, 2, fmt, bf16, sinks=None)


@pytest.mark.parametrize("fmt,bf16", FORMS)
def test_groups_of_all_kinds(gkv, cuda, fmt, bf16):
    """Odd and even numbers of blocks, one block, none; sequences that end with the shared blocks, before
    them, or are empty; a group of one, one of none, and sequences in no group."""
    lens = [5 * BT + 3, 5 * BT, 5 * BT + 40, 7, 0,   # five blocks; two are shorter
            6 * BT + 1, 6 * BT + 100,                # six
            12 * BT + 16,                            # alone
            BT + 1, BT + 2, BT, 3,                   # one block
            50, 60,                                  # nothing shared
            90, 0, 1, 17]                            # in no group
    check(gkv, lens, [5, 2, 1, 0, 4, 2], [5, 6, 12, 9, 1, 0], 16, 2, fmt, bf16)


@pytest.mark.parametrize("fmt,bf16", FORMS)
@pytest.mark.parametrize("Hq,Hkv", [(64, 8), (40, 8), (6, 3), (7, 7), (8, 1), (5, 1), (21, 3), (32, 4)])
def test_head_counts(gkv, cuda, fmt, bf16, Hq, Hkv):
    rng = np.random.default_rng(Hq)
    check(gkv, 7 * BT + rng.integers(1, 60, 11), [4, 7], [7, 3], Hq, Hkv, fmt, bf16, seed=Hq)


@pytest.mark.parametrize("fmt,bf16", FORMS)
@pytest.mark.parametrize("sizes,blocks", [([2], 40), ([3], 41), ([9], 64), ([17, 2, 30], 21), ([70], 33), ([200], 9)])
def test_group_sizes_and_splits(gkv, cuda, fmt, bf16, sizes, blocks):
    """One query tile and many, shared blocks in one part and in many."""
    rng = np.random.default_rng(blocks)
    n = sum(sizes)
    check(gkv, blocks * BT + rng.integers(0, 40, n), sizes, [blocks - i for i in range(len(sizes))], 8, 1, fmt, bf16,
          seed=blocks)


@pytest.mark.parametrize("fmt,bf16", FORMS)
def test_long_prefix(gkv, cuda, fmt, bf16):
    check(gkv, [9000 + 5, 9000 + 70], [2], [562], 8, 1, fmt, bf16)


@pytest.mark.parametrize("fmt,bf16", FORMS)
@pytest.mark.parametrize("hints", [None, (0, 0), (3, 16), (1000, 16), (3, 100000), (4000, 100000)])
def test_bounds_only_pick_the_form(gkv, cuda, fmt, bf16, hints):
    """Own tokens in one workgroup or in pieces, whatever the call was told."""
    check(gkv, [16 * 30 + 5200, 16 * 30 + 3, 16 * 30 + 2400, 700], [3], [30], 8, 1, fmt, bf16, hints=hints)


@pytest.mark.parametrize("fmt,bf16", FORMS)
def test_rotated_queries_and_strides(gkv, cuda, fmt, bf16):
    lens = [100, 64, 80, 99]
    check(gkv, lens, [4], [4], 16, 2, fmt, bf16, rotate=False)
    check(gkv, lens, [4], [4], 16, 2, fmt, bf16, pad=12)


@pytest.mark.parametrize("fmt,bf16", FORMS)
def test_sinks_and_large_scores(gkv, cuda, fmt, bf16):
    lens, args = [200, 180, 177, 161], ([4], [10], 8, 2, fmt, bf16)
    check(gkv, lens, *args, sinks=np.full(8, -np.inf, np.float32))
    check(gkv, lens, *args, sinks=np.linspace(-40, 60, 8).astype(np.float32))
    check(gkv, lens, *args, q_scale=6.0, seed=3)
    check(gkv, lens, *args, q_scale=6.0, sinks=None, spread=True, seed=4)


@pytest.mark.parametrize("fmt,bf16", FORMS)
def test_what_nothing_sees_counts_for_nothing(gkv, cuda, fmt, bf16):
    """(Every slot behind a sequence's last token holds a NaN in Cache.)"""
    check(gkv, [3 * BT + 1, 3 * BT + 15, 4 * BT, 3 * BT], [4], [3], 8, 2, fmt, bf16, sinks=None)


@pytest.mark.parametrize("fmt,bf16", FORMS)
@pytest.mark.parametrize("which", [[0], [2], [3, 4], [0, 1, 2, 3, 4]])
def test_ids_outside_the_pool(gkv, cuda, fmt, bf16, which):
    """Their tokens count for nothing, and are flagged."""
    lens = [5 * BT + 4, 5 * BT, 5 * BT + 20]
    seen = [np.array([t for t in range(L) if t // BT not in which]) for L in lens]

    def spoil(s):
        for i, j in enumerate(which):
            s.c.table[0, j] = [-1, s.c.nb, 2**31 - 1, -2**31, -7][i]

    for sinks in ("some", None):
        check(gkv, lens, [3], [5], 8, 1, fmt, bf16, sinks=sinks, prepare=spoil, seen=seen, err=1)


def test_nothing_seen_gives_zeros(gkv, cuda):
    def spoil(s):
        s.c.table[:] = -3

    got = check(gkv, [64, 64], [2], [4], 8, 1, BF16, False, sinks=None, prepare=spoil,
                seen=[np.zeros(0, int)] * 2, err=1)
    assert (got == 0).all()


def test_a_scale_that_is_nan(gkv, cuda):
    s = Shared([100, 90, 30], [2], [5], 1, BLOCK)
    s.c.s[s.c.table[0, 2], 0, 0] = np.nan
    got = s.run(gkv, 8, None, True)[0]
    assert np.isnan(got[:2]).all() and np.isfinite(got[2]).all()


def test_lengths_past_the_bound(gkv, cuda):
    """Taken at the bound, and flagged; more shared blocks than a row has, too."""
    s = Shared([100, 90], [2], [5], 1, BF16)
    whole = s.run(gkv, 8, None, False)[0]
    assert int(s.c.err.item()) == 0
    got = s.run(gkv, 8, None, False, max_len=90)[0]
    assert int(s.c.err.item()) == 2 and np.array_equal(got[1], whole[1]) and np.isfinite(got).all()
    s.c.table[1, :5] = s.c.table[0, :5]
    s.shared[:] = 2**31 - 1
    got = s.run(gkv, 8, None, False, hints=(5, 100))[0]  # (no sequence is that long: each on its own)
    assert int(s.c.err.item()) == 2 and np.allclose(got[0], whole[0], atol=1e-5)
    s.shared[:] = -5
    s.run(gkv, 8, None, False, hints=(5, 100))


@pytest.mark.parametrize("cu", [[0, 9], [-5, 3], [3, 0], [2**31 - 1, 2**31 - 1], [-2**31, -2**31], [1, 2]])
def test_groups_that_are_none(gkv, cuda, cu):
    """Offsets outside the batch read and write nothing outside it."""
    s = Shared([100, 90, 80], [3], [0], 1, BF16)
    s.c.table[:] = s.c.table[:1]
    for b in (1, 2):
        for x, y in zip(s.c.kv[b], s.c.kv[0]):
            x[:] = y[:len(x)]
    s.cu = np.asarray(cu, np.int32)
    s.shared = np.array([4], np.int32)
    got = s.run(gkv, 8, None, False, hints=(4, 50))[0]
    assert np.isfinite(got).all()


def test_the_same_as_the_other_decode(gkv, cuda):
    """A table whose rows do hold the shared blocks, read both ways."""
    for fmt, bf16 in FORMS:
        s = Shared(np.arange(130, 142), [5, 7], [8, 8], 8, fmt)
        for g in (0, 1):
            s.c.table[s.cu[g]:s.cu[g + 1], :8] = s.c.table[s.cu[g], :8]
        got, q, x, out, _ = s.run(gkv, 64, None, bf16, rotate=False)
        other = torch.empty_like(out)
        view = gkv.cache_view(s.c.dk, s.c.dv, s.c.dt, 8, v_scale=s.c.ds, v_format=fmt)
        gkv.kept_decode(x, 64, dev(s.c.lens), 141, view, other, dev_err=s.c.err)
        _, pav, qk, qm = s.expect(q, None)
        within(got, other.float().cpu().numpy().reshape(got.shape), 2 * shared_bound(got, pav, qk, qm, fmt, bf16))


def test_the_same_bits_again(gkv, cuda):
    s = Shared(np.arange(900, 916), [16], [50], 8, BLOCK)
    first = s.run(gkv, 64, None, True)
    for _ in range(3):
        first[4]()
        assert np.array_equal(first[3].float().cpu().numpy().reshape(first[0].shape), first[0])


def test_many_sequences(gkv, cuda):
    """More of them than pieces are kept for; a sample is looked at."""
    n = 5000
    s = Shared(np.full(n, 3 * BT) + np.arange(n) % 20, [n - 40, 40], [3, 3], 1, BF16, extra=0)
    got, q, *_ = s.run(gkv, 4, None, True)
    for b in (0, 1, 63, 64, 4095, n - 41, n - 40, n - 1):
        one = Shared.__new__(Shared)
        one.c, one.B = s.c, 1
        keep = s.c.lens, s.c.kv
        s.c.lens, s.c.kv = keep[0][b:b + 1], keep[1][b:b + 1]
        out, pav, qk, qm = one.expect(q[b:b + 1], None)
        s.c.lens, s.c.kv = keep
        within(got[b:b + 1], out, shared_bound(out, pav, qk, qm, BF16, True), f"sequence {b}")


@pytest.mark.parametrize("fmt,bf16", FORMS)
def test_captured_calls_share_a_workspace_in_order(gkv, cuda, fmt, bf16):
    """Two captured calls on one workspace, replayed in turn on a stream of their own, with lengths
    and counts of shared blocks that change."""
    a = Shared([300, 330, 310, 290], [4], [18], 8, fmt, seed=1)
    b = Shared(np.arange(200, 209), [5, 4], [12, 10], 8, fmt, seed=2)
    parts, ws = [], None
    for s in (a, b):
        for g in range(len(s.shared)):  # rows that hold the shared blocks: any count up to theirs is right
            s.c.table[s.cu[g]:s.cu[g + 1], :s.shared[g]] = s.c.table[s.cu[g], :s.shared[g]]
        view = s.c.device(gkv)
        q = torch.randn(s.B, 64 * 64, device="cuda")
        out = torch.zeros(s.B, 64 * 64, dtype=torch.bfloat16 if bf16 else torch.float32, device="cuda")
        parts.append((s, view, q, out, dev(s.cu), dev(s.shared), dev(s.c.lens)))
    n = max(gkv.shared_workspace_bytes(s.B, len(s.shared), 64, 8, 18, 200) for s in (a, b))
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    side, graphs = torch.cuda.Stream(), []
    side.wait_stream(torch.cuda.current_stream())
    for s, view, q, out, cu, sh, lens in parts:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=side):
            gkv.shared_decode(q, 64, cu, sh, lens, 400, view, out, 18, 200, workspace=ws, dev_err=s.c.err)
    for i in range(4):
        for s, view, q, out, cu, sh, lens in parts:
            lens.copy_(dev(s.c.lens - 5 * i))
            sh.copy_(dev(np.maximum(s.shared - 3 * i, 0)))
            q.normal_()
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.default_stream())
            for g in graphs:
                g.replay()
        torch.cuda.synchronize()
        for s, view, q, out, cu, sh, lens in parts:
            eager = torch.empty_like(out)
            gkv.shared_decode(q, 64, cu, sh, lens, 400, view, eager, 18, 200, workspace=ws, dev_err=s.c.err)
            assert torch.equal(eager, out)
            assert int(s.c.err.item()) == 0


def test_on_another_stream(gkv, cuda):
    """Inputs made on a stream of its own, the call on that stream, by name or as the current one."""
    s = Shared([300, 310, 290], [3], [18], 8, BLOCK, seed=4)
    whole = s.run(gkv, 64, None, True)
    x, out = whole[2], whole[3]
    view = s.c.device(gkv)
    cu, sh, lens, ws = dev(s.cu), dev(s.shared), dev(s.c.lens), s.ws
    cos, sin = (dev(t) for t in O.rope_table(310))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for named in (True, False):
        q, got = torch.zeros_like(x), torch.zeros_like(out)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(2000000)
            q.copy_(x)
            call = dict(sinks=None, cos_tab=cos, sin_tab=sin, workspace=ws, dev_err=s.c.err)
            if not named:
                gkv.shared_decode(q, 64, cu, sh, lens, 310, view, got, 18, 20, **call)
        if named:
            gkv.shared_decode(q, 64, cu, sh, lens, 310, view, got, 18, 20, stream=side, **call)
        side.synchronize()
        assert torch.equal(got, out)


@pytest.mark.parametrize("shared", [2**27, 2**27 + 1, 2**31 - 1, 9])
def test_more_shared_blocks_than_a_sequence_has(gkv, cuda, shared):
    """(A row of 40 entries.) Nobody is that long: each on its own."""
    s = Shared([100, 90], [2], [5], 1, BF16)
    whole = s.run(gkv, 8, None, False)[0]
    s.c.table[1, :5] = s.c.table[0, :5]
    s.shared[:] = shared
    got = s.run(gkv, 8, None, False, hints=(min(shared, 2**20), 100))[0]
    assert int(s.c.err.item()) == (2 if shared > s.c.table.shape[1] else 0)
    assert np.allclose(got, whole, atol=1e-5)


@pytest.mark.parametrize("fmt,bf16", FORMS)
@pytest.mark.parametrize("size", [3, 7, 14, 40])
def test_many_steps_of_a_wave(gkv, cuda, fmt, bf16, size):
    """75 or 150 steps of two blocks, ids outside the pool among them: 24, 56, 112 and 320 query heads to
    a kv head, all blocks in one part (told of no shared ones)."""
    blocks, which = 299, [0, 63, 64, 127, 128, 131, 192, 298]
    lens = blocks * BT + np.arange(size) % 18
    seen = [np.array([t for t in range(L) if t // BT not in which]) for L in lens]

    def spoil(s):
        s.c.table[0, which] = [-1, s.c.nb, 2**31 - 1, -2**31, -7, -5, s.c.nb + 1, -1]

    check(gkv, lens, [size], [blocks], 8, 1, fmt, bf16, hints=(0, 0), prepare=spoil, seen=seen, err=1, seed=size)


@pytest.mark.parametrize("fmt", [BF16, BLOCK])
def test_blocks_past_4_gib(gkv, cuda, fmt):
    """The same blocks behind 4 GiB of others: the same bits."""
    s = Shared([300, 310, 290], [3], [17], 8, fmt, seed=4)
    got, q, x, out, _ = s.run(gkv, 64, None, True, rotate=False)
    ahead = 2**32 // (8 * BT * D * (2 if fmt == BF16 else 1)) + 5
    far = [None if t is None else torch.zeros((ahead + s.c.nb,) + t.shape[1:], dtype=t.dtype, device="cuda")
           for t in (s.c.dk, s.c.dv, s.c.ds)]
    for t, f in zip((s.c.dk, s.c.dv, s.c.ds), far):
        if t is not None:
            f[ahead:] = t
    table = dev(np.where(s.c.table >= 0, s.c.table + ahead, s.c.table).astype(np.int32))
    view = gkv.cache_view(far[0], far[1], table, 8, v_scale=far[2], v_format=fmt)
    again = torch.zeros_like(out)
    gkv.shared_decode(x, 64, dev(s.cu), dev(s.shared), dev(s.c.lens), 310, view, again, 17, 38, workspace=s.ws,
                      dev_err=s.c.err)
    assert torch.equal(again, out) and int(s.c.err.item()) == 0


@pytest.mark.parametrize("fmt,bf16", FORMS)
def test_no_groups(gkv, cuda, fmt, bf16):
    """Every sequence on its own: short ones, and ones of several pieces."""
    check(gkv, [17, 0, 1, 300], [], [], 16, 2, fmt, bf16)
    check(gkv, [5000, 17], [], [], 8, 1, fmt, bf16)
