"""The gkv_kept_* entry points where a call takes another way than the short ones: long
bounds, many sequences, pools past 4 GiB, other streams, padded rows, values at the range's end."""
import numpy as np
import pytest
import torch

from keptcase import BF16, BLOCK, D, Cache, Layout, attend, decode_bound, prefill_bound
from oracle import kv_oracle as O
from test_gpu_kept import dev, run_decode, run_prefill

pytestmark = pytest.mark.gpu

LONG = 20000  # a bound past which the decode cuts sequences into ranges, whatever their lengths
WIDE = 4800   # a window past it


@pytest.mark.parametrize("fmt", [BF16, BLOCK])
@pytest.mark.parametrize("kept,window,ring", [(0, 0, False), (16, WIDE, True), (48, WIDE, False)])
@pytest.mark.parametrize("lens", [[1], [0, 0, 0], [0, 1, 15, 16, 17], [33, 250, 0, 64, 31, 129], [700, 3]])
def test_ranges_of_short_sequences(gkv, cuda, fmt, kept, window, ring, lens):
    assert gkv.kept_workspace_bytes(len(lens), 2, LONG, kept, window) > 0
    run_decode(gkv, lens, 16, 2, Layout(kept, window, ring), fmt, seed=kept + len(lens), max_len=LONG,
               sinks=len(lens) % 2 == 0, bf16=len(lens) == 5, spread=len(lens) == 6)


@pytest.mark.parametrize("fmt", [BF16, BLOCK])
@pytest.mark.parametrize("Hq,Hkv", [(64, 8), (6, 3), (7, 7), (8, 1), (5, 5), (24, 4)])
def test_ranges_of_all_head_counts(gkv, cuda, fmt, Hq, Hkv):
    run_decode(gkv, [40, 0, 900, 17], Hq, Hkv, Layout(0, 0, False), fmt, seed=Hq, sinks=Hq % 2 == 0, max_len=LONG)


@pytest.mark.parametrize("fmt", [BF16, BLOCK])
@pytest.mark.parametrize("kept,window,ring", [(0, 0, False), (16, WIDE, True), (32, WIDE, False)])
def test_ranges_of_long_sequences(gkv, cuda, fmt, kept, window, ring):
    run_decode(gkv, [7003, 5, 0, 5200], 8, 2, Layout(kept, window, ring), fmt, max_len=LONG)


@pytest.mark.parametrize("fmt", [BF16, BLOCK])
@pytest.mark.parametrize("B,Hkv,window", [(300, 8, 0), (300, 8, 32), (150, 8, 0), (70, 8, 48), (70, 5, 0), (40, 8, 0)])
def test_many_sequences(gkv, cuda, fmt, B, Hkv, window):
    """One, two, four and eight waves per sequence and head."""
    lens = [int(x) for x in np.random.default_rng(B).integers(0, 90, B)]
    run_decode(gkv, lens, Hkv, Hkv, Layout(16 if window else 0, window, bool(window)), fmt, max_len=512)


def test_the_workspace_of_a_batch_does_for_a_smaller_one(gkv, cuda):
    for kept, window, max_len in ((0, 0, 3000), (64, 4096, 9000), (0, 0, 2000), (16, 128, 100000)):
        need = [gkv.kept_workspace_bytes(B, 8, max_len, kept, window) for B in (1, 11, 12, 500)]
        assert sorted(need) == need and need[0] in (0, need[-1])


@pytest.mark.parametrize("fmt", [BF16, BLOCK])
@pytest.mark.parametrize("kept,window,ring", [(0, 0, False), (32, 128, True)])
def test_prefill_of_any_scales(gkv, cuda, fmt, kept, window, ring):
    """Block scales that are no powers of two, blocks of very different size (magnitudes
    2^-9 .. 2^2)."""
    run_prefill(gkv, [208, 16, 336], [70, 33, 5], 16, 2, Layout(kept, window, ring), fmt, spread=True, scale=0.125)


@pytest.mark.parametrize("fmt", [BF16, BLOCK])
@pytest.mark.parametrize("kept,window,ring", [(0, 0, False), (16, 32, True), (0, 16, True), (96, 48, True),
                                              (32, 256, False)])
@pytest.mark.parametrize("Hq,Hkv", [(16, 2), (4, 2), (4, 1)])
@pytest.mark.parametrize("max_len", [130, 20000])
def test_prefill_in_one_and_two_groups(gkv, cuda, fmt, kept, window, ring, Hq, Hkv, max_len):
    """Few workgroups split their tiles between two groups of waves, many do not (the bound of
    the lengths decides)."""
    run_prefill(gkv, [0, 16, 208, 336, 48, 1024], [5, 33, 70, 16, 130, 40], Hq, Hkv, Layout(kept, window, ring), fmt,
                sinks=Hq % 8 == 0, seed=kept, bf16=Hq == 4, max_len=max_len)


HUGE = 2**31 - 16


@pytest.mark.parametrize("kept,window", [(0, HUGE), (HUGE, 16), (HUGE, HUGE), (1 << 30, 1 << 30)])
def test_masks_wider_than_any_sequence(gkv, cuda, kept, window):
    """... are the causal mask."""
    lay = Layout(0, 0, False)
    c = Cache([96, 33], 2, lay, BLOCK)
    view = c.device(gkv)
    g = torch.Generator(device="cuda").manual_seed(3)
    q = torch.randn(60, 4 * D, generator=g, device="cuda")
    kv = [torch.randn(60, 2 * D, generator=g, device="cuda").bfloat16() for _ in "kv"]
    cu, start = dev(np.array([0, 40, 60], np.int32)), dev(np.array([80, 32], np.int32))
    lens = dev(np.array([96, 33], np.int32))
    outs = []
    for k, w in ((0, 0), (kept, window)):
        out = torch.zeros(60, 4 * D, device="cuda")
        gkv.kept_prefill(cu, 40, q, 4, view, out, start_pos=start, k=kv[0], v=kv[1], kept=k, window=w, dev_err=c.err)
        one = torch.zeros(2, 4 * D, device="cuda")
        gkv.kept_decode(q[:2], 4, lens, 96, view, one, kept=k, window=w, dev_err=c.err)
        outs.append((out, one))
    assert all(torch.equal(x, y) for x, y in zip(*outs)) and int(c.err.item()) == 0


def test_prefill_leaves_other_rows_alone(gkv, cuda):
    """Prompts without rows, rows behind the last prompt, padding between the rows."""
    g = torch.Generator(device="cuda").manual_seed(4)
    q = torch.randn(50, 4 * D + 4, generator=g, device="cuda")
    k, v = (torch.randn(50, 2 * D, generator=g, device="cuda").bfloat16() for _ in "kv")
    cu = dev(np.array([0, 0, 33, 33, 40], np.int32))
    for dt in (torch.bfloat16, torch.float32):
        pad = torch.full((50, 4 * D + 8), 7.0, dtype=dt, device="cuda")
        out = torch.zeros(50, 4 * D, dtype=dt, device="cuda")
        view = gkv.CacheView(n_kv_heads=2)
        gkv.kept_prefill(cu, 33, q[:, :4 * D], 4, view, pad[:, :4 * D], k=k, v=v, window=16)
        gkv.kept_prefill(cu, 33, q[:, :4 * D].contiguous(), 4, view, out, k=k, v=v, window=16)
        assert torch.equal(pad[:40, :4 * D], out[:40])
        assert (pad[40:] == 7).all() and (pad[:, 4 * D:] == 7).all() and (out[40:] == 0).all()


@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("x,flag", [(65280.0, False), (65536.0, True), (-1e30, True), (float("inf"), True)])
def test_prefill_flags_values_beyond_its_range(gkv, cuda, where, x, flag):
    x = x if where == "k" else x * 1024  # V is taken as v * 2^-10
    k, v = torch.zeros(40, D, dtype=torch.bfloat16, device="cuda"), torch.ones(40, D, dtype=torch.bfloat16, device="cuda")
    (k if where == "k" else v)[7, 3] = x
    q = torch.ones(40, D, device="cuda")
    out, err = torch.zeros(40, D, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    gkv.kept_prefill(dev(np.array([0, 40], np.int32)), 40, q, 1, gkv.CacheView(n_kv_heads=1), out, k=k, v=v,
                     dev_err=err)
    assert int(err.item()) == (gkv.DEVERR_RANGE if flag else 0)
    assert torch.isfinite(out).all() or flag


def test_a_cached_k_beyond_the_range_is_flagged(gkv, cuda):
    c = Cache([32], 1, Layout(0, 0, False), BF16)
    view = c.device(gkv)
    c.dk[int(c.table[0, 1])].fill_(int(np.float32(-1e9).view(np.int32)) >> 16)
    q, kv = torch.ones(4, D, device="cuda"), torch.zeros(4, D, dtype=torch.bfloat16, device="cuda")
    out = torch.zeros(4, D, device="cuda")
    gkv.kept_prefill(dev(np.array([0, 4], np.int32)), 4, q, 1, view, out, start_pos=dev(np.array([32], np.int32)),
                     k=kv, v=kv, dev_err=c.err)
    assert int(c.err.item()) == gkv.DEVERR_RANGE


@pytest.mark.parametrize("fmt,blocks", [(BF16, 265000), (BLOCK, 530000)])
def test_a_pool_past_32_bits(gkv, cuda, fmt, blocks):
    """Blocks beyond 4 GiB of K: append, decode (whole and ranges), prefill and copies give what
    they give at the pool's start."""
    Hq, Hkv, B, n = 16, 8, 2, 40
    dt, el = (torch.int16, 1024) if fmt == BF16 else (torch.uint8, 1024)
    ids = np.arange(B * n).reshape(B, n).astype(np.int32)
    pools = []
    for nb, table in ((2 * B * n, ids), (blocks, blocks - 1 - ids)):
        k, v = (torch.empty(nb, Hkv, el, dtype=dt, device="cuda") for _ in "kv")
        s = torch.empty(nb, Hkv, 2, device="cuda") if fmt == BLOCK else None
        t = dev(np.ascontiguousarray(table))
        pools.append((gkv.cache_view(k, v, t, Hkv, v_scale=s, v_format=fmt), k, v, s, t))
    assert pools[1][1].nbytes > 2**32
    g = torch.Generator(device="cuda").manual_seed(5)
    lens, rows = np.array([515, 300], np.int32), np.array([400, 300], np.int32)
    qkv = torch.randn(int(rows.sum()), (Hq + 2 * Hkv) * D, generator=g, device="cuda")
    cos, sin = (dev(x) for x in O.rope_table(LONG))
    cu = dev(np.concatenate([[0], np.cumsum(rows)]).astype(np.int32))
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    ws = torch.zeros(gkv.kept_workspace_bytes(B, Hkv, LONG), dtype=torch.uint8, device="cuda")

    def attention(view):
        res = []
        for bound in (600, LONG):
            out = torch.zeros(B, Hq * D, device="cuda")
            gkv.kept_decode(qkv[:B], Hq, dev(lens), bound, view, out, cos_tab=cos, sin_tab=sin, workspace=ws,
                            dev_err=err)
            res.append(out)
        out = torch.zeros(6, Hq * D, device="cuda")
        gkv.kept_prefill(dev(np.array([0, 3, 6], np.int32)), 3, qkv[:6], Hq, view, out,
                         start_pos=dev(np.array([496, 288], np.int32)), cos_tab=cos, sin_tab=sin, dev_err=err)
        return res + [out]

    got = []
    for view, *_ in pools:
        # (the first sequence's older tokens in a call of their own: a block is continued)
        gkv.kept_append(qkv[:115], Hq, cos, sin, dev(np.array([115, 0], np.int32)), view, max_rows=115,
                        cu_seqlens=dev(np.array([0, 115, 115], np.int32)), dev_err=err)
        gkv.kept_append(qkv, Hq, cos, sin, dev(lens), view, max_rows=400, cu_seqlens=cu, dev_err=err)
        got.append(attention(view))
    assert all(torch.equal(x, y) for x, y in zip(*got)) and all(torch.isfinite(x).all() for x in got[0])
    # far blocks to near places of the same pool
    view, _, _, _, table = pools[1]
    near = dev(ids.reshape(-1))
    gkv.copy_blocks([view], table.reshape(-1), near, dev_err=err)
    view.block_table = near.data_ptr()
    assert all(torch.equal(x, y) for x, y in zip(got[0], attention(view)))
    assert int(err.item()) == 0


@pytest.mark.parametrize("fmt", [BF16, BLOCK])
def test_two_streams_with_workspaces_of_their_own(gkv, cuda, fmt):
    lay = Layout(0, 0, False)
    c = Cache([5000, 900, 2600], 2, lay, fmt)
    view = c.device(gkv)
    g = torch.Generator(device="cuda").manual_seed(6)
    q = [torch.randn(3, 4 * D, generator=g, device="cuda") for _ in range(2)]
    lens = [dev(np.array(x, np.int32)) for x in ([5000, 900, 2600], [3000, 1, 2599])]
    ws = [torch.zeros(gkv.kept_workspace_bytes(3, 2, LONG), dtype=torch.uint8, device="cuda") for _ in range(2)]
    out = [torch.zeros(3, 4 * D, device="cuda") for _ in range(4)]
    for i in range(2):
        gkv.kept_decode(q[i], 4, lens[i], LONG, view, out[i], workspace=ws[i], dev_err=c.err)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for i, s in enumerate(streams):
            gkv.kept_decode(q[i], 4, lens[i], LONG, view, out[2 + i], workspace=ws[i], dev_err=c.err, stream=s)
    torch.cuda.synchronize()
    assert torch.equal(out[0], out[2]) and torch.equal(out[1], out[3]) and int(c.err.item()) == 0


@pytest.mark.parametrize("fmt", [BF16, BLOCK])
def test_captured_ranges_share_a_workspace_in_order(gkv, cuda, fmt):
    """Two captured calls of one workspace, replayed in turn with lengths that change."""
    c = Cache([4000, 900], 1, Layout(0, 0, False), fmt)
    view = c.device(gkv)
    q = torch.randn(2, 4 * D, generator=torch.Generator(device="cuda").manual_seed(7), device="cuda")
    now = torch.zeros(2, dtype=torch.int32, device="cuda")
    ws = torch.zeros(gkv.kept_workspace_bytes(2, 1, LONG), dtype=torch.uint8, device="cuda")
    outs = [torch.zeros(2, 4 * D, device="cuda") for _ in range(3)]

    def call(i):
        gkv.kept_decode(qs[i], 4, now, LONG, view, outs[i], workspace=ws, dev_err=c.err)

    qs = [q, q * 0.5]
    call(0)
    torch.cuda.synchronize()
    graphs = []
    for i in range(2):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            call(i)
        graphs.append(graph)
    for lens in ([4000, 900], [1, 0], [2500, 64], [0, 0]):
        now.copy_(dev(np.array(lens, np.int32)))
        for i in (0, 1, 0):
            graphs[i].replay()
            torch.cuda.synchronize()
            got = outs[i].clone()
            gkv.kept_decode(qs[i], 4, now, LONG, view, outs[2], workspace=ws, dev_err=c.err)
            assert torch.equal(got, outs[2])
    assert int(c.err.item()) == 0


@pytest.mark.parametrize("max_len", [64, LONG])
@pytest.mark.parametrize("fmt", [BF16, BLOCK])
def test_fp32_outputs_keep_more_than_two_bf16_pieces(gkv, cuda, fmt, max_len):
    """Two positions, scores near 0. In units of 2^-24: the scores' sums 70 of sum |q k|, their
    exponent's argument 1, exp2 and its place in both sums 4, the sum 2, six products and
    their sums 8, joining the pieces 1, the quotient and its product 2, q's pieces below
    these: 24 with the rest. Two bf16 pieces of a weight leave up to 2^-18 of it."""
    lay = Layout(0, 0, False)
    c = Cache([2] * 40, 2, lay, fmt, seed=9)
    view = c.device(gkv)
    q = (np.random.default_rng(9).standard_normal((40, 16, D)) / 256).astype(np.float32)
    out = torch.zeros(40, 16 * D, device="cuda")
    ws = torch.zeros(max(16, gkv.kept_workspace_bytes(40, 2, max_len)), dtype=torch.uint8, device="cuda")
    gkv.kept_decode(dev(q.reshape(40, -1)), 16, dev(np.full(40, 2, np.int32)), max_len, view, out, workspace=ws,
                    dev_err=c.err)
    got = out.cpu().numpy().reshape(40, 16, D)
    for b in range(40):
        want, pav, qk = attend(q[b:b + 1].astype(np.float64), *c.kv[b], np.ones((1, 2), bool), None)
        bound = pav * (2 * qk * 70 + 24) * 2.0 ** -24
        assert (np.abs(got[b] - want[0]) <= bound[0]).all()


def test_calls_go_to_the_current_stream(gkv, cuda):
    s = torch.cuda.Stream()
    assert gkv.stream_handle() == torch.cuda.current_stream().cuda_stream
    with torch.cuda.stream(s):
        assert gkv.stream_handle() == s.cuda_stream
    assert gkv.stream_handle(s) == s.cuda_stream


@pytest.mark.parametrize("fmt", [BF16, BLOCK])
@pytest.mark.parametrize("max_len", [64, LONG])
def test_far_more_sequences_than_workgroups(gkv, cuda, fmt, max_len):
    """70001 sequences that read the same two blocks, every seventh of them empty."""
    B = 70001
    c = Cache([20], 1, Layout(0, 0, False), fmt, seed=3)
    view = c.device(gkv)
    table = c.dt[:, :2].repeat(B, 1).contiguous()
    view.block_table, view.table_stride = table.data_ptr(), 2
    q = torch.randn(1, 2 * D, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").repeat(B, 1)
    lens = torch.full((B,), 20, dtype=torch.int32, device="cuda")
    lens[::7] = 0
    out = torch.full((B, 2 * D), 7.0, device="cuda")
    ws = torch.zeros(max(16, gkv.kept_workspace_bytes(B, 1, max_len)), dtype=torch.uint8, device="cuda")
    gkv.kept_decode(q, 2, lens, max_len, view, out, workspace=ws, dev_err=c.err)
    assert int(c.err.item()) == 0
    empty = lens == 0
    assert (out[empty] == 0).all() and (out[~empty] == out[1]).all()
    want, pav, qk = attend(q[:1].cpu().numpy().reshape(1, 2, D).astype(np.float64), *c.kv[0], np.ones((1, 20), bool), None)
    assert (np.abs(out[1].cpu().numpy().reshape(2, D) - want[0]) <= decode_bound(want, pav, qk, fmt, False)[0]).all()


@pytest.mark.parametrize("fmt", [BF16, BLOCK])
@pytest.mark.parametrize("max_len", [3, 20000])
def test_a_million_tokens(gkv, cuda, fmt, max_len):
    """... of one block, which every table entry names: attention over that block. In the
    prefill a lane's sums take 32768 steps, 2^-24 of themselves each; the rows' own keys are
    zeros."""
    n = 65536
    c = Cache([16], 1, Layout(0, 0, False), fmt, seed=3)
    view = c.device(gkv)
    table = c.dt[:, :1].repeat(1, n + 1).contiguous()
    view.block_table, view.table_stride = table.data_ptr(), n + 1
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn(3, 4 * D, generator=g, device="cuda")
    k, v = c.kv[0]
    want, pav, qk = attend(q.cpu().numpy().reshape(3, 4, D).astype(np.float64), k, v, np.ones((3, 16), bool), None)
    out = torch.zeros(1, 4 * D, device="cuda")
    ws = torch.zeros(gkv.kept_workspace_bytes(1, 1, 16 * n), dtype=torch.uint8, device="cuda")
    gkv.kept_decode(q[:1], 4, dev(np.array([16 * n], np.int32)), 16 * n, view, out, workspace=ws, dev_err=c.err)
    bound = decode_bound(want, pav, qk, fmt, False)
    assert (np.abs(out.cpu().numpy().reshape(4, D) - want[0]) <= bound[0]).all()
    out = torch.zeros(3, 4 * D, device="cuda")
    zero = torch.zeros(3, D, dtype=torch.bfloat16, device="cuda")
    gkv.kept_prefill(dev(np.array([0, 3], np.int32)), max_len, q, 4, view, out, start_pos=dev(np.array([16 * n], np.int32)),
                     k=zero, v=zero, dev_err=c.err)
    # (3 own keys of score 0 beside 2^20 of at least -max |score|)
    top = np.abs(np.einsum("nhd,td->nht", q.cpu().numpy().reshape(3, 4, D).astype(np.float64), k[:, 0])).max() / 8
    own = 3 * np.exp(top) / 2 ** 20
    bound = prefill_bound(want, pav, qk, 16, np.abs(v).max(), False) + pav * (2 * 32768 * 2.0 ** -24) + np.abs(want) * own
    assert (np.abs(out.cpu().numpy().reshape(3, 4, D) - want) <= bound).all() and int(c.err.item()) == 0


@pytest.mark.parametrize("fmt", [BF16, BLOCK])
@pytest.mark.parametrize("kept,window,ring", [(0, 0, False), (32, 64, False), (16, 128, True)])
@pytest.mark.parametrize("max_len", [70, 20000])
@pytest.mark.parametrize("Hq,Hkv", [(8, 1), (3, 1)])
def test_prefill_masks_missing_blocks(gkv, cuda, fmt, kept, window, ring, max_len, Hq, Hkv):
    """Blocks whose ids lie outside the pool are flagged, and their tokens count for nothing."""
    lay = Layout(kept, window, ring)
    starts, rows = [208, 64], [70, 40]
    c = Cache(starts, Hkv, lay, fmt, seed=8)
    gone = [np.zeros(s, bool) for s in starts]
    for b, blocks in enumerate(([0, 5, 8, 9, 12], [1, 3])):
        for j in blocks:
            c.table[b, lay.entry(j)] = [-1, c.nb, 2**31 - 1][j % 3]
        for j in range(starts[b] // 16):  # (on a ring a place is several blocks', the last one counts)
            gone[b][16 * j:16 * j + 16] = lay.entry(j) in [lay.entry(i) for i in blocks]
    view = c.device(gkv)
    rng = np.random.default_rng(8)
    q = rng.standard_normal((110, Hq, D)).astype(np.float32)
    kv = [torch.from_numpy(rng.standard_normal((110, Hkv, D)).astype(np.float32)).bfloat16() for _ in "kv"]
    out = torch.zeros(110, Hq * D, device="cuda")
    cu = np.array([0, 70, 110], np.int32)
    gkv.kept_prefill(dev(cu), max_len, dev(q.reshape(110, -1)), Hq, view, out, start_pos=dev(np.array(starts, np.int32)),
                     k=kv[0].cuda(), v=kv[1].cuda(), kept=kept, window=window, dev_err=c.err)
    assert int(c.err.item()) == gkv.DEVERR_BLOCK_ID
    got = out.cpu().numpy().reshape(110, Hq, D)
    for b in range(2):
        r = slice(cu[b], cu[b + 1])
        k, v = (np.concatenate([np.nan_to_num(x), y[r].double().numpy()]) for x, y in zip(c.kv[b], kv))
        t = np.arange(len(k))
        ok = np.stack([lay.sees(p, t) for p in range(starts[b], starts[b] + rows[b])])
        ok[:, :starts[b]] &= ~gone[b]
        want, pav, qk = attend(q[r].astype(np.float64), k, v, ok, None)
        assert (np.abs(got[r] - want) <= prefill_bound(want, pav, qk, len(k), np.abs(v).max(), False)).all()


def test_prefill_of_nothing_but_missing_blocks_is_zero(gkv, cuda):
    c = Cache([80], 1, Layout(0, 0, False), BLOCK)
    c.table[:] = -1
    view = c.device(gkv)
    for max_len in (40, 20000):
        out = torch.full((40, 2 * D), 7.0, device="cuda")
        gkv.kept_prefill(dev(np.array([0, 40], np.int32)), max_len, torch.ones(40, 2 * D, device="cuda"), 2, view, out,
                         start_pos=dev(np.array([32], np.int32)), dev_err=c.err)
        assert (out == 0).all() and int(c.err.item()) == gkv.DEVERR_BLOCK_ID


@pytest.mark.parametrize("fmt", [BF16, BLOCK])
@pytest.mark.parametrize("Hq,Hkv", [(40, 8), (6, 1), (14, 2), (64, 8)])
@pytest.mark.parametrize("kept,window,ring", [(0, 0, False), (16, 64, True)])
def test_prefill_of_all_group_sizes(gkv, cuda, fmt, Hq, Hkv, kept, window, ring):
    run_prefill(gkv, [128, 0, 320], [33, 1, 48], Hq, Hkv, Layout(kept, window, ring), fmt, sinks=Hq % 4 == 0, seed=Hq)
