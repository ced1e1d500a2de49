"""The pool's forks, trims and compactions, and a run of the kept-token entry points together on a
pool, as a serving loop uses them: prompts, decode steps, a fork, a trim, a free, a compaction.

In the run, every layer's cache is read back through the device table after each
append: each new token has to stand for its K and V within the format's rounding, every older one
must still do, and the attention is checked in 64 bits on what the cache holds."""
import numpy as np
import pytest
import torch

from keptcase import BF16, BLOCK, BT, D, PLACES, Layout, attend, decode_bound, e4m3_values, prefill_bound
from oracle import kv_oracle as O
from test_gpu_pool import dev_table

pytestmark = pytest.mark.gpu


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def pulled(gkv, ptr, n, dtype):
    t = torch.empty(n, dtype=dtype, device="cuda")
    gkv.hip_memcpy_d2d(t.data_ptr(), ptr, n * t.element_size())
    torch.cuda.synchronize()
    return t.cpu().numpy()


def fill(gkv, view, fmt, seed):
    """Random bytes in a layer's arrays; returns them."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    sizes = {BF16: (2048, 2048, 0), BLOCK: (1024, 1024, 8)}[fmt]
    got = []
    for p, n in zip((view.k, view.v, view.v_scale), sizes):
        if n:
            t = torch.randint(0, 255, (view.num_blocks * view.n_kv_heads * n,), dtype=torch.uint8, device="cuda",
                              generator=g)
            gkv.hip_memcpy_d2d(p, t.data_ptr(), t.numel())
            got.append(t.cpu().numpy().reshape(view.num_blocks, -1))
    torch.cuda.synchronize()
    return got


def content(gkv, view, fmt):
    sizes = {BF16: (2048, 2048, 0), BLOCK: (1024, 1024, 8)}[fmt]
    return [pulled(gkv, p, view.num_blocks * view.n_kv_heads * n, torch.uint8).reshape(view.num_blocks, -1)
            for p, n in zip((view.k, view.v, view.v_scale), sizes) if n]


@pytest.mark.parametrize("fmt", [BF16, BLOCK])
def test_fork_shares_full_blocks_and_copies_the_last(gkv, cuda, fmt):
    pool = gkv.Pool(n_layers=4, n_kv_heads=2, max_seqs=4, max_seq_len=160, window=32, num_blocks=12,
                    shuffle_seed=3, v_format=fmt, kept=16)
    a = pool.seq_alloc()
    assert pool.reserve(a, 50) == 0  # 4 blocks
    data = [fill(gkv, pool.view(l), fmt, l) for l in range(4)]
    rings = dev_table(torch, gkv, pool.view(0), 4)
    assert pool.view(0).ring == 48 and pool.view(0).table_stride == 4
    c = pool.fork(a, 50)
    assert pool.free_blocks() == 7  # one copy
    d = pool.fork(c, 48)            # whole blocks only: none
    assert pool.free_blocks() == 7
    ba, bc, bd = pool.seq_blocks(a), pool.seq_blocks(c), pool.seq_blocks(d)
    assert list(ba[:3]) == list(bc[:3]) == list(bd) and ba[3] != bc[3]
    pool.sync()
    t = dev_table(torch, gkv, pool.view(1), 4)
    assert list(t[c, :4]) == list(bc) and list(t[d, :4]) == list(bd) + [-1]
    for l in range(4):
        for x, y in zip(data[l], content(gkv, pool.view(l), fmt)):
            want = x.copy()
            if l % 2:
                want[bc[3]] = x[ba[3]]
            else:  # the parent's ring, kept block included, block by block: 50 tokens use all 4, 48 three
                want[rings[c]] = x[rings[a]]
                want[rings[d][:3]] = x[rings[a]][:3]
            assert np.array_equal(want, y), l
    # a block goes back with its last holder
    assert pool.free(a) == 0
    assert pool.free_blocks() == 8
    assert pool.free(c) == 0
    assert pool.free_blocks() == 9
    assert pool.free(d) == 0
    assert pool.free_blocks() == 12
    pool.close()


def test_fork_takes_nothing_when_it_fails(gkv, cuda):
    pool = gkv.Pool(n_layers=1, n_kv_heads=1, max_seqs=2, max_seq_len=64, window=0, num_blocks=2, v_format=BLOCK)
    a = pool.seq_alloc()
    assert pool.reserve(a, 20) == 0
    for n, why in ((20, gkv.GKV_ERR_CAPACITY), (33, gkv.GKV_ERR_ARG), (-1, gkv.GKV_ERR_ARG), (65, gkv.GKV_ERR_ARG)):
        with pytest.raises(gkv.GkvError) as e:
            pool.fork(a, n)
        assert e.value.status == why
    with pytest.raises(gkv.GkvError) as e:
        pool.fork(1, 0)
    assert e.value.status == gkv.GKV_ERR_BLOCK
    b = pool.fork(a, 32)  # shared whole blocks need none
    assert pool.free_blocks() == 0 and list(pool.seq_blocks(b)) == list(pool.seq_blocks(a))
    with pytest.raises(gkv.GkvError) as e:
        pool.fork(a, 0)   # no sequence id left
    assert e.value.status == gkv.GKV_ERR_CAPACITY
    pool.close()


def test_trim_frees_and_never_leaves_a_shared_partial_block(gkv, cuda):
    pool = gkv.Pool(n_layers=2, n_kv_heads=1, max_seqs=3, max_seq_len=96, window=0, num_blocks=7, v_format=BF16)
    a = pool.seq_alloc()
    assert pool.reserve(a, 80) == 0
    data = [fill(gkv, pool.view(l), BF16, l) for l in range(2)]
    b = pool.fork(a, 64)
    before = list(pool.seq_blocks(a))
    pool.trim(a, 80)
    assert list(pool.seq_blocks(a)) == before
    pool.trim(a, 64)       # its own last block
    assert pool.free_blocks() == 3 and list(pool.seq_blocks(a)) == before[:4]
    pool.trim(b, 40)       # the third block is shared and now appended to: a copy
    bb = list(pool.seq_blocks(b))
    assert bb[:2] == before[:2] and bb[2] not in before[:4] and pool.free_blocks() == 2
    pool.sync()
    t = dev_table(torch, gkv, pool.view(0), 3)
    assert list(t[b]) == bb + [-1] * 3 and list(t[a]) == before[:4] + [-1, -1]
    for l in range(2):
        for x, y in zip(data[l], content(gkv, pool.view(l), BF16)):
            assert np.array_equal(y[bb[2]], x[before[2]])
    with pytest.raises(gkv.GkvError):
        pool.trim(b, 49)   # it does not hold so many
    # no block left for the copy: nothing happens
    c = pool.seq_alloc()
    assert pool.reserve(c, 32) == 0 and pool.free_blocks() == 0
    pool.trim(b, 16)
    assert pool.free_blocks() == 1
    assert pool.reserve(c, 48) == 0
    with pytest.raises(gkv.GkvError) as e:
        pool.trim(b, 7)
    assert e.value.status == gkv.GKV_ERR_CAPACITY and len(pool.seq_blocks(b)) == 1
    pool.trim(a, 0)
    assert pool.free_blocks() == 3 and len(pool.seq_blocks(a)) == 0
    pool.close()


@pytest.mark.parametrize("n_blocks,fmt", [(40, BLOCK), (40, BF16), (900, BLOCK)])
def test_compact_moves_what_lies_behind(gkv, cuda, n_blocks, fmt):
    per = n_blocks // 10
    pool = gkv.Pool(n_layers=3, n_kv_heads=3, max_seqs=10, max_seq_len=16 * per + 32, window=0, num_blocks=n_blocks,
                    shuffle_seed=11, v_format=fmt)
    s = [pool.seq_alloc() for _ in range(8)]
    for x in s:
        assert pool.reserve(x, 16 * per) == 0
    data = [fill(gkv, pool.view(l), fmt, l) for l in range(3)]
    f = pool.fork(s[7], 16 * (per - 1))
    for x in s[:5]:
        assert pool.free(x) == 0
    was = {x: list(pool.seq_blocks(x)) for x in s[5:] + [f]}
    live = len({b for r in was.values() for b in r})
    assert pool.compact() == live == n_blocks - pool.free_blocks()
    pool.sync()
    t = dev_table(torch, gkv, pool.view(0), 10)
    now = {x: list(pool.seq_blocks(x)) for x in was}
    assert sorted({b for r in now.values() for b in r}) == list(range(live))
    for l in range(3):
        for x, y in zip(data[l], content(gkv, pool.view(l), fmt)):
            for q in was:
                assert np.array_equal(y[now[q]], x[was[q]])
    for q in was:
        assert list(t[q, :len(now[q])]) == now[q]
    assert list(now[f]) == list(now[s[7]][:per - 1])  # still shared
    assert pool.compact() == live                     # nothing left to move
    n = pool.seq_alloc()
    assert pool.reserve(n, 16) == 0 and list(pool.seq_blocks(n)) == [live]
    pool.close()


class Serving:
    """A pool with a window layer (kept first block) and a full layer, driven step by step."""

    Hq, Hkv, S = 8, 2, 4

    def __init__(self, gkv, fmt):
        self.gkv, self.fmt = gkv, fmt
        self.pool = gkv.Pool(n_layers=2, n_kv_heads=self.Hkv, max_seqs=self.S, max_seq_len=256, window=32,
                             num_blocks=40, shuffle_seed=7, v_format=fmt, kept=16)
        self.lay = [Layout(16, 32, True), Layout(0, 0, False)]
        self.rng = np.random.default_rng(fmt)
        self.cos, self.sin = O.rope_table(256)
        self.dcos, self.dsin = dev(self.cos), dev(self.sin)
        self.lens = [0] * self.S
        # the true K (rotated) and V of every position, per layer and sequence
        self.kv = [[[np.zeros((0, self.Hkv, D))] * 2 for _ in range(self.S)] for _ in range(2)]
        self.sinks = self.rng.standard_normal(self.Hq).astype(np.float32)
        self.err = torch.zeros(1, dtype=torch.int32, device="cuda")

    def held(self, layer, b):
        """K and V of sequence b as the device cache holds them, through the device table; NaN
        where the layer's table row does not hold a position."""
        view, lay = self.pool.view(layer), self.lay[layer]
        table = dev_table(torch, self.gkv, view, self.S)
        raw = content(self.gkv, view, self.fmt)
        out = []
        for i in range(2):
            x = raw[i].reshape(view.num_blocks, self.Hkv, -1)
            x = x.view(np.uint16) if self.fmt == BF16 else x
            res = np.full((self.lens[b], self.Hkv, D), np.nan)
            nb = -(-self.lens[b] // BT)
            for j in range(nb):
                if lay.ring and lay.entry(j) in [lay.entry(q) for q in range(j + 1, nb)]:
                    continue
                blk = table[b, lay.entry(j)]
                n = min(self.lens[b] - j * BT, BT)
                cells = x[blk][:, PLACES[self.fmt][i][:n]].transpose(1, 0, 2)
                if self.fmt == BF16:
                    cells = O.from_bf16(np.ascontiguousarray(cells)).astype(np.float64)
                else:
                    sc = raw[2].reshape(view.num_blocks, self.Hkv, 8).view(np.float32)[blk, :, i]
                    cells = e4m3_values(cells).astype(np.float64) * sc[None, :, None]
                res[j * BT:j * BT + n] = cells
            out.append(res)
        return out

    def check_cache(self, layer):
        for b in range(self.S):
            held = self.held(layer, b) if self.lens[b] else [np.zeros((0, self.Hkv, D))] * 2
            for true, got in zip(self.kv[layer][b], held):
                ok = ~np.isnan(got)
                seen = self.lay[layer].sees(self.lens[b] - 1, np.arange(self.lens[b]))
                assert ok[seen].all()
                err = np.abs(got - true)[ok]
                if self.fmt == BF16:
                    assert (err <= np.abs(true[ok]) * 2.0 ** -8).all()
                else:  # half a step, twice (a code that was moved), of the value or the subnormals
                    s_max = 2 * np.abs(true).max(initial=0) / 448
                    assert (err <= 2 * np.maximum(np.abs(true[ok]) * 2.0 ** -4, 2.0 ** -10 * s_max)).all()

    def rows(self, lens_new, layer):
        """qkv rows of the sequences' new positions; remembers their K and V."""
        pos = np.concatenate([np.arange(a, a + n) for a, n in zip(self.lens, lens_new)]).astype(np.int32)
        qkv = self.rng.standard_normal((len(pos), (self.Hq + 2 * self.Hkv) * D)).astype(np.float32)
        q, k, kb, vb = O.kv_append(qkv, self.Hq, self.Hkv, self.cos, self.sin, pos)
        k, v = np.asarray(k).reshape(-1, self.Hkv, D), qkv[:, (self.Hq + self.Hkv) * D:].reshape(-1, self.Hkv, D)
        o = 0
        for b, n in enumerate(lens_new):
            self.kv[layer][b] = [np.concatenate([x, y[o:o + n]]) for x, y in zip(self.kv[layer][b], (k, v))]
            o += n
        return qkv, q.reshape(-1, self.Hq, D), kb, vb

    def prompts(self, lens_new):
        """Chunks of whole blocks behind what is cached: attention, then the append."""
        assert all(x % BT == 0 for x, n in zip(self.lens, lens_new) if n)
        for b, n in enumerate(lens_new):
            assert self.pool.reserve(b, self.lens[b] + n) == 0 if n else True
        self.pool.sync()
        cu = np.concatenate([[0], np.cumsum(lens_new)]).astype(np.int32)
        after = [a + n for a, n in zip(self.lens, lens_new)]
        for layer, lay in enumerate(self.lay):
            held = [self.held(layer, b) if self.lens[b] else [np.zeros((0, self.Hkv, D))] * 2
                    for b in range(self.S)]
            qkv, q, kb, vb = self.rows(lens_new, layer)
            x, view = dev(qkv), self.pool.view(layer)
            kp, vp = (torch.empty(len(qkv), self.Hkv, D, dtype=torch.int16, device="cuda") for _ in "kv")
            none = self.gkv.CacheView(n_kv_heads=self.Hkv)
            self.gkv.kept_append(x, self.Hq, self.dcos, self.dsin, dev(np.array(after, np.int32)), none,
                                 cu_seqlens=dev(cu), max_rows=max(lens_new), k_pack=kp, v_pack=vp)
            assert np.array_equal(kp.cpu().numpy().view(np.uint16).reshape(kb.shape), kb)
            out = torch.empty(len(qkv), self.Hq * D, device="cuda")
            self.gkv.kept_prefill(dev(cu), max(lens_new), x, self.Hq, view, out,
                                  start_pos=dev(np.array(self.lens, np.int32)), k=kp, v=vp,
                                  sinks=dev(self.sinks), kept=lay.kept, window=lay.window, cos_tab=self.dcos,
                                  sin_tab=self.dsin, dev_err=self.err)
            self.gkv.kept_append(x, self.Hq, self.dcos, self.dsin, dev(np.array(after, np.int32)), view,
                                 kept=lay.kept, window=lay.window, cu_seqlens=dev(cu), max_rows=max(lens_new),
                                 dev_err=self.err)
            got = out.cpu().numpy().reshape(-1, self.Hq, D).astype(np.float64)
            kf, vf = (O.from_bf16(z).astype(np.float64).reshape(-1, self.Hkv, D) for z in (kb, vb))
            for b in range(self.S):
                r = slice(cu[b], cu[b + 1])
                if lens_new[b] == 0:
                    continue
                k, v = (np.concatenate([h, z[r]]) for h, z in zip(held[b], (kf, vf)))
                ok = np.stack([lay.sees(p, np.arange(len(k))) for p in range(self.lens[b], after[b])])
                want, pav, qk = attend(q[r].astype(np.float64), k, v, ok, self.sinks)
                bound = prefill_bound(want, pav, qk, len(k), np.nanmax(np.abs(v)), False)
                assert (np.abs(got[r] - want) <= bound).all()
        self.lens = after
        for layer in range(2):
            self.check_cache(layer)
        assert int(self.err.item()) == 0

    def step(self, active):
        """One decode step of the sequences in `active`; the others idle at length 0."""
        for b in active:
            assert self.pool.reserve(b, self.lens[b] + 1) == 0
        self.pool.sync()
        new = [1 if b in active else 0 for b in range(self.S)]
        now = dev(np.array([self.lens[b] + 1 if b in active else 0 for b in range(self.S)], np.int32))
        after = [a + n for a, n in zip(self.lens, new)]
        outs = []
        for layer, lay in enumerate(self.lay):
            qkv, q, _, _ = self.rows(new, layer)
            full = np.zeros((self.S, qkv.shape[1]), np.float32)
            full[active] = qkv
            x, view = dev(full), self.pool.view(layer)
            self.gkv.kept_append(x, self.Hq, self.dcos, self.dsin, now, view, kept=lay.kept, window=lay.window,
                                 dev_err=self.err)
            n = self.gkv.kept_workspace_bytes(self.S, self.Hkv, 256, lay.kept, lay.window)
            ws = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")
            out = torch.full((self.S, self.Hq * D), 3.0, device="cuda")
            self.gkv.kept_decode(x, self.Hq, now, 256, view, out, sinks=dev(self.sinks), kept=lay.kept,
                                 window=lay.window, cos_tab=self.dcos, sin_tab=self.dsin, workspace=ws,
                                 dev_err=self.err)
            outs.append((q, out.cpu().numpy().reshape(self.S, self.Hq, D)))
        self.lens = after
        for layer, lay in enumerate(self.lay):
            self.check_cache(layer)
            q, got = outs[layer]
            for i, b in enumerate(active):
                k, v = self.held(layer, b)
                ok = lay.sees(self.lens[b] - 1, np.arange(self.lens[b]))[None]
                want, pav, qk = attend(q[i:i + 1].astype(np.float64), k, v, ok, self.sinks)
                assert (np.abs(got[b] - want[0]) <= decode_bound(want, pav, qk, self.fmt, False)[0]).all()
            idle = [b for b in range(self.S) if b not in active]
            assert (got[idle] == 0).all()
        assert int(self.err.item()) == 0

    def fork(self, a):
        c = self.pool.fork(a, self.lens[a])
        self.lens[c] = self.lens[a]
        for layer in range(2):
            self.kv[layer][c] = list(self.kv[layer][a])
        return c

    def trim(self, b, n):
        self.pool.trim(b, n)
        self.lens[b] = n
        for layer in range(2):
            self.kv[layer][b] = [x[:n] for x in self.kv[layer][b]]

    def free(self, b):
        assert self.pool.free(b) == 0
        self.lens[b] = 0
        for layer in range(2):
            self.kv[layer][b] = [np.zeros((0, self.Hkv, D))] * 2


@pytest.mark.parametrize("fmt", [BF16, BLOCK])
def test_a_serving_run(gkv, cuda, fmt):
    s = Serving(gkv, fmt)
    a, b = s.pool.seq_alloc(), s.pool.seq_alloc()
    s.prompts([80, 21, 0, 0] if (a, b) == (0, 1) else None)
    s.prompts([37, 0, 0, 0])              # a second chunk behind 80 tokens
    for _ in range(3):
        s.step([a, b])
    c = s.fork(a)                          # at 120 tokens: inside a block
    for _ in range(10):
        s.step([a, b, c])                  # the two go their own ways
    s.trim(c, s.lens[c] - 2)               # (128: a block's border)
    s.step([a, c])
    d = s.fork(c)
    s.free(b)
    s.pool.compact()
    for _ in range(3):
        s.step([a, c, d])
    s.free(a)
    for _ in range(18):                    # a window's ring goes round
        s.step([c, d])
    s.pool.close()


@pytest.mark.parametrize("fmt", [BF16, BLOCK])
@pytest.mark.parametrize("lay", [Layout(16, 32, True), Layout(0, 0, False)])
def test_a_captured_step_replays(gkv, cuda, fmt, lay):
    """Append and decode captured once; replayed with other rows and lengths in the same buffers,
    eager work between the replays; each equals the eager call's result bit for bit."""
    from keptcase import Cache
    lens = np.array([37, 5, 0, 290], np.int32)
    cases = [Cache(lens, 2, lay, fmt, seed=5) for _ in range(2)]
    views = [c.device(gkv) for c in cases]
    cos, sin = (dev(x) for x in O.rope_table(400))
    n = max(16, gkv.kept_workspace_bytes(4, 2, 400, lay.kept, lay.window))
    wss = [torch.zeros(n, dtype=torch.uint8, device="cuda") for _ in range(2)]
    outs = [torch.zeros(4, 4 * D, device="cuda") for _ in range(2)]
    x, now = torch.zeros(4, 8 * D, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")

    def step(i):
        gkv.kept_append(x, 4, cos, sin, now, views[i], kept=lay.kept, window=lay.window, dev_err=cases[i].err)
        gkv.kept_decode(x, 4, now, 400, views[i], outs[i], kept=lay.kept, window=lay.window, cos_tab=cos,
                        sin_tab=sin, workspace=wss[i], dev_err=cases[i].err)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        step(0)  # (lengths 0: nothing happens)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s):
        step(0)
    g = torch.Generator(device="cuda").manual_seed(2)
    for r in range(4):
        x.copy_(torch.randn(4, 8 * D, generator=g, device="cuda"))
        # (the third sequence has a token every second step: idle, 1, idle, 2)
        now.copy_(dev(np.where([True, True, False, True], lens + 1 + r, (r + 1) // 2 * (r % 2)).astype(np.int32)))
        graph.replay()
        step(1)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[1]) and torch.isfinite(outs[0]).all()
        for p, q in zip(cases[0].pulled(), cases[1].pulled()):
            assert p is None or np.array_equal(p.view(np.uint8), q.view(np.uint8))
        (x * 2).sum().item()
    assert int(cases[0].err.item()) == int(cases[1].err.item()) == 0
