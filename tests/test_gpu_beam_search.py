"""A whole beam search on the GPU: tables taken from the prompts' lengths, appends, attention over
shared blocks, the choice, rows that follow it, copies of shared last blocks. Every call is checked
on what the one before it left, and a captured step against the eager one."""
import numpy as np
import pytest
import torch

from keptcase import BF16, BLOCK, BT, PLACES, attend, e4m3_values
from oracle import kv_oracle as O
from sharedcase import D, Model, dev, shared_bound, within
from test_gpu_beam import expect

pytestmark = pytest.mark.gpu
HQ, HKV, V = 16, 2, 300
EOS = 7


class Search:
    def __init__(self, gkv, prompts, K, fmt, n_layers=2, cap=160, seed=0):
        self.gkv, self.K, self.R, self.fmt = gkv, K, len(prompts), fmt
        S = self.S = K * len(prompts)
        g = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda *n: torch.randn(n, generator=g, device="cuda")  # noqa: E731
        self.emb, self.w, self.sinks = r(V, (HQ + 2 * HKV) * D), r(HQ * D, V) * 0.4, r(HQ)
        cos, sin = O.rope_table(cap)
        self.hcos, self.hsin = cos, sin
        self.cos, self.sin = dev(cos), dev(sin)
        stride, nb = cap // BT, S * (cap // BT) // 2 + 8
        i32 = lambda *n: torch.zeros(n, dtype=torch.int32, device="cuda")  # noqa: E731
        self.table, self.lens, self.refs = i32(S, stride), i32(S), i32(nb)
        self.t = gkv.block_tables(self.table, self.lens, self.refs)
        gkv.tables_init(self.t)
        dt = torch.int16 if fmt == BF16 else torch.uint8
        bad = 0x7FC0 if fmt == BF16 else 0x7F
        pool = lambda: torch.full((nb, HKV, BT * D), bad, dtype=dt, device="cuda")  # noqa: E731
        self.layers = [(pool(), pool(), torch.full((nb, HKV, 2), float("nan"), device="cuda") if fmt == BLOCK else None)
                       for _ in range(n_layers)]
        self.views = [gkv.cache_view(k, v, self.table, HKV, v_scale=sc, v_format=fmt) for k, v, sc in self.layers]
        self.array = gkv.cache_views(self.views)
        self.src, self.dst, self.cu = i32(S), i32(S), i32(S + 1)
        self.err = i32(1)
        self.ws_t = torch.empty(gkv.tables_workspace_bytes(S, nb), dtype=torch.uint8, device="cuda")
        self.ws_b = torch.empty(gkv.beam_workspace_bytes(self.R, K, V, K), dtype=torch.uint8, device="cuda")
        self.ws_a = torch.empty(gkv.shared_workspace_bytes(S, self.R, HQ, HKV, stride, cap), dtype=torch.uint8,
                                device="cuda")
        self.groups = dev(np.arange(self.R + 1, dtype=np.int32) * K)
        self.shared = i32(self.R)
        self.cum = torch.full((S,), -np.inf, device="cuda")
        self.cum[::K] = 0
        self.done = i32(S)
        self.scores, self.parents, self.tokens = torch.zeros(self.R, K, device="cuda"), i32(self.R, K), i32(self.R, K)
        self.row_seq = i32(S)
        self.out = [torch.zeros(S, HQ * D, device="cuda") for _ in range(n_layers)]
        # the prompts, into each request's first row; the other rows become forks of it
        lens = np.zeros(S, np.int32)
        lens[::K] = [len(p) for p in prompts]
        rows = int(lens.sum())
        seq, pos, slot = i32(rows), i32(rows), torch.zeros(rows, dtype=torch.int64, device="cuda")
        gkv.tables_resize(self.t, dev(lens), cu_rows=self.cu, row_seq=seq, row_pos=pos, row_slot=slot,
                          workspace=self.ws_t, dev_err=self.err)
        self.maps = seq, pos, slot
        x = self.emb[dev(np.concatenate(prompts)).long()]
        for view in self.views:
            gkv.kept_append(x, HQ, self.cos, self.sin, self.lens, view, cu_seqlens=self.cu, max_rows=max(map(len, prompts)),
                            dev_err=self.err)
        self.q = torch.zeros(S, (HQ + 2 * HKV) * D, device="cuda")
        self.q[:] = self.emb[dev(np.repeat([p[-1] for p in prompts], K)).long()]
        gkv.tables_reorder(self.t, dev(np.arange(S, dtype=np.int32) // K * K), K, shared_blocks=self.shared,
                           dev_err=self.err)

    def step(self, watch=lambda *a: None):
        gkv, cap = self.gkv, self.cos.shape[0]
        for view, out in zip(self.views, self.out):
            gkv.shared_decode(self.q, HQ, self.groups, self.shared, self.lens, cap, view, out, 8, cap, sinks=self.sinks,
                              cos_tab=self.cos, sin_tab=self.sin, workspace=self.ws_a, dev_err=self.err)
        watch("attend", self)
        logits = sum(self.out[1:], self.out[0]) @ self.w
        watch("logits", logits)
        done = self.done.clone()
        gkv.beam_select(logits, self.cum.clone(), self.K, self.scores, self.parents, self.tokens, done=done, eos=EOS,
                        done_out=self.done.view(self.R, self.K), workspace=self.ws_b, dev_err=self.err)
        self.cum.copy_(self.scores.view(-1))
        watch("select", self)
        gkv.tables_reorder(self.t, self.parents, self.K, shared_blocks=self.shared, dev_err=self.err)
        watch("reorder", self)
        new = self.lens + (1 - self.done)
        gkv.tables_resize(self.t, new, self.src, self.dst, cu_rows=self.cu, row_seq=self.row_seq, workspace=self.ws_t,
                          dev_err=self.err)
        gkv.copy_blocks(self.array, self.src, self.dst, dev_err=self.err)
        watch("resize", new)
        token = self.tokens.view(-1).long()
        self.q.copy_(self.emb[token])
        x = self.emb[token[self.row_seq.long()]]
        for view in self.views:
            gkv.kept_append(x, HQ, self.cos, self.sin, self.lens, view, cu_seqlens=self.cu, max_rows=1, dev_err=self.err)


def history(s, layer, b):
    """K and V of sequence b as the cache holds them, in 64 bits."""
    k, v, sc = (None if x is None else x.cpu().numpy() for x in s.layers[layer])
    L, row = int(s.lens[b]), s.table[b].cpu().numpy()
    out = []
    for i, pool in enumerate((k, v)):
        x = pool[row[:-(-L // BT)]][:, :, PLACES[s.fmt][i]]     # [blocks, H, 16, 64]
        if s.fmt == BF16:
            x = O.from_bf16(x.view(np.uint16)).astype(np.float64)
        else:
            x = e4m3_values(x).astype(np.float64) * sc[row[:-(-L // BT)], :, i][..., None, None]
        out.append(x.transpose(0, 2, 1, 3).reshape(-1, HKV, D)[:L])
    return out


def prompts(seed, lens):
    rng = np.random.default_rng(seed)
    return [rng.integers(8, V, n).astype(np.int32) for n in lens]


@pytest.mark.parametrize("fmt", [BF16, BLOCK])
@pytest.mark.parametrize("lens,K", [([37, 5, 64], 4), ([16], 8), ([100, 33], 1)])
def test_every_step(gkv, cuda, fmt, lens, K):
    p = prompts(1, lens)
    s = Search(gkv, p, K, fmt)
    m = Model(s.S, s.table.shape[1], s.refs.numel())
    first = np.zeros(s.S, np.int32)
    first[::K] = lens
    _, _, _, _, seq, pos, slot, _ = m.resize(first)
    assert [t.tolist() for t in s.maps] == [seq, pos, slot]
    m.reorder(np.arange(s.S) // K * K, K)
    text = [list(p[b // K]) for b in range(s.S)]   # every row's tokens
    emb = s.emb.cpu().numpy()
    was = {}

    def watch(what, x):
        if what == "attend":
            was.update(cum=s.cum.cpu().numpy(), done=s.done.cpu().numpy(), lens=s.lens.cpu().numpy())
            q = s.q.cpu().numpy()
            rot = O.kv_append(q, HQ, HKV, s.hcos, s.hsin, (was["lens"] - 1).astype(np.int32))[0].reshape(s.S, HQ, D)
            for b in range(s.S):
                for layer in range(len(s.layers)):
                    k, v = history(s, layer, b)
                    if fmt == BF16 and layer == 0:
                        # the row's own tokens, in order, nothing of another beam's
                        at = np.arange(len(text[b]), dtype=np.int32)
                        _, _, kb, vb = O.kv_append(emb[text[b]], HQ, HKV, s.hcos, s.hsin, at)
                        assert np.array_equal(O.from_bf16(kb.reshape(-1, HKV, D)), k)
                        assert np.array_equal(O.from_bf16(vb.reshape(-1, HKV, D)), v)
                    one = rot[b:b + 1].astype(np.float64)
                    out, pav, qk = attend(one, k, v, np.ones((1, len(k)), bool), s.sinks.cpu().numpy())
                    qm = np.abs(one).max(-1)[..., None] * np.repeat(np.abs(k).sum(-1).max(0), HQ // HKV)[None, :, None] / 8
                    within(s.out[layer][b:b + 1].cpu().numpy().reshape(1, HQ, D), out,
                           shared_bound(out, pav, qk, qm, fmt, False), f"row {b}")
        elif what == "logits":
            was["logits"] = x.cpu().numpy()
        elif what == "select":
            sc, par, tok, ended = expect(was["logits"], was["cum"], K, K, was["done"], EOS)
            assert np.array_equal(s.parents.cpu().numpy(), par) and np.array_equal(s.tokens.cpu().numpy(), tok)
            assert np.array_equal(s.done.cpu().numpy(), ended.reshape(-1))
            fin = np.isfinite(sc)
            assert (np.abs(s.scores.cpu().numpy()[fin] - sc[fin]) <= 2.0 ** -12 + np.abs(sc[fin]) * 2.0 ** -24).all()
        elif what == "reorder":
            shared, _ = m.reorder(s.parents.cpu().numpy().reshape(-1), K)
            assert np.array_equal(s.shared.cpu().numpy(), shared)
            par = s.parents.view(-1).tolist()
            text[:] = [list(text[i]) for i in par]
        else:
            new = x.cpu().numpy()
            ok, src, dst, cu, seq, *_ = m.resize(new)
            assert ok and s.src.tolist() == src.tolist() and s.dst.tolist() == dst.tolist() and s.cu.tolist() == cu.tolist()
            assert s.row_seq[:len(seq)].tolist() == seq
            for b, t in enumerate(s.tokens.view(-1).tolist()):
                if cu[b + 1] > cu[b]:
                    text[b].append(t)
            assert np.array_equal(s.table.cpu().numpy(), m.table) and np.array_equal(s.refs.cpu().numpy(), m.refs)

    for _ in range(22):
        s.step(watch)
    assert int(s.err.item()) == 0
    # a request leaves: its blocks are free again
    new = s.lens.clone()
    new[:K] = 0
    gkv.tables_resize(s.t, new, s.src, s.dst, workspace=s.ws_t, dev_err=s.err)
    m.resize(new.cpu().numpy())
    assert np.array_equal(s.refs.cpu().numpy(), m.refs)


@pytest.mark.parametrize("fmt", [BF16, BLOCK])
def test_a_captured_step(gkv, cuda, fmt):
    """The whole step in a graph, replayed, against the same steps called one by one."""
    p = prompts(2, [50, 20, 31])
    a, b = Search(gkv, p, 4, fmt, seed=3), Search(gkv, p, 4, fmt, seed=3)
    for s in (a, b):
        s.step()  # (the product's library starts up outside the capture)
    torch.cuda.synchronize()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        b.step()
    for _ in range(25):
        a.step()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in ((a.tokens, b.tokens), (a.parents, b.parents), (a.table, b.table), (a.refs, b.refs), (a.lens, b.lens),
                     (a.scores, b.scores), (a.out[0], b.out[0]), (a.shared, b.shared)):
            assert torch.equal(x, y)
    assert int(a.err.item()) == 0 and int(b.err.item()) == 0
