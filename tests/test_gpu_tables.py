"""gkv_tables_* on the GPU against a plain model (tests/sharedcase.py): every entry, length, holder,
copy and row."""
import numpy as np
import pytest
import torch

from sharedcase import BT, Model, dev

pytestmark = pytest.mark.gpu


class Tables:
    def __init__(self, gkv, n_seqs, stride, blocks, rows=4096):
        i32 = lambda *n: torch.full(n, 77, dtype=torch.int32, device="cuda")  # noqa: E731
        self.gkv, self.n = gkv, n_seqs
        self.table, self.lens, self.refs = i32(n_seqs, stride), i32(n_seqs), i32(blocks)
        self.t = gkv.block_tables(self.table, self.lens, self.refs)
        self.src, self.dst, self.cu = i32(n_seqs), i32(n_seqs), i32(n_seqs + 1)
        self.seq, self.pos = i32(rows), i32(rows)
        self.slot = torch.full((rows,), 77, dtype=torch.int64, device="cuda")
        self.err = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.ws = torch.full((gkv.tables_workspace_bytes(n_seqs, blocks),), 0xEE, dtype=torch.uint8, device="cuda")
        gkv.tables_init(self.t)
        self.m = Model(n_seqs, stride, blocks)

    def resize(self, new, stream=None):
        self.gkv.tables_resize(self.t, new if torch.is_tensor(new) else dev(np.asarray(new, np.int32)), self.src,
                               self.dst, cu_rows=self.cu, row_seq=self.seq, row_pos=self.pos, row_slot=self.slot,
                               workspace=self.ws, dev_err=self.err, stream=stream)

    def same_state(self):
        assert np.array_equal(self.lens.cpu().numpy(), self.m.lens)
        assert np.array_equal(self.table.cpu().numpy(), self.m.table)
        assert np.array_equal(self.refs.cpu().numpy(), self.m.refs)

    def check_resize(self, new):
        keep = [x.clone() for x in (self.seq, self.pos, self.slot)]
        self.resize(new)
        ok, src, dst, cu, seq, pos, slot, flags = self.m.resize(new, self.seq.numel())
        self.same_state()
        assert np.array_equal(self.src.cpu().numpy(), src) and np.array_equal(self.dst.cpu().numpy(), dst)
        assert np.array_equal(self.cu.cpu().numpy(), cu)
        for got, was, want in zip((self.seq, self.pos, self.slot), keep, (seq, pos, slot)):
            assert got[:len(want)].tolist() == list(want)
            assert torch.equal(got[len(want):], was[len(want):])  # rows behind the last: as they were
        assert int(self.err.item()) == flags
        self.err.zero_()
        return ok

    def check_reorder(self, parents, per):
        shared = torch.full((self.n // per,), 77, dtype=torch.int32, device="cuda")
        self.gkv.tables_reorder(self.t, dev(np.asarray(parents, np.int32)), per, shared_blocks=shared, dev_err=self.err)
        want, flags = self.m.reorder(parents, per)
        self.same_state()
        assert np.array_equal(shared.cpu().numpy(), want)
        assert int(self.err.item()) == flags
        self.err.zero_()


def test_init(gkv, cuda):
    Tables(gkv, 5, 7, 33).same_state()


def test_one_token_at_a_time(gkv, cuda):
    t = Tables(gkv, 3, 4, 9)
    for n in range(1, 40):
        assert t.check_resize([n, n // 2, 0])
    assert t.check_resize([0, 0, 64])


def test_shared_last_blocks_are_replaced(gkv, cuda):
    t = Tables(gkv, 8, 6, 64)
    assert t.check_resize([20, 0, 0, 0, 32, 0, 0, 0])
    t.check_reorder([0, 0, 0, 0, 4, 4, 4, -1], 4)
    assert int(t.refs.max()) == 4
    assert t.check_resize([21, 23, 20, 40, 33, 33, 32, 1])  # 2 stays at 20 and keeps the block
    assert t.dst.count_nonzero() == 3
    t.check_reorder([1, 1, 2, 0, 5, 4, 6, 7], 4)
    assert t.check_resize([24, 24, 20, 22, 34, 34, 32, 0])
    assert t.check_resize([0] * 8)
    assert int(t.refs.sum()) == 0


def test_a_block_is_given_back_with_its_last_holder(gkv, cuda):
    t = Tables(gkv, 2, 8, 16)
    t.check_resize([100, 0])
    t.check_reorder([0, 0], 2)
    t.check_resize([0, 100])
    t.check_resize([0, 17])
    t.check_resize([50, 17])
    t.check_resize([0, 0])


def test_what_is_given_back_is_free_from_the_next_call_on(gkv, cuda):
    t = Tables(gkv, 2, 8, 8)
    assert t.check_resize([128, 0])
    assert not t.check_resize([0, 16])
    assert t.check_resize([0, 0])
    assert t.check_resize([0, 128])


def test_nothing_changes_without_room(gkv, cuda):
    t = Tables(gkv, 3, 10, 6, rows=90)
    assert t.check_resize([33, 0, 16])
    assert not t.check_resize([33, 48, 0])   # 3 blocks, 2 are free
    assert not t.check_resize([96, 16, 16])
    assert t.check_resize([33, 32, 16])
    assert t.check_resize([0, 0, 0])
    assert not t.check_resize([91, 0, 0])    # more rows than their arrays hold
    assert t.check_resize([90, 0, 0])


def test_lengths_that_a_row_cannot_have(gkv, cuda):
    t = Tables(gkv, 4, 3, 40)
    assert t.check_resize([48, 49, -1, 5])
    assert t.check_resize([2**31 - 1, 48, 7, -2**31])


def test_the_lengths_themselves(gkv, cuda):
    t = Tables(gkv, 2, 4, 8)
    t.check_resize([30, 5])
    t.resize(t.lens)
    t.same_state()
    assert t.cu.tolist() == [0, 0, 0]


def test_parents_outside_the_group(gkv, cuda):
    t = Tables(gkv, 6, 4, 30)
    t.check_resize([10, 20, 30, 40, 50, 60])
    t.check_reorder([1, 3, -2, 3, 2**31 - 1, 4], 3)


@pytest.mark.parametrize("per", [1, 2, 5, 64, 2048])
def test_group_sizes(gkv, cuda, per):
    rng = np.random.default_rng(per)
    S = max(2 * per, 6) // per * per
    t = Tables(gkv, S, 40, 30 * S + 8, rows=64 * S)
    t.check_resize(rng.integers(0, 64, S))
    for _ in range(3):
        t.check_reorder(np.arange(S) // per * per + rng.integers(0, per, S), per)
        t.check_resize(np.maximum(t.m.lens + rng.integers(0, 20, S), 0))


@pytest.mark.parametrize("seed", range(12))
def test_random_steps(gkv, cuda, seed):
    rng = np.random.default_rng(seed)
    per = int(rng.choice([1, 3, 8, 16]))
    S = per * int(rng.integers(1, 9))
    stride = int(rng.integers(2, 70))
    blocks = int(S * stride * rng.uniform(0.3, 1.2)) + 1
    t = Tables(gkv, S, stride, blocks, rows=S * 200)
    for _ in range(12):
        if rng.random() < 0.4:
            p = np.arange(S) // per * per + rng.integers(0, per, S)
            p[rng.random(S) < 0.1] = -1
            t.check_reorder(p, per)
        else:
            new = t.m.lens.astype(np.int64) + rng.integers(-20, 30, S)
            new[rng.random(S) < 0.1] = 0
            new[rng.random(S) < 0.1] = rng.integers(0, stride * BT + 1)
            t.check_resize(np.clip(new, 0, stride * BT))


def test_many_sequences_and_blocks(gkv, cuda):
    rng = np.random.default_rng(0)
    S, blocks = 5000, 60001
    t = Tables(gkv, S, 32, blocks, rows=S * 300)
    t.check_resize(rng.integers(0, 200, S))
    t.check_resize(rng.integers(0, 150, S))
    t.check_reorder(np.arange(S) // 50 * 50 + rng.integers(0, 50, S), 50)
    t.check_resize(t.m.lens + 1)


def test_long_rows(gkv, cuda):
    t = Tables(gkv, 4, 20000, 50000, rows=300000)
    t.check_resize([250000, 7, 0, 16])
    t.check_reorder([0, 0, 1, 1], 2)
    t.check_reorder([0, 0, 3, 2], 4)
    t.check_resize([250001, 250016, 250017, 0])
    t.check_reorder([1, 0, 3, 2], 4)


def test_no_sequences(gkv, cuda):
    t = gkv.BlockTables(0x1000, 0x1000, 0x1000, 4, 0, 8)
    err, cu = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.full((1,), 7, dtype=torch.int32, device="cuda")
    ws = torch.empty(gkv.tables_workspace_bytes(0, 8), dtype=torch.uint8, device="cuda")
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    refs = torch.zeros(8, dtype=torch.int32, device="cuda")
    t.refs = refs.data_ptr()
    st = gkv.lib().gkv_tables_resize(gkv.stream_handle(), t, refs.data_ptr(), None, None, 0, cu.data_ptr(), None, None,
                                     None, ws.data_ptr(), ws.numel(), err.data_ptr())
    assert st == gkv.GKV_OK and cu.tolist() == [0] and int(err.item()) == 0
    assert gkv.lib().gkv_tables_reorder(gkv.stream_handle(), t, 4, refs.data_ptr(), None, None) == gkv.GKV_OK
    assert none.numel() == 0


def test_only_what_is_asked_for(gkv, cuda):
    t = Tables(gkv, 3, 4, 16)
    gkv.tables_resize(t.t, dev(np.array([5, 30, 0], np.int32)), workspace=t.ws, dev_err=t.err)
    t.m.resize([5, 30, 0])
    t.same_state()
    gkv.tables_resize(t.t, dev(np.array([6, 30, 3], np.int32)), row_pos=t.pos, workspace=t.ws, dev_err=t.err)
    t.m.resize([6, 30, 3])
    t.same_state()
    assert t.pos[:4].tolist() == [5, 0, 1, 2]
    gkv.tables_reorder(t.t, dev(np.array([1, 0, 2], np.int32)), 3, dev_err=t.err)
    t.m.reorder([1, 0, 2], 3)
    t.same_state()


def test_captured_steps_on_a_stream(gkv, cuda):
    """A reorder and a resize captured, replayed with other parents in the same buffer."""
    rng = np.random.default_rng(5)
    per, S = 4, 12
    t = Tables(gkv, S, 30, 600)
    t.check_resize(rng.integers(1, 60, S))
    parents = torch.zeros(S, dtype=torch.int32, device="cuda")
    shared = torch.zeros(S // per, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    new = torch.empty_like(t.lens)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        gkv.tables_reorder(t.t, parents, per, shared_blocks=shared, dev_err=t.err)
        torch.add(t.lens, 3, out=new)
        t.resize(new)
    for _ in range(6):
        p = np.arange(S) // per * per + rng.integers(0, per, S)
        parents.copy_(dev(p.astype(np.int32)))
        graph.replay()
        want, _ = t.m.reorder(p, per)
        ok, src, dst, cu, seq, pos, slot, _ = t.m.resize(t.m.lens + 3)
        assert ok and np.array_equal(shared.cpu().numpy(), want)
        t.same_state()
        assert t.slot[:len(slot)].tolist() == slot and t.dst.tolist() == dst.tolist()
    assert int(t.err.item()) == 0


def test_on_another_stream(gkv, cuda):
    t = Tables(gkv, 70, 8, 600)
    side = torch.cuda.Stream()
    new, parents = torch.zeros(70, dtype=torch.int32, device="cuda"), torch.zeros(70, dtype=torch.int32, device="cuda")
    a, b = np.arange(70, dtype=np.int32) + 5, np.arange(70, dtype=np.int32) // 10 * 10
    da, db = dev(a), dev(b)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(2000000)
        new.copy_(da)
        parents.copy_(db)
    t.resize(new, stream=side)
    gkv.tables_reorder(t.t, parents, 10, dev_err=t.err, stream=side)
    side.synchronize()
    t.m.resize(a)
    t.m.reorder(b, 10)
    t.same_state()


@pytest.mark.parametrize("S,rows", [(64, 4096), (64, 4097), (65, 4096), (1024, 30000), (1025, 30000)])
def test_both_sides_of_the_forms(gkv, cuda, S, rows):
    """One launch, two, and more sequences than threads."""
    rng = np.random.default_rng(S + rows)
    t = Tables(gkv, S, 12, S * 14, rows=rows)
    t.check_resize(rng.integers(0, 26, S))
    t.check_reorder(rng.integers(0, S, S), S)
    t.check_resize(np.minimum(t.m.lens + rng.integers(0, 4, S), 190))
    t.check_resize(rng.integers(0, 26, S))
