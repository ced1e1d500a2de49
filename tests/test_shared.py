"""The refusals of gkv_shared_decode, gkv_beam_select and gkv_tables_*, in the C interface and in the
Python binding, on the CPU: every check fails before anything is launched."""
from types import SimpleNamespace

import pytest
import torch

from test_kept import FAKE, view

NO_STREAM = SimpleNamespace(cuda_stream=None)


def shared(gkv, v=None, **o):
    a = dict(B=4, n=2, cu=FAKE, sh=FAKE, ms=8, mo=100, hq=64, q=FAKE, stride=80 * 64, cos=FAKE, sin=FAKE, lens=FAKE,
             max_len=100, sinks=None, ws=FAKE, ws_bytes=1 << 40, out=FAKE, out_stride=64 * 64, dtype=0)
    a.update(o)
    return gkv.lib().gkv_shared_decode(None, a["B"], a["n"], a["cu"], a["sh"], a["ms"], a["mo"], a["hq"], a["q"],
                                       a["stride"], a["cos"], a["sin"], a["lens"], a["max_len"], v or view(gkv),
                                       a["sinks"], a["ws"], a["ws_bytes"], a["out"], a["out_stride"], a["dtype"], None)


@pytest.mark.parametrize("cache,why", [
    (dict(v_format=1), "UNSUPPORTED"), (dict(v_format=2), "UNSUPPORTED"), (dict(v_format=4), "ARG"),
    (dict(v_scale=None), "ARG"), (dict(v_scale=FAKE + 4), "ARG"), (dict(k=FAKE + 8), "ARG"), (dict(v=None), "ARG"),
    (dict(block_table=None), "ARG"), (dict(table_stride=0), "ARG"), (dict(num_blocks=0), "ARG"),
    (dict(n_kv_heads=0), "ARG"), (dict(ring=16), "ARG"), (dict(ring=-16), "ARG")])
def test_shared_caches(gkv, cache, why):
    assert shared(gkv, view(gkv, **cache)) == getattr(gkv, "GKV_ERR_" + why)


@pytest.mark.parametrize("bad,why", [
    (dict(B=-1), "ARG"), (dict(n=-1), "ARG"), (dict(cu=None), "ARG"), (dict(sh=None), "ARG"), (dict(ms=-1), "ARG"),
    (dict(mo=-1), "ARG"), (dict(hq=0), "ARG"), (dict(hq=60), "ARG"), (dict(hq=72), "UNSUPPORTED"), (dict(q=None), "ARG"),
    (dict(q=FAKE + 4), "ARG"), (dict(stride=64 * 64 - 4), "ARG"), (dict(stride=64 * 64 + 2), "ARG"),
    (dict(cos=None), "ARG"), (dict(sin=FAKE + 8), "ARG"), (dict(lens=None), "ARG"), (dict(max_len=-1), "ARG"),
    (dict(out=None), "ARG"), (dict(out=FAKE + 8), "ARG"), (dict(out=FAKE + 4, dtype=1), "ARG"),
    (dict(out_stride=64 * 64 - 4), "ARG"), (dict(out_stride=64 * 64 + 2), "ARG"), (dict(dtype=2), "ARG"),
    (dict(cu=FAKE + 2), "ARG"), (dict(sh=FAKE + 1), "ARG"), (dict(ws=FAKE + 8), "ARG"), (dict(ws=None), "WORKSPACE"),
    (dict(ws_bytes=1000), "WORKSPACE"), (dict(B=2**31 - 1), "UNSUPPORTED"), (dict(n=2**31 - 1), "UNSUPPORTED")])
def test_shared_arguments(gkv, bad, why):
    assert shared(gkv, **bad) == getattr(gkv, "GKV_ERR_" + why)


def test_shared_heads_and_nothing(gkv):
    assert shared(gkv, view(gkv, n_kv_heads=9), hq=9) == gkv.GKV_ERR_UNSUPPORTED
    assert shared(gkv, B=0, ws=None) == gkv.GKV_OK
    assert gkv.shared_workspace_bytes(4, 1, 9, 9, 8, 100) == 0
    assert gkv.shared_workspace_bytes(4, 0, 64, 8, 0, 100) > 0
    assert gkv.shared_workspace_bytes(0, 1, 64, 8, 8, 100) == 0


def beam(gkv, **o):
    a = dict(R=2, K=4, V=1000, x=FAKE, stride=1000, dtype=0, cum=FAKE, done=None, eos=2, n=8, s=FAKE, p=FAKE, t=FAKE,
             d=None, ws=FAKE, ws_bytes=1 << 40)
    a.update(o)
    return gkv.lib().gkv_beam_select(None, a["R"], a["K"], a["V"], a["x"], a["stride"], a["dtype"], a["cum"], a["done"],
                                     a["eos"], a["n"], a["s"], a["p"], a["t"], a["d"], a["ws"], a["ws_bytes"], None)


@pytest.mark.parametrize("bad,why", [
    (dict(R=-1), "ARG"), (dict(K=0), "ARG"), (dict(V=0), "ARG"), (dict(n=0), "ARG"), (dict(n=1001), "ARG"),
    (dict(V=5, n=6), "ARG"), (dict(n=65), "UNSUPPORTED"), (dict(K=65), "UNSUPPORTED"), (dict(R=1 << 23), "UNSUPPORTED"), (dict(V=(1 << 30) + 1, stride=1 << 31), "UNSUPPORTED"),
    (dict(x=None), "ARG"), (dict(x=FAKE + 2), "ARG"), (dict(x=FAKE + 1, dtype=1), "ARG"), (dict(stride=999), "ARG"),
    (dict(dtype=2), "ARG"), (dict(cum=None), "ARG"), (dict(cum=FAKE + 2), "ARG"), (dict(done=FAKE, eos=-1), "ARG"),
    (dict(done=FAKE + 2), "ARG"), (dict(eos=1000), "ARG"), (dict(s=None), "ARG"), (dict(p=None), "ARG"),
    (dict(t=None), "ARG"), (dict(t=FAKE + 1), "ARG"), (dict(d=FAKE + 2), "ARG"), (dict(ws=None), "WORKSPACE"),
    (dict(ws_bytes=8), "WORKSPACE"), (dict(ws=FAKE + 8), "ARG")])
def test_beam_arguments(gkv, bad, why):
    assert beam(gkv, **bad) == getattr(gkv, "GKV_ERR_" + why)


def test_beam_nothing(gkv):
    assert beam(gkv, R=0) == gkv.GKV_OK
    assert gkv.beam_workspace_bytes(2, 65, 1000, 8) == 0
    # (room for all means room for fewer)
    most = [gkv.beam_workspace_bytes(r, 4, 5000, 8) for r in range(1, 400)]
    assert most == sorted(most)


def tables(gkv, **o):
    a = dict(table=FAKE, lens=FAKE, refs=FAKE, table_stride=4, n_seqs=8, num_blocks=16)
    a.update(o)
    return gkv.BlockTables(*a.values())


def resize(gkv, t=None, **o):
    a = dict(new=FAKE, src=None, dst=None, rows=8, cu=None, seq=FAKE, pos=FAKE, slot=FAKE, ws=FAKE, ws_bytes=1 << 40)
    a.update(o)
    return gkv.lib().gkv_tables_resize(None, t or tables(gkv), a["new"], a["src"], a["dst"], a["rows"], a["cu"], a["seq"],
                                       a["pos"], a["slot"], a["ws"], a["ws_bytes"], None)


def reorder(gkv, t=None, per=4, parents=FAKE, sh=None):
    return gkv.lib().gkv_tables_reorder(None, t or tables(gkv), per, parents, sh, None)


@pytest.mark.parametrize("bad,why", [
    (dict(table=None), "ARG"), (dict(lens=None), "ARG"), (dict(refs=None), "ARG"), (dict(table=FAKE + 2), "ARG"),
    (dict(refs=FAKE + 1), "ARG"), (dict(table_stride=0), "ARG"), (dict(n_seqs=-4), "ARG"), (dict(num_blocks=0), "ARG"),
    (dict(table_stride=(1 << 17) + 1), "UNSUPPORTED")])
def test_tables_that_are_none(gkv, bad, why):
    t = tables(gkv, **bad)
    want = getattr(gkv, "GKV_ERR_" + why)
    assert gkv.lib().gkv_tables_init(None, t) == want and resize(gkv, t) == want and reorder(gkv, t) == want


@pytest.mark.parametrize("bad,why", [
    (dict(new=None), "ARG"), (dict(src=FAKE), "ARG"), (dict(dst=FAKE), "ARG"), (dict(rows=-1), "ARG"),
    (dict(new=FAKE + 2), "ARG"), (dict(cu=FAKE + 2), "ARG"), (dict(seq=FAKE + 2), "ARG"), (dict(slot=FAKE + 4), "ARG"),
    (dict(ws=None), "WORKSPACE"), (dict(ws_bytes=100), "WORKSPACE"), (dict(ws=FAKE + 8), "ARG")])
def test_resize_arguments(gkv, bad, why):
    assert resize(gkv, **bad) == getattr(gkv, "GKV_ERR_" + why)


def test_reorder_arguments(gkv):
    for kw in (dict(per=0), dict(per=3), dict(per=-4), dict(parents=None), dict(parents=FAKE + 2), dict(sh=FAKE + 2)):
        assert reorder(gkv, **kw) == gkv.GKV_ERR_ARG
    assert reorder(gkv, tables(gkv, n_seqs=4096), per=4096) == gkv.GKV_ERR_UNSUPPORTED
    assert reorder(gkv, tables(gkv, n_seqs=0)) == gkv.GKV_OK
    assert gkv.tables_workspace_bytes(-1, 4) == 0 and gkv.tables_workspace_bytes(4, 0) == 0


# ---- the binding -----------------------------------------------------------------


def ints(*n):
    return torch.zeros(n, dtype=torch.int32)


def py_shared(gkv, **o):
    a = dict(q=torch.zeros(2, 128), cu_groups=ints(3), shared_blocks=ints(2), seq_lens=ints(2), out=torch.zeros(2, 128),
             sinks=torch.zeros(2), cos_tab=torch.zeros(8, 32), sin_tab=torch.zeros(8, 32))
    a.update(o)
    gkv.shared_decode(n_q_heads=2, max_seq_len=8, view=gkv.CacheView(n_kv_heads=1), max_shared_blocks=1, max_own=8,
                      stream=NO_STREAM, **a)


def py_beam(gkv, **o):
    a = dict(logits=torch.zeros(4, 10), cum_scores=torch.zeros(4), scores=torch.zeros(2, 3), parents=ints(2, 3),
             tokens=ints(2, 3), done=ints(4), done_out=ints(2, 3))
    a.update(o)
    gkv.beam_select(n_beams=2, eos=1, stream=NO_STREAM, **a)


def py_tables(gkv, **o):
    a = dict(table=ints(4, 3), lens=ints(4), refs=ints(9))
    a.update(o)
    gkv.block_tables(**a)


def py_resize(gkv, **o):
    a = dict(new_lens=ints(8), copy_src=ints(8), copy_dst=ints(8), cu_rows=ints(9), row_seq=ints(5), row_pos=ints(5),
             row_slot=torch.zeros(5, dtype=torch.int64))
    a.update(o)
    gkv.tables_resize(tables(gkv), stream=NO_STREAM, **a)


def py_reorder(gkv, **o):
    a = dict(parents=ints(8), shared_blocks=ints(2))
    a.update(o)
    gkv.tables_reorder(tables(gkv), group_size=4, stream=NO_STREAM, **a)


L4, HALF = torch.zeros(4, dtype=torch.int64), torch.float16
CASES = [(py_shared, dict(q=torch.zeros(2, 128, dtype=HALF))), (py_shared, dict(cu_groups=ints(2))),
         (py_shared, dict(cu_groups=L4[:3])), (py_shared, dict(shared_blocks=L4[:2])), (py_shared, dict(seq_lens=ints(3))),
         (py_shared, dict(out=torch.zeros(1, 128))), (py_shared, dict(out=torch.zeros(2, 128, dtype=HALF))),
         (py_shared, dict(sinks=torch.zeros(2, dtype=HALF))), (py_shared, dict(cos_tab=torch.zeros(8, 32, dtype=HALF))),
         (py_shared, dict(sinks=torch.zeros(1))), (py_shared, dict(sin_tab=torch.zeros(32, 8).t())),
         (py_shared, dict(q=torch.zeros(2, 64))), (py_shared, dict(out=torch.zeros(2, 64))),
         (py_shared, dict(workspace=torch.zeros(8, 2)[:, 0])),
         (py_beam, dict(logits=torch.zeros(4, 10, dtype=HALF))), (py_beam, dict(logits=torch.zeros(10, 4).t())),
         (py_beam, dict(logits=torch.zeros(3, 10))), (py_beam, dict(cum_scores=torch.zeros(3))),
         (py_beam, dict(cum_scores=torch.zeros(4, dtype=torch.float64))), (py_beam, dict(parents=ints(2, 2))),
         (py_beam, dict(tokens=torch.zeros(2, 3))), (py_beam, dict(done=torch.zeros(4, dtype=torch.bool))),
         (py_beam, dict(done_out=ints(6, 2)[:, 0])), (py_beam, dict(scores=torch.zeros(3, 2).t())),
         (py_tables, dict(table=ints(3, 4).t())), (py_tables, dict(lens=ints(3))), (py_tables, dict(refs=L4)),
         (py_tables, dict(table=ints(4, 4)[:, :3])),
         (py_resize, dict(new_lens=ints(7))), (py_resize, dict(copy_src=ints(7))), (py_resize, dict(copy_dst=L4)),
         (py_resize, dict(cu_rows=ints(8))), (py_resize, dict(row_pos=ints(4))), (py_resize, dict(row_slot=ints(5))),
         (py_reorder, dict(parents=ints(7))), (py_reorder, dict(shared_blocks=ints(3)))]


@pytest.mark.parametrize("call,bad", CASES)
def test_refused_tensors(gkv, monkeypatch, call, bad):
    monkeypatch.setattr(torch.Tensor, "is_pinned", lambda self: True)  # (host memory that the GPU can read)
    with pytest.raises(ValueError, match=next(iter(bad))):
        call(gkv, **bad)


@pytest.mark.parametrize("call", [py_shared, py_beam, py_tables, py_resize, py_reorder])
def test_host_memory_is_refused(gkv, call):
    with pytest.raises(ValueError, match="not in GPU memory"):
        call(gkv)


@pytest.mark.parametrize("call,what", [
    (py_shared, "q"), (py_shared, "out"), (py_shared, "cos_tab"), (py_shared, "sin_tab"), (py_shared, "sinks"),
    (py_beam, "logits"), (py_beam, "scores"), (py_resize, "row_slot"), (py_shared, "workspace"), (py_beam, "workspace"),
    (py_resize, "workspace")])
def test_any_tensor_in_host_memory_is_refused(gkv, monkeypatch, call, what):
    """All others are where the GPU reads."""
    far = {"sinks": torch.zeros(2), "logits": torch.zeros(4, 10), "scores": torch.zeros(2, 3),
           "row_slot": torch.zeros(5, dtype=torch.int64)}.get(what, torch.zeros(2, 128))
    monkeypatch.setattr(torch.Tensor, "is_pinned", lambda self: self is not far)
    with pytest.raises(ValueError, match=what + ": not in GPU memory"):
        call(gkv, **{what: far})
