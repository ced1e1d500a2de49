"""What the Python binding of the shared decode refuses beside tests/test_shared.py's cases, on the CPU."""
import pytest
import torch

from test_shared import NO_STREAM, ints


def decode(gkv, rows=(8, 8), max_seq_len=8, stride=4, made=lambda n: torch.zeros(n, 32)):
    cos, sin = (None if n is None else made(n) for n in rows)
    gkv.shared_decode(q=torch.zeros(2, 128), n_q_heads=2, cu_groups=ints(3), shared_blocks=ints(2), seq_lens=ints(2),
                      max_seq_len=max_seq_len, view=gkv.CacheView(n_kv_heads=1, table_stride=stride),
                      out=torch.zeros(2, 128), max_shared_blocks=1, max_own=8, cos_tab=cos, sin_tab=sin, stream=NO_STREAM)


@pytest.mark.parametrize("kw,what", [
    (dict(rows=(7, 8)), "cos_tab"), (dict(rows=(8, 7)), "sin_tab"), (dict(rows=(0, 8)), "cos_tab"),
    (dict(rows=(8, 0)), "sin_tab"), (dict(rows=(63, 64), max_seq_len=1000), "cos_tab"),
    (dict(rows=(64, 63), max_seq_len=1000), "sin_tab"), (dict(rows=(8, 8), made=lambda n: torch.zeros(n, 31)), "cos_tab")])
def test_tables_of_too_few_angles(gkv, monkeypatch, kw, what):
    """A sequence may be as long as max_seq_len, or a whole row of the block table."""
    monkeypatch.setattr(torch.Tensor, "is_pinned", lambda self: True)
    with pytest.raises(ValueError, match=what):
        decode(gkv, **kw)


@pytest.mark.parametrize("kw", [dict(), dict(rows=(None, None)), dict(rows=(9, 20)), dict(rows=(64, 64), max_seq_len=1000)])
def test_tables_of_enough_angles(gkv, monkeypatch, kw):
    """They pass on to the C interface, which refuses the view (it has no cache)."""
    monkeypatch.setattr(torch.Tensor, "is_pinned", lambda self: True)
    with pytest.raises(gkv.GkvError) as e:
        decode(gkv, **kw)
    assert e.value.status == gkv.GKV_ERR_ARG


class Calls:
    """Stands for the library: keeps what a call was given."""

    def __getattr__(self, name):
        def call(*args):
            self.name, self.args = name, args
            return 0
        return call


@pytest.mark.parametrize("given", [("row_seq",), ("row_pos",), ("row_slot",), ("row_seq", "row_pos", "row_slot")])
@pytest.mark.parametrize("rows", [0, 5])
def test_row_maps_that_are_empty_are_asked_for_all_the_same(gkv, monkeypatch, given, rows):
    """A tensor without elements has no address; as none at all it would lift the bound of the rows."""
    monkeypatch.setattr(torch.Tensor, "is_pinned", lambda self: True)
    calls = Calls()
    monkeypatch.setattr(gkv, "lib", lambda: calls)
    maps = {n: torch.zeros(rows, dtype=torch.int64 if n == "row_slot" else torch.int32) for n in given}
    gkv.tables_resize(gkv.BlockTables(0x1000, 0x1000, 0x1000, 4, 8, 16), ints(8), stream=NO_STREAM, **maps)
    assert calls.name == "gkv_tables_resize" and calls.args[5] == rows
    for n, address in zip(("row_seq", "row_pos", "row_slot"), calls.args[7:10]):
        assert bool(address) == (n in given)
        assert not address or address % 8 == 0
