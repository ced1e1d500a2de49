"""gkv_tables_resize with row maps of no elements: they bound the new rows as any others do."""
import pytest
import torch

from test_gpu_tables import Tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("S", [2, 65])
def test_no_room_for_a_row(gkv, cuda, S):
    """Nothing changes where there are new rows; rows that end take none."""
    t = Tables(gkv, S, 4, 4 * S, rows=0)
    idle = [0] * (S - 1)
    assert not t.check_resize([5] + idle)
    assert t.check_resize([0] + idle)
    gkv.tables_resize(t.t, torch.tensor([40] + idle, dtype=torch.int32, device="cuda"), workspace=t.ws, dev_err=t.err)  # (no maps: no bound)
    t.m.resize([40] + idle)
    t.same_state()
    assert not t.check_resize([41] + idle)
    assert t.check_resize([7] + idle)
