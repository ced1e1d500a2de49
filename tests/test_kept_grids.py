"""Calls of more workgroups than a launch counts are refused, on the CPU, before anything is launched."""
import pytest

from test_kept import append, decode, view


def test_append_of_too_many_rows(gkv):
    for rows in (2**31 - 1, 2**28, 2**28 - 30):
        assert append(gkv, rows=rows) == gkv.GKV_ERR_UNSUPPORTED


@pytest.mark.parametrize("B,max_len,heads", [(2**23, 100, 8), (2**21, 2000, 8), (2**26, 1, 1)])
def test_decode_of_too_many_sequences(gkv, B, max_len, heads):
    assert decode(gkv, view(gkv, n_kv_heads=heads), B=B, hq=heads, max_len=max_len) == gkv.GKV_ERR_UNSUPPORTED
