"""Calls of more workgroups than a launch counts, or of rows past 32-bit offsets, are refused, on the
CPU, before anything is launched."""
import pytest

from test_kept import append, decode, prefill, view


def test_append_of_too_many_rows(gkv):
    for rows in (2**31 - 1, 2**28, 2**28 - 30):
        assert append(gkv, rows=rows) == gkv.GKV_ERR_UNSUPPORTED


@pytest.mark.parametrize("B,max_len,heads", [(2**23, 100, 8), (2**21, 2000, 8), (2**26, 1, 1)])
def test_decode_of_too_many_sequences(gkv, B, max_len, heads):
    assert decode(gkv, view(gkv, n_kv_heads=heads), B=B, hq=heads, max_len=max_len) == gkv.GKV_ERR_UNSUPPORTED


def test_prefill_of_packed_rows_past_32_bits(gkv):
    n = 1 << 20  # 16 rows of them are 2^31 bytes
    assert prefill(gkv, view(gkv, n_kv_heads=n), hq=n, stride=64 * n, out_stride=64 * n) == gkv.GKV_ERR_UNSUPPORTED
