"""What the Python binding of the kept-token entry points refuses before any pointer is handed over,
and where it takes its stream from."""
from types import SimpleNamespace

import pytest
import torch

D = 64
NO_STREAM = SimpleNamespace(cuda_stream=None)


def ints(*n):
    return torch.zeros(n, dtype=torch.int32)


def rows(n, width, dtype=torch.float32):
    return torch.zeros(n, width, dtype=dtype)


def append(gkv, **o):
    a = dict(qkv=rows(4, 4 * D), cos_tab=rows(8, 32), sin_tab=rows(8, 32), seq_lens=ints(2), cu_seqlens=ints(3),
             k_pack=rows(4, D, torch.bfloat16), v_pack=rows(4, D, torch.int16))
    a.update(o)
    gkv.kept_append(n_q_heads=2, view=gkv.CacheView(n_kv_heads=1), max_rows=4, stream=NO_STREAM, **a)


def decode(gkv, **o):
    a = dict(q=rows(2, 2 * D), seq_lens=ints(2), out=rows(2, 2 * D), sinks=torch.zeros(2), cos_tab=rows(8, 32),
             sin_tab=rows(8, 32))
    a.update(o)
    gkv.kept_decode(n_q_heads=2, max_seq_len=8, view=gkv.CacheView(n_kv_heads=1), stream=NO_STREAM, **a)


def prefill(gkv, **o):
    a = dict(cu_seqlens=ints(3), q=rows(4, 2 * D), out=rows(4, 2 * D), start_pos=ints(2), k=rows(4, D, torch.bfloat16),
             v=rows(4, D, torch.bfloat16), sinks=torch.zeros(2), cos_tab=rows(8, 32), sin_tab=rows(8, 32))
    a.update(o)
    gkv.kept_prefill(max_len=4, n_q_heads=2, view=gkv.CacheView(n_kv_heads=1), stream=NO_STREAM, **a)


def copy(gkv, **o):
    a = dict(src=ints(4), dst=ints(4))
    a.update(o)
    gkv.copy_blocks([gkv.CacheView(n_kv_heads=1)], stream=NO_STREAM, **a)


LONGS, HALF = torch.zeros(4, dtype=torch.int64), torch.float16
CASES = [(append, dict(qkv=rows(4, 4 * D, torch.bfloat16))), (append, dict(qkv=rows(4 * D, 4).t())),
         (append, dict(seq_lens=LONGS[:2])), (append, dict(cu_seqlens=LONGS[:3])), (append, dict(seq_lens=ints(4)[::2])),
         (append, dict(cos_tab=rows(8, 32, torch.float64))), (append, dict(k_pack=rows(4, D))),
         (append, dict(k_pack=rows(4, D, HALF))),
         (append, dict(v_pack=rows(4, 2 * D, torch.int16)[:, :D])),
         (decode, dict(q=rows(2, 2 * D, HALF))), (decode, dict(out=rows(2, 2 * D, HALF))),
         (decode, dict(out=rows(2 * D, 2).t())), (decode, dict(seq_lens=LONGS[:2])), (decode, dict(sinks=torch.zeros(2, dtype=HALF))),
         (decode, dict(sin_tab=rows(8, 32, torch.bfloat16))),
         (prefill, dict(q=rows(4, 2 * D, torch.bfloat16))), (prefill, dict(out=rows(4, 2 * D, HALF))),
         (prefill, dict(cu_seqlens=LONGS[:3])), (prefill, dict(start_pos=LONGS[:2])), (prefill, dict(k=rows(4, D))),
         (prefill, dict(v=rows(4, D, torch.float64))), (prefill, dict(sinks=torch.zeros(2, dtype=torch.bfloat16))),
         (copy, dict(src=LONGS)), (copy, dict(dst=LONGS)), (copy, dict(src=ints(8)[::2])), (copy, dict(dst=ints(4, 2)[:, 0])),
         (copy, dict(dst=ints(3)))]


@pytest.mark.parametrize("call,bad", CASES)
def test_refused_tensors(gkv, monkeypatch, call, bad):
    monkeypatch.setattr(torch.Tensor, "is_pinned", lambda self: True)  # (host memory that the GPU can read)
    with pytest.raises(ValueError, match=next(iter(bad)) + "|src and dst"):
        call(gkv, **bad)


@pytest.mark.parametrize("call", [append, decode, prefill, copy])
def test_host_memory_is_refused(gkv, call):
    with pytest.raises(ValueError, match="not in GPU memory"):
        call(gkv)


def test_the_current_stream_by_the_public_way(gkv, monkeypatch):
    """A torch without the private function."""
    monkeypatch.delattr(torch._C, "_cuda_getCurrentRawStream", raising=False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda: SimpleNamespace(cuda_stream=0x70))
    assert gkv.stream_handle() == 0x70
    assert gkv.stream_handle(SimpleNamespace(cuda_stream=0x80)) == 0x80
