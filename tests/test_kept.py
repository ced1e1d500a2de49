"""The refusals of the gkv_kept_* entry points, gkv_copy_blocks and the pool's sharing calls,
on the CPU: every check fails before anything is launched."""
import ctypes

import pytest

FAKE = 0x1000  # never dereferenced


def view(gkv, **kw):
    d = dict(k=FAKE, v=FAKE, block_table=FAKE, table_stride=8, num_blocks=8, n_kv_heads=8, ring=0,
             v_scale=FAKE, v_format=gkv.KV_FP8_BLOCK)
    d.update(kw)
    return gkv.CacheView(**d)


VIEWS = [  # what every entry point refuses of a cache
    (dict(v_format=1), {}, "UNSUPPORTED"), (dict(v_format=2), {}, "UNSUPPORTED"),
    (dict(v_format=4), {}, "ARG"), (dict(v_format=-1), {}, "ARG"),
    (dict(v_scale=None), {}, "ARG"), (dict(v_scale=FAKE + 4), {}, "ARG"),
    (dict(k=FAKE + 8), {}, "ARG"), (dict(v=None), {}, "ARG"), (dict(block_table=None), {}, "ARG"),
    (dict(block_table=FAKE + 2), {}, "ARG"), (dict(table_stride=0), {}, "ARG"),
    (dict(num_blocks=0), {}, "ARG"), (dict(n_kv_heads=0), {}, "ARG"), (dict(ring=-16), {}, "ARG"),
    (dict(ring=48), {}, "ARG"),                         # a ring without a window
    (dict(ring=32), dict(window=32), "ARG"),            # exactly W slots
    (dict(ring=112), dict(window=96, kept=32), "ARG"),  # 9 entries, the row has 8
    ({}, dict(kept=8), "UNSUPPORTED"), ({}, dict(window=8), "UNSUPPORTED"),
    ({}, dict(kept=-16), "ARG"), ({}, dict(window=-16), "ARG"),
]


def append(gkv, v=None, **o):
    a = dict(B=2, cu=FAKE, lens=FAKE, rows=4, qkv=FAKE, stride=80 * 64, hq=64, cos=FAKE, sin=FAKE,
             kept=0, window=0, kp=None, vp=None)
    a.update(o)
    return gkv.lib().gkv_kept_append(None, a["B"], a["cu"], a["lens"], a["rows"], a["qkv"], a["stride"],
                                     a["hq"], a["cos"], a["sin"], v or view(gkv), a["kept"], a["window"],
                                     a["kp"], a["vp"], None)


def decode(gkv, v=None, **o):
    a = dict(B=2, hq=64, q=FAKE, stride=80 * 64, cos=FAKE, sin=FAKE, lens=FAKE, max_len=100, kept=0,
             window=0, sinks=None, ws=FAKE, ws_bytes=1 << 40, out=FAKE, out_stride=64 * 64, dtype=0)
    a.update(o)
    return gkv.lib().gkv_kept_decode(None, a["B"], a["hq"], a["q"], a["stride"], a["cos"], a["sin"],
                                     a["lens"], a["max_len"], v or view(gkv), a["kept"], a["window"],
                                     a["sinks"], a["ws"], a["ws_bytes"], a["out"], a["out_stride"],
                                     a["dtype"], None)


def prefill(gkv, cache=None, **o):
    a = dict(B=2, cu=FAKE, start=FAKE, max_len=100, hq=64, q=FAKE, stride=80 * 64, cos=FAKE, sin=FAKE,
             k=FAKE, v=FAKE, kept=0, window=0, sinks=None, out=FAKE, out_stride=64 * 64, dtype=0)
    a.update(o)
    return gkv.lib().gkv_kept_prefill(None, a["B"], a["cu"], a["start"], a["max_len"], a["hq"], a["q"],
                                      a["stride"], a["cos"], a["sin"], a["k"], a["v"], cache or view(gkv),
                                      a["kept"], a["window"], a["sinks"], a["out"], a["out_stride"],
                                      a["dtype"], None)


@pytest.mark.parametrize("call", [append, decode, prefill])
@pytest.mark.parametrize("cache,args,why", VIEWS)
def test_refused_caches(gkv, call, cache, args, why):
    assert call(gkv, view(gkv, **cache), **args) == getattr(gkv, "GKV_ERR_" + why)


@pytest.mark.parametrize("bad,why", [
    (dict(B=-1), "ARG"), (dict(lens=None), "ARG"), (dict(rows=-1), "ARG"), (dict(qkv=None), "ARG"),
    (dict(cos=None), "ARG"), (dict(hq=60), "ARG"), (dict(hq=0), "ARG"), (dict(stride=80 * 64 - 1), "ARG"),
    (dict(stride=80 * 64 + 2), "ARG"), (dict(qkv=FAKE + 4), "ARG"), (dict(sin=FAKE + 8), "ARG"),
    (dict(kp=FAKE + 2), "ARG"), (dict(cu=None, rows=2), "ARG"), (dict(B=65536), "UNSUPPORTED")])
def test_append_refusals(gkv, bad, why):
    assert append(gkv, **bad) == getattr(gkv, "GKV_ERR_" + why)


def test_nothing_to_do(gkv):
    none = view(gkv, k=None, v=None, v_scale=None)
    assert append(gkv, B=0) == gkv.GKV_OK
    assert append(gkv, rows=0) == gkv.GKV_OK
    assert append(gkv, none) == gkv.GKV_OK  # no cache and no packed rows
    assert decode(gkv, B=0) == gkv.GKV_OK
    assert prefill(gkv, B=0) == gkv.GKV_OK
    assert prefill(gkv, max_len=0) == gkv.GKV_OK


@pytest.mark.parametrize("bad,why", [
    (dict(B=-1), "ARG"), (dict(q=None), "ARG"), (dict(lens=None), "ARG"), (dict(out=None), "ARG"),
    (dict(max_len=-1), "ARG"), (dict(dtype=2), "ARG"), (dict(cos=None), "ARG"), (dict(hq=60), "ARG"),
    (dict(stride=64 * 64 - 4), "ARG"), (dict(stride=64 * 64 + 2), "ARG"), (dict(out_stride=64 * 64 - 4), "ARG"),
    (dict(out_stride=64 * 64 + 2), "ARG"), (dict(q=FAKE + 4), "ARG"), (dict(out=FAKE + 8), "ARG"),
    (dict(out=FAKE + 4, dtype=1), "ARG"), (dict(hq=72), "UNSUPPORTED"),
    (dict(max_len=20000, ws=None), "WORKSPACE"), (dict(max_len=20000, ws_bytes=1000), "WORKSPACE"),
    (dict(max_len=20000, ws=FAKE + 8), "ARG"), (dict(B=1 << 30, max_len=1 << 20), "UNSUPPORTED")])
def test_decode_refusals(gkv, bad, why):
    assert decode(gkv, **bad) == getattr(gkv, "GKV_ERR_" + why)


def test_decode_head_limits(gkv):
    assert decode(gkv, view(gkv, n_kv_heads=9), hq=9) == gkv.GKV_ERR_UNSUPPORTED
    assert gkv.lib().gkv_kept_workspace_bytes(4, 9, 100, 0, 0) == 0


@pytest.mark.parametrize("bad,why", [
    (dict(cu=None), "ARG"), (dict(q=None), "ARG"), (dict(out=None), "ARG"), (dict(k=None), "ARG"),
    (dict(sin=None), "ARG"), (dict(hq=60), "ARG"), (dict(hq=72), "UNSUPPORTED"), (dict(dtype=2), "ARG"),
    (dict(stride=64 * 64 + 2), "ARG"), (dict(k=FAKE + 4), "ARG"), (dict(max_len=-1), "ARG")])
def test_prefill_refusals(gkv, bad, why):
    assert prefill(gkv, **bad) == getattr(gkv, "GKV_ERR_" + why)


def test_prefill_needs_keys_from_somewhere(gkv):
    none = view(gkv, k=None, v=None)
    assert prefill(gkv, none) == gkv.GKV_ERR_ARG                            # a history without a cache
    assert prefill(gkv, none, start=None, k=None, v=None) == gkv.GKV_ERR_ARG
    # a ring holds the history only
    assert prefill(gkv, view(gkv, ring=48), window=32, k=None, v=None) == gkv.GKV_ERR_ARG


@pytest.mark.parametrize("bad", [dict(k=None), dict(v=None), dict(num_blocks=0), dict(n_kv_heads=0),
                                 dict(v_format=4), dict(v_scale=None), dict(k=FAKE + 8), dict(v_scale=FAKE + 4)])
def test_copy_refusals(gkv, bad):
    views = gkv.cache_views([view(gkv), view(gkv, **bad)])
    assert gkv.lib().gkv_copy_blocks(None, views, 2, 1, FAKE, FAKE, None) == gkv.GKV_ERR_ARG


def test_copy_argument_checks(gkv):
    L, views = gkv.lib(), gkv.cache_views([view(gkv)])
    assert L.gkv_copy_blocks(None, None, 1, 1, FAKE, FAKE, None) == gkv.GKV_ERR_ARG
    assert L.gkv_copy_blocks(None, views, 1, -1, FAKE, FAKE, None) == gkv.GKV_ERR_ARG
    assert L.gkv_copy_blocks(None, views, -1, 1, FAKE, FAKE, None) == gkv.GKV_ERR_ARG
    assert L.gkv_copy_blocks(None, views, 1, 1, None, FAKE, None) == gkv.GKV_ERR_ARG
    assert L.gkv_copy_blocks(None, views, 1, 1, FAKE, None, None) == gkv.GKV_ERR_ARG
    assert L.gkv_copy_blocks(None, views, 1, 0, None, None, None) == gkv.GKV_OK
    assert L.gkv_copy_blocks(None, None, 0, 5, FAKE, FAKE, None) == gkv.GKV_OK


def test_pool_refusals(gkv):
    L, h = gkv.lib(), ctypes.c_void_p()
    cfg = lambda window=32, fmt=3: gkv.PoolConfig(2, 2, 64, window, 2, 100, 8, 0, 0, fmt)  # noqa: E731
    make = lambda c, kept: L.gkv_pool_create_kept(ctypes.byref(c), kept, ctypes.byref(h))  # noqa: E731
    assert make(cfg(), 8) == gkv.GKV_ERR_UNSUPPORTED
    assert make(cfg(), -16) == gkv.GKV_ERR_ARG
    assert make(cfg(window=0), 16) == gkv.GKV_ERR_ARG
    assert make(cfg(window=24), 16) == gkv.GKV_ERR_UNSUPPORTED
    assert make(cfg(fmt=1), 16) == gkv.GKV_ERR_UNSUPPORTED
    assert make(cfg(fmt=2), 16) == gkv.GKV_ERR_UNSUPPORTED
    assert make(cfg(), 2000000000) == gkv.GKV_ERR_ARG
    assert L.gkv_pool_create_kept(None, 16, ctypes.byref(h)) == gkv.GKV_ERR_ARG
    # rings of exactly W slots cannot hold the block format
    assert L.gkv_pool_create(ctypes.byref(cfg()), ctypes.byref(h)) == gkv.GKV_ERR_UNSUPPORTED
    s = ctypes.c_int32()
    assert L.gkv_pool_seq_fork(None, 0, 0, None, ctypes.byref(s)) == gkv.GKV_ERR_ARG
    assert L.gkv_pool_seq_trim(None, 0, 0, None) == gkv.GKV_ERR_ARG
    assert L.gkv_pool_compact(None, None, None) == gkv.GKV_ERR_ARG


def test_other_entry_points_refuse_the_block_format(gkv):
    L, v = gkv.lib(), view(gkv)
    assert L.gkv_kv_append(None, 1, FAKE, 80 * 64, 64, FAKE, FAKE, FAKE, None, None, v, None, 0, None, None,
                           None) == gkv.GKV_ERR_ARG
    assert L.gkv_decode_attention(None, 1, 64, FAKE, 80 * 64, None, None, FAKE, 100, v, 0, FAKE, 0, FAKE,
                                  1 << 40, FAKE, 4096, 0, None) == gkv.GKV_ERR_ARG
    assert L.gkv_prefill_paged(None, 1, FAKE, FAKE, 10, 64, FAKE, 80 * 64, None, None, FAKE, FAKE, v, FAKE, 0,
                               FAKE, 4096, 0, None) == gkv.GKV_ERR_ARG
