"""Prefill weights far below the largest one: a sink far above every score, a kept first key that
takes nearly all the weight, scores that climb or fall along the sequence.

Tolerance (n keys, W the sum of a row's weights, beside the sink's): scores, products and sums as in
keptcase.prefill_bound, relative to sum p |v| (V here is 0 or at least 2^-4, which is staged
exactly); a weight is stored as fp16 of 2^8 times its ratio to the largest, or more, so one
of the subnormal ones is off by at most 2^-25 2^-8 of the largest, in the weights and in
their sum: 2 n 2^-33 W max |v|."""
import numpy as np
import pytest
import torch

from keptcase import BF16, BLOCK, BT, D, PLACES, Cache, Layout, e4m3
from oracle import kv_oracle as O

pytestmark = pytest.mark.gpu


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def exact(q, k, v, ok, sinks):
    """Outputs of q [n, H, 64] over one kv head's k, v [T, 64] in 64 bits, and their tolerance."""
    z = np.einsum("nhd,td->nht", q, k) / 8
    qk = np.where(ok[:, None], np.einsum("nhd,td->nht", np.abs(q), np.abs(k)) / 8, 0).max(-1)
    z = np.where(ok[:, None], z, -np.inf)
    sk = np.full(q.shape[1], -np.inf) if sinks is None else sinks.astype(np.float64)
    top = np.maximum(z.max(-1), sk[None])
    w = np.exp(z - top[..., None])
    w /= (w.sum(-1) + np.exp(sk[None] - top))[..., None]
    out, pav, W = w @ v, w @ np.abs(v), w.sum(-1)
    d = qk * (2.0 ** -11 + 2.0 ** -18 + 66 * 2.0 ** -24)
    bound = pav * (2 * d + 2.0 ** -10 + 2.0 ** -11 + 2.0 ** -17)[..., None] + np.abs(out) * 2.0 ** -24
    bound += (W * 2 * len(k) * 2.0 ** -33 * np.abs(v).max())[..., None]
    return out, bound


def run(gkv, k, v, q, start, lay, fmt, sinks, max_len=None):
    """k, v [T, 64] (bf16 values): positions below start in the cache, the others packed rows;
    q [T - start, H, 64]."""
    c = Cache([start], 1, lay, fmt)
    for j in range(start // BT):
        if lay.ring and lay.entry(j) in [lay.entry(i) for i in range(j + 1, start // BT)]:
            continue
        phys = c.table[0, lay.entry(j)]
        for i, (pool, x) in enumerate(((c.k, k), (c.v, v))):
            x = x[j * BT:j * BT + BT]
            if fmt == BF16:
                pool[phys, 0, PLACES[fmt][i].reshape(-1)] = O.to_bf16(np.ascontiguousarray(x, np.float32)).reshape(-1)
            else:
                c.s[phys, 0, i] = 1.0 / 32
                pool[phys, 0, PLACES[fmt][i].reshape(-1)] = e4m3(x * 32).reshape(-1)
    n, H = q.shape[:2]
    view = c.device(gkv)
    out = torch.full((n, H * D), float("nan"), device="cuda")
    packed = [torch.from_numpy(np.ascontiguousarray(x[start:], np.float32)).bfloat16().cuda() for x in (k, v)]
    gkv.kept_prefill(dev(np.array([0, n], np.int32)), max_len or n, dev(q.reshape(n, -1).astype(np.float32)), H, view, out,
                     start_pos=dev(np.array([start], np.int32)), k=packed[0], v=packed[1],
                     sinks=None if sinks is None else dev(sinks), kept=lay.kept, window=lay.window, dev_err=c.err)
    assert int(c.err.item()) == 0
    t = np.arange(len(k))
    ok = np.stack([lay.sees(p, t) for p in range(start, start + n)])
    want, bound = exact(q, k, v, ok, sinks)
    err = np.abs(out.cpu().numpy().reshape(n, H, D) - want)
    assert (err <= bound).all(), float((err / bound).max())


def values(rng, shape):
    """Multiples of 1/16 up to 14/16 of both signs: values of both formats (codes of scale 1/32)."""
    return rng.integers(-14, 15, shape) / 16.0


LAYOUTS = [Layout(0, 0, False), Layout(16, 256, True), Layout(64, 512, False)]
FORMS = [(BF16, None), (BLOCK, None), (BLOCK, 20000)]  # (format, bound of the rows: one group of waves)


@pytest.mark.parametrize("lay", LAYOUTS)
@pytest.mark.parametrize("fmt,max_len", FORMS)
def test_sinks_far_above_the_scores(gkv, cuda, lay, fmt, max_len):
    rng = np.random.default_rng(1)
    T, start = 700, 624
    sinks = np.array([-np.inf, -80, 0, 12, 16, 20, 40, 60], np.float32)
    run(gkv, values(rng, (T, D)), values(rng, (T, D)), rng.standard_normal((T - start, 8, D)).astype(np.float32), start, lay,
        fmt, sinks, max_len)


@pytest.mark.parametrize("lay", LAYOUTS)
@pytest.mark.parametrize("fmt,max_len", FORMS)
@pytest.mark.parametrize("nats", [8, 10, 12, 14, 16, 18])
def test_a_first_key_that_takes_the_weight(gkv, cuda, lay, fmt, max_len, nats):
    """Its V is zero: the output is the others', whose V is positive. Dimension 0 is its alone."""
    rng = np.random.default_rng(nats)
    T, start = 2100, 2048
    k, v = values(rng, (T, D)), np.abs(values(rng, (T, D)))
    q = rng.standard_normal((T - start, 8, D)).astype(np.float32)
    k[:, 0], q[:, :, 0] = 0, 8
    k[0], v[0] = 0, 0
    k[0, 0] = nats / (1 if fmt == BF16 else 2)
    q[:, :, 0] *= 1 if fmt == BF16 else 2
    run(gkv, k, v, q, start, lay, fmt, None, max_len)


@pytest.mark.parametrize("fmt,max_len", FORMS)
@pytest.mark.parametrize("top", [30, -30, 4, -4])
def test_scores_that_climb_or_fall(gkv, cuda, fmt, max_len, top):
    """... by `top` nats over the sequence, in steps of 16 tokens, beside their own spread."""
    rng = np.random.default_rng(7)
    T, start = 1100, 1024
    k, v = values(rng, (T, D)), values(rng, (T, D))
    q = rng.standard_normal((T - start, 8, D)).astype(np.float32)
    step = np.arange(T) // 128 / 8.0                 # 0 .. 1 in eighths: values of both formats
    k[:, 0], q[:, :, 0] = step * 8, top
    run(gkv, k, v, q, start, Layout(0, 0, False), fmt, None, max_len)
