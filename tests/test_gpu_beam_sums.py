"""The sums of gkv_beam_select: the same for equal rows wherever those lie and however they are cut, and close to
the definition.

Tolerance: sixteen neighbouring logits' exponentials are summed in fp32 against their largest. A
difference d from it, times log2 e, is off by 2^-24 + 2^-24 + 2^-25 of itself, which moves its term by at most
d 2^-22.6, and 15 terms d exp(-d) against 1 + 15 exp(-d) are at most 1.4; the exponential 2^-23; 15
additions 2^-24 each; the largest's own exponential and the product with it 2^-23 + 2^-23 + 2^-24: under
2^-19 together. All beyond that is in 64 bits. The output rounds to fp32."""
import numpy as np
import pytest
import torch

from test_gpu_beam import expect, logits, run

pytestmark = pytest.mark.gpu
FP32, BF16 = torch.float32, torch.bfloat16


def within(got, want):
    scores, parents, tokens, ended, err = got
    s, p, t, _ = want
    assert np.array_equal(parents, p) and np.array_equal(tokens, t) and err == 0
    fin = np.isfinite(s)
    assert np.array_equal(scores[~fin], s[~fin])
    assert (np.abs(scores[fin] - s[fin]) <= 2.0 ** -19 + np.abs(s[fin]) * 2.0 ** -24).all()


def rows_of(x, dtype, pad=0, shift=0):
    """x as rows of a larger array, at a stride and a start of their own."""
    n, V = x.shape
    whole = torch.full((n * (V + pad) + shift + 8,), 50.0, dtype=dtype, device="cuda")
    t = whole[shift:shift + n * (V + pad)].view(n, V + pad)[:, :V]
    t.copy_(torch.from_numpy(x))
    return t


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("dtype,V,pad,shift", [(FP32, 2001, 0, 0), (FP32, 32001, 0, 0), (FP32, 2000, 1, 2),
                                               (BF16, 2001, 0, 0), (BF16, 32003, 2, 1), (FP32, 131, 0, 1)])
def test_equal_rows_tie(gkv, cuda, dtype, V, pad, shift, seed):
    """Of equal beams the lower one comes first, wherever their rows begin."""
    rng = np.random.default_rng(seed)
    x = np.repeat(logits(rng, 2, V), 4, 0)
    for n in (4, 9):
        t = rows_of(x, dtype, pad, shift)
        cum = np.repeat(rng.standard_normal(2) - 5, 4)
        within(run(gkv, t, cum, 4, n), expect(t.float().cpu().numpy(), cum.astype(np.float32), 4, n))


@pytest.mark.parametrize("dtype,V", [(FP32, 2001), (FP32, 50001), (BF16, 9003)])
def test_equal_beams_alone_and_in_a_batch(gkv, cuda, dtype, V):
    """Requests of which two beams are equal, alone (rows cut among many workgroups) and among 300 (few)."""
    rng = np.random.default_rng(V)
    x = logits(rng, 900, V)
    x[2::3] = x[::3]
    cum = (rng.standard_normal(900) - 5).astype(np.float32)
    cum[2::3] = cum[::3]
    t = rows_of(x, dtype)
    many = run(gkv, t, cum, 3, 7)
    for r in (0, 1, 150, 299):
        one = run(gkv, t[3 * r:3 * r + 3], cum[3 * r:3 * r + 3], 3, 7)
        within(one, expect(t[3 * r:3 * r + 3].float().cpu().numpy(), cum[3 * r:3 * r + 3], 3, 7))
        assert np.array_equal(one[1][0] + 3 * r, many[1][r]) and np.array_equal(one[2][0], many[2][r])
        assert (np.abs(one[0][0] - many[0][r]) <= np.abs(one[0][0]) * 2.0 ** -23).all()


@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("V,scale,at", [(1, 1, 0), (17, 3, 0), (1000, 0.1, 0), (5003, 2.5, 0), (40001, 4, 0), (150000, 1, 0),
                                        (3001, 20, 0), (3001, 2, 500), (3001, 2, -500), (3001, 2, -640), (3001, 2, 660),
                                        (3001, 2, -2000), (3001, 2, 2000), (3001, 30, 90000), (3001, 30, -90000)])
def test_scores(gkv, cuda, dtype, V, scale, at):
    """Logits of all sizes, near 0 and far from it."""
    rng = np.random.default_rng(V)
    for n in (1, min(V, 40)):
        t = rows_of(logits(rng, 6, V, scale) + np.float32(at), dtype)
        cum = (rng.standard_normal(6) * 3 - 10).astype(np.float32)
        within(run(gkv, t, cum, 2, n), expect(t.float().cpu().numpy(), cum, 2, n))


@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("mask", [-1e4, -65504.0, -1e9, -1e30, float("-inf"), None])
def test_masked_rows_tie(gkv, cuda, dtype, mask):
    """All but some tokens masked, a row of masked ones alone, equal rows of both."""
    rng = np.random.default_rng(3)
    V = 20001
    low = float(torch.finfo(dtype).min) if mask is None else mask
    x = np.full((8, V), low, np.float32)
    x[:2, rng.permutation(V)[:30]] = logits(rng, 1, 30)
    x[3], x[2] = x[1], x[0]
    t = rows_of(x, dtype)
    cum = np.array([-3, -4, -3, -4, -2, -2, -1, -1], np.float32)
    within(run(gkv, t, cum, 4, 6), expect(t.float().cpu().numpy(), cum, 4, 6))
