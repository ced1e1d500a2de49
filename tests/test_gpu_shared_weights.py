"""Weights and scores of shared tokens keep the bits that the other decode's keep: outputs that are what
two nearly equal sums leave of each other, where a weight or a query of fewer bits shows whole.

Tolerance of a bf16 output: q in two pieces (2^-16 against bf16 K, 2^-22 against codes; an fp16 piece
below 2^-14 of the head's largest element is subnormal, 2^-25 of that), 64 products and their pieces summed,
66 roundings of 2^-24 of each piece's sum: a score is off by d, a weight by at most 2 d of itself;
p in two bf16 pieces, 2^-8 of 2^-8; exponential, scale and sums over the tokens 2^-17 together; the
output's own rounding 2^-8 of it."""
import numpy as np
import pytest
import torch

from keptcase import BF16, BLOCK, BT, PLACES, e4m3
from oracle import kv_oracle as O
from sharedcase import D, Shared, dev, within

pytestmark = pytest.mark.gpu
G = 8


def fill(s, k, v):
    """The same K and V [tokens, 64] for every sequence, as far as it goes (values of both formats)."""
    c = s.c
    for b in range(s.B):
        L = int(c.lens[b])
        c.kv[b] = tuple(x[:L, None].astype(np.float64) for x in (k, v))
        for j in range(-(-L // BT)):
            phys, n = c.table[b, j], min(L - j * BT, BT)
            if phys < 0:
                continue
            for i, (pool, x) in enumerate(((c.k, k), (c.v, v))):
                x, at = np.ascontiguousarray(x[j * BT:j * BT + n], np.float32), PLACES[c.fmt][i][:n].reshape(-1)
                if c.fmt == BF16:
                    pool[phys, 0, at] = O.to_bf16(x).reshape(-1)
                else:
                    c.s[phys, 0, i] = 0.25
                    pool[phys, 0, at] = e4m3(x * 4).reshape(-1)


def check(gkv, fmt, lens, blocks, q, k, v):
    """q [8 heads, 64], for every sequence."""
    s = Shared(lens, [len(lens)], [blocks], 1, fmt)
    fill(s, k, v)
    view = s.c.device(gkv)
    qs = np.repeat(np.asarray(q, np.float32)[None], s.B, 0)
    out = torch.zeros(s.B, G * D, dtype=torch.bfloat16, device="cuda")
    mo = int(s.c.lens.max()) - blocks * BT
    ws = torch.empty(gkv.shared_workspace_bytes(s.B, 1, G, 1, blocks, mo), dtype=torch.uint8, device="cuda")
    gkv.shared_decode(dev(qs.reshape(s.B, -1)), G, dev(s.cu), dev(s.shared), dev(s.c.lens), int(s.c.lens.max()), view, out,
                      blocks, mo, workspace=ws, dev_err=s.c.err)
    want, pav, qk, qmax = s.expect(qs, None)
    d = qk * ((2.0 ** -16 if fmt == BF16 else 2.0 ** -22) + 2 * 66 * 2.0 ** -24) + qmax * 2.0 ** -25
    bound = pav * (2 * d + 2.0 ** -16 + 2.0 ** -17) + np.abs(want) * 2.0 ** -8 + 1e-30
    within(out.float().cpu().numpy().reshape(want.shape), want, bound, f"{fmt} {len(lens)}")
    assert int(s.c.err.item()) == 0


# (group sizes of all the shapes that query heads are dealt out in)
SIZES = [2, 4, 8, 16, 40]


@pytest.mark.parametrize("fmt", [BF16, BLOCK])
@pytest.mark.parametrize("size", SIZES)
def test_weights_that_bf16_does_not_hold(gkv, cuda, fmt, size):
    """Half of the tokens weigh 1 and hold 1, the others weigh 1 / r and hold -r: outputs of nearly 0."""
    blocks = 12
    T = blocks * BT + 3
    ratio = np.array([1.5, 1.25, 1.75, 3.0, 5.0, 7.0, 1.375, 1.625])
    rng = np.random.default_rng(size)
    kind = rng.permutation(np.arange(T) % 2)
    k, v = np.zeros((T, D)), np.zeros((T, D))
    k[kind == 0, 0] = 1.0
    q = np.zeros((G, D))
    q[:, 0] = 8 * np.log(ratio)
    v[kind == 0] = 1.0
    v[kind == 1] = -np.repeat(ratio, D // G)  # (each head's outputs vanish in eight of the dims)
    check(gkv, fmt, T - np.arange(size) % 3, blocks, q, k, v)


@pytest.mark.parametrize("fmt", [BF16, BLOCK])
@pytest.mark.parametrize("size", SIZES)
def test_queries_that_11_bits_do_not_hold(gkv, cuda, fmt, size):
    """Tokens that see the half of the query that 11 bits round up, against ones that see the other: scores
    of about 96 that are nearly equal, and values of both signs."""
    blocks = 12
    T = blocks * BT + 3
    rng = np.random.default_rng(size)
    kind = rng.permutation(np.arange(T) % 2)
    k = np.zeros((T, D))
    k[kind == 0, :32] = 24.0
    k[kind == 1, 32:] = 24.0
    q = np.ones((G, D))
    q[:, :32] += np.linspace(0.44, 0.49, G)[:, None] * 2.0 ** -10
    q[:, 32:] += np.linspace(0.56, 0.51, G)[:, None] * 2.0 ** -10
    v = np.where(kind[:, None] == 0, 1.0, -1.0) * np.ones((T, D))
    check(gkv, fmt, T - np.arange(size) % 3, blocks, q, k, v)
