"""Caches of whole blocks with kept first tokens and a window: seeded contents, and what
the append, the decode and the prefill must give, in 64 bits.

Every slot that no query may see (unwritten, out of the window, in a freed block) holds a
NaN or an infinity, and every block that nothing sees has a table entry outside the pool
where the layout allows it, so that a kernel that lets them count shows it.
"""
from __future__ import annotations

import numpy as np
import torch

from kvcase import k_block_offsets, k_fp8_offsets, v_block_offsets, v_int8_offsets
from oracle import kv_oracle as O

D, BT = 64, 16
BF16, BLOCK = 0, 3  # gkv.V_BF16, gkv.KV_FP8_BLOCK
T = np.arange(BT)[:, None]
PLACES = {BF16: (k_block_offsets(), v_block_offsets().T),
          BLOCK: (k_fp8_offsets(T), v_int8_offsets(T))}  # [token, dim] -> element


def e4m3(x):
    """Codes of float32 values that are in range or NaN (to nearest, ties to even)."""
    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(torch.float8_e4m3fn).view(
        torch.uint8).numpy()


def e4m3_values(c):
    return torch.from_numpy(np.ascontiguousarray(c)).view(torch.float8_e4m3fn).float().numpy()


def block_scale(amax):
    """The smallest power of two s with amax <= 448 s, per element; 0 for 0."""
    amax = np.asarray(amax, np.float64)
    s = 2.0 ** np.maximum(np.ceil(np.log2(np.maximum(amax, 1e-300) / 448)), -126)
    return np.where(amax > 0, s, 0).astype(np.float32)


class Layout:
    def __init__(self, kept, window, ring):
        self.kept, self.window, self.ring = kept, window, window + BT if ring else 0

    def entry(self, j):
        kb = self.kept // BT
        if not self.ring or j < kb:
            return j
        return kb + (j - kb) % (self.ring // BT)

    def entries(self, max_len):
        return (self.kept + self.ring) // BT if self.ring else max(1, -(-max_len // BT))

    def sees(self, p, t):
        t = np.asarray(t)
        ok = t <= p
        return ok & ((t < self.kept) | (t > p - self.window)) if self.window else ok


class Cache:
    """A pool with the positions of each sequence that its layout holds before position
    lens[b]; seen(b) says which of them a query may see."""

    def __init__(self, lens, Hkv, layout, fmt, seed=0, scale=1.0, extra=3, spread=False):
        rng = self.rng = np.random.default_rng(seed)
        self.lens, self.Hkv, self.lay, self.fmt = np.asarray(lens, np.int32), Hkv, layout, fmt
        self.B = B = len(lens)
        n = layout.entries(int(max(self.lens.max(initial=0), 1)) + 512)
        self.nb = B * n + extra
        self.table = rng.permutation(self.nb)[:B * n].reshape(B, n).astype(np.int32)
        bad = 0x7FC0 if fmt == BF16 else 0x7F
        dt = np.uint16 if fmt == BF16 else np.uint8
        self.k = np.full((self.nb, Hkv, BT * D), bad, dt)
        self.v = np.full((self.nb, Hkv, BT * D), bad, dt)
        self.s = np.full((self.nb, Hkv, 2), np.nan, np.float32) if fmt == BLOCK else None
        self.kv = []  # per sequence: float64 K and V of every position (NaN where not held)
        for b in range(B):
            L = int(self.lens[b])
            kk, vv = np.full((L, Hkv, D), np.nan), np.full((L, Hkv, D), np.nan)
            for j in range(-(-L // BT)):
                if layout.ring and layout.entry(j) in [layout.entry(i) for i in range(j + 1, -(-L // BT))]:
                    continue  # replaced since
                lo, hi = j * BT, min(L, j * BT + BT)
                phys = self.table[b, layout.entry(j)]
                for i, (pool, out) in enumerate(((self.k, kk), (self.v, vv))):
                    mag = scale * (2.0 ** rng.integers(-6, 6) if spread else 1.0)
                    x = (rng.standard_normal((hi - lo, Hkv, D)) * mag).astype(np.float32)
                    at = PLACES[fmt][i][:hi - lo]
                    if fmt == BF16:
                        h = O.to_bf16(x)
                        out[lo:hi] = O.from_bf16(h)
                        pool[phys, :, at.reshape(-1)] = h.transpose(0, 2, 1).reshape(-1, Hkv)
                    else:
                        # any scale, not only the append's powers of two
                        sc = (np.abs(x).max((0, 2)) / 448 * rng.uniform(1, 3, Hkv)).astype(np.float32)
                        if not spread:
                            sc = block_scale(np.abs(x).max((0, 2)))
                        c = e4m3(np.clip(x / sc[None, :, None], -448, 448))
                        out[lo:hi] = e4m3_values(c).astype(np.float64) * sc[None, :, None]
                        pool[phys, :, at.reshape(-1)] = c.transpose(0, 2, 1).reshape(-1, Hkv)
                        self.s[phys, :, i] = sc
            self.kv.append((kk, vv))

    def poison(self, first_query, last_query, free=True):
        """Fills every slot that the queries first_query[b] .. last_query[b] do not see."""
        lay = self.lay
        for b in range(self.B):
            L = int(self.lens[b])
            qs = range(int(first_query[b]), int(last_query[b]) + 1)
            seen = np.zeros(L, bool)
            for p in qs:
                seen |= lay.sees(p, np.arange(L))
            for j in range(-(-L // BT)):
                t = np.arange(j * BT, min(L, j * BT + BT))
                if np.isnan(self.kv[b][0][t[0]]).all():
                    continue
                gone = t[~seen[t]] % BT
                phys = self.table[b, lay.entry(j)]
                for i, pool in enumerate((self.k, self.v)):
                    at = PLACES[self.fmt][i][gone].reshape(-1)
                    pool[phys, :, at] = (0x7FC0 if i else 0x7F80) if self.fmt == BF16 else 0x7F
                if len(gone) == len(t) and not lay.ring and free:
                    self.table[b, j] = -5  # freed
        return self

    def device(self, gkv):
        t = lambda a: torch.from_numpy(np.ascontiguousarray(a.view(np.int16) if a.dtype == np.uint16 else a)).cuda()  # noqa: E731
        self.dk, self.dv, self.dt = t(self.k), t(self.v), t(self.table)
        self.ds = None if self.s is None else t(self.s)
        self.err = torch.zeros(1, dtype=torch.int32, device="cuda")
        return gkv.cache_view(self.dk, self.dv, self.dt, self.Hkv, ring=self.lay.ring,
                              v_scale=self.ds, v_format=self.fmt)

    def pulled(self):
        u = lambda x, like: x.cpu().numpy().view(like.dtype)  # noqa: E731
        return u(self.dk, self.k), u(self.dv, self.v), None if self.s is None else u(self.ds, self.s)


def attend(q, k, v, ok, sinks):
    """q [n, Hq, 64], k and v [T, Hkv, 64], ok [n, T] in 64 bits: outputs [n, Hq, 64], sum of
    p |v| and the largest sum |q k| / 8 per row and head (for the tolerances)."""
    n, Hq, _ = q.shape
    G = Hq // k.shape[1]
    out, pav, qk = np.zeros((n, Hq, D)), np.zeros((n, Hq, D)), np.zeros((n, Hq, 1))
    for i in range(n):
        t = np.nonzero(ok[i])[0]
        for h in range(Hq):
            z = k[t, h // G] @ q[i, h] / 8
            zs = z if sinks is None else np.append(z, sinks[h])
            if not len(zs) or zs.max() == -np.inf:
                continue
            w = np.exp(zs - zs.max())
            w = (w / w.sum())[:len(t)]
            out[i, h] = w @ v[t, h // G]
            pav[i, h] = w @ np.abs(v[t, h // G])
            if len(t):
                qk[i, h] = (np.abs(k[t, h // G]) @ np.abs(q[i, h])).max() / 8
    return out, pav, qk


def decode_bound(out, pav, qk, fmt, bf16):
    """Largest error of a decode output. Scores: the pieces of q leave 2^-18 of it against bf16
    K (two bf16 roundings of at most 2^-9 each), 2^-22 against codes (two fp16 ones), the sums
    of 64 products 66 roundings of 2^-24; a score error d moves every weight by at most
    2 d (it and the normalisation); p's two bf16 pieces leave 2^-18, exp2, the scale and the sums
    over the tokens 2^-17 together."""
    d = qk * ((2.0 ** -18 if fmt == BF16 else 2.0 ** -22) + 66 * 2.0 ** -24)
    e = pav * (2 * d + 2.0 ** -18 + 2.0 ** -17) + 1e-30
    return e + np.abs(out) * (2.0 ** -8 if bf16 else 2.0 ** -24)


def prefill_bound(out, pav, qk, n_keys, v_max, bf16):
    """Largest error of a prefill output: q as one fp16 piece of its row over the power of two
    below the row's largest element (2^-11 of an element; one below 2^-14 of that power is
    subnormal and off by 2^-25 of it: with q and k of one distribution, as here, the few of
    them stay within 2^-18 of the sum of |q k|), the sums as in decode_bound; p as one fp16 piece (2^-11, in the weight and in the
    sum: 2^-10; 2^-25 each where it is subnormal), V staged as fp16 of v 2^-10 (2^-11, or 2^-15
    where that is subnormal)."""
    d = qk * (2.0 ** -11 + 2.0 ** -18 + 66 * 2.0 ** -24)
    e = pav * (2 * d + 2.0 ** -10 + 2.0 ** -11 + 2.0 ** -17) + 2.0 ** -15 + n_keys * 2.0 ** -25 * v_max
    return e + np.abs(out) * (2.0 ** -8 if bf16 else 2.0 ** -24)
