"""Sequences that share their first blocks: seeded caches, what a decode over them must give in 64
bits, and a plain model of the block tables."""
from __future__ import annotations

import numpy as np
import torch

from keptcase import BF16, BT, Cache, Layout, attend
from oracle import kv_oracle as O

D = 64


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


class Shared:
    """sizes: sequences per group (what is left of lens is in no group); shared: blocks per group.
    The rows of a group's later sequences hold no ids where the group's blocks stand, unless
    the sequence is shorter than those."""

    def __init__(self, lens, sizes, shared, Hkv, fmt, seed=0, **kw):
        self.c = c = Cache(lens, Hkv, Layout(0, 0, False), fmt, seed=seed, **kw)
        self.cu = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
        self.shared = np.asarray(shared, np.int32)
        for g, n in enumerate(shared):
            b0, b1 = self.cu[g], self.cu[g + 1]
            for b in range(b0 + 1, b1):
                if c.lens[b] < n * BT:
                    continue
                for x, y in zip(c.kv[b], c.kv[b0]):
                    x[:n * BT] = y[:n * BT]
                c.table[b, :n] = -9
            assert b0 >= b1 or c.lens[b0] >= n * BT
        self.B = c.B

    def run(self, gkv, Hq, sinks=None, bf16=False, rotate=True, pad=0, hints=None, max_len=None, seed=1,
            q_scale=1.0, stream=None):
        """Outputs, and (out, sum p|v|, largest sum |qk|/8, rest of q's pieces) in 64 bits."""
        c = self.c
        rng = np.random.default_rng(seed)
        q = (rng.standard_normal((self.B, Hq, D)) * q_scale).astype(np.float32)
        cap = int(max(c.lens.max(initial=0), 1))
        cos, sin = O.rope_table(cap)
        view = c.device(gkv)
        x = torch.full((self.B, Hq * D + pad), float("nan"), device="cuda")
        x[:, :Hq * D] = dev(q.reshape(self.B, -1))
        out = torch.full((self.B, Hq * D + pad), 7.0, dtype=torch.bfloat16 if bf16 else torch.float32, device="cuda")
        if hints is None:
            first = np.repeat(np.append(self.shared, 0), np.append(np.diff(self.cu), self.B - self.cu[-1])) * BT
            hints = int(self.shared.max(initial=0)), max(int((c.lens - first).max(initial=0)), 0)
        ms, mo = hints
        n = gkv.shared_workspace_bytes(self.B, len(self.shared), Hq, c.Hkv, ms, mo)
        self.ws = torch.full((max(n, 16),), 0xFF, dtype=torch.uint8, device="cuda")
        call = lambda: gkv.shared_decode(  # noqa: E731
            x[:, :Hq * D], Hq, dev(self.cu), dev(self.shared), dev(c.lens), cap if max_len is None else max_len, view,
            out[:, :Hq * D], ms, mo, sinks=None if sinks is None else dev(sinks),
            cos_tab=dev(cos) if rotate else None, sin_tab=dev(sin) if rotate else None, workspace=self.ws[:n],
            dev_err=c.err, stream=stream)
        call()
        torch.cuda.synchronize()
        if pad:
            assert (out[:, Hq * D:] == 7.0).all()
        if rotate:
            at = np.maximum(c.lens - 1, 0)
            q = O.kv_append(np.concatenate([q.reshape(self.B, -1), np.zeros((self.B, 2 * c.Hkv * D), np.float32)], 1),
                            Hq, c.Hkv, cos, sin, at.astype(np.int32))[0].reshape(self.B, Hq, D)
        return out[:, :Hq * D].float().cpu().numpy().reshape(self.B, Hq, D), q, x, out, call

    def expect(self, q, sinks, seen=None):
        """seen[b]: positions that count (None: all)."""
        Hq = q.shape[1]
        G = Hq // self.c.Hkv
        got = [np.zeros((self.B, Hq, D)) for _ in range(2)] + [np.zeros((self.B, Hq, 1)) for _ in range(2)]
        for b in range(self.B):
            L = int(self.c.lens[b])
            t = np.arange(L) if seen is None else np.asarray(seen[b], int)
            k, v = self.c.kv[b][0][t], self.c.kv[b][1][t]
            o, pav, qk = attend(q[b:b + 1].astype(np.float64), k, v, np.ones((1, len(t)), bool), sinks)
            got[0][b], got[1][b], got[2][b] = o[0], pav[0], qk[0]
            if len(t):
                ks = np.abs(k).sum(-1).max(0)  # [Hkv]
                got[3][b, :, 0] = np.abs(q[b]).max(-1) * np.repeat(ks, G) / 8
        return got


def shared_bound(out, pav, qk, qmax, fmt, bf16):
    """Largest error of an output. q: one rounding to fp16 against codes (2^-11 of an element) and
    two to bf16 against bf16 K (2^-16), for fp32 outputs two (2^-22) and three (2^-24); a piece
    of fp16 below 2^-14 of the head's largest element is subnormal: 2^-25 of that. 64 products
    and their pieces summed: 66 roundings of 2^-24 of each piece's sum. A score error d moves a
    weight by at most 2 d. p: one rounding to bf16 (2^-8), three (2^-24) for fp32 outputs; the
    exponential, the scale and the sums over the tokens 2^-17 together. The output's own rounding."""
    pieces = (2.0 ** -16 if fmt == BF16 else 2.0 ** -11) if bf16 else 2.0 ** -24 if fmt == BF16 else 2.0 ** -22
    d = qk * (pieces + 2 * 66 * 2.0 ** -24) + qmax * 2.0 ** -25
    return pav * (2 * d + (2.0 ** -8 if bf16 else 2.0 ** -24) + 2.0 ** -17) + 1e-30 + np.abs(out) * (
        2.0 ** -8 if bf16 else 2.0 ** -24)


def within(got, want, bound, what=""):
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), f"{what}: {bad.sum()} outputs off, first at {np.argwhere(bad)[0].tolist()}, by " \
                          f"{np.nanmax(np.abs(got - want)[bad]):.3g} (bound {bound[bad].min():.3g})"


# ---- block tables -----------------------------------------------------------------


class Model:
    """The tables as they have to be, one row and block at a time."""

    def __init__(self, n_seqs, stride, blocks):
        self.table = np.full((n_seqs, stride), -1, np.int32)
        self.lens = np.zeros(n_seqs, np.int32)
        self.refs = np.zeros(blocks, np.int32)

    def resize(self, new, max_rows=None):
        """(ok, src, dst, cu, seq, pos, slot, flags)"""
        S, stride = self.table.shape
        flags = 0
        new = np.asarray(new, np.int64).copy()
        for s in range(S):
            if new[s] < 0 or -(-new[s] // BT) > stride:
                new[s] = self.lens[s]
                flags |= 2
        free = list(np.nonzero(self.refs == 0)[0])
        want = []  # (s, entry, block replaced or None)
        for s in range(S):
            L = int(self.lens[s])
            if new[s] > L:
                if L % BT and self.refs[self.table[s, L // BT]] > 1:
                    want.append((s, L // BT, int(self.table[s, L // BT])))
                want += [(s, j, None) for j in range(-(-L // BT), -(-int(new[s]) // BT))]
        rows = int(np.maximum(new - self.lens, 0).sum())
        src, dst = np.zeros(S, np.int32), np.zeros(S, np.int32)
        if len(want) > len(free) or (max_rows is not None and rows > max_rows):
            return False, src, dst, np.zeros(S + 1, np.int32), [], [], [], flags | 32
        old = self.lens.copy()
        for s in range(S):
            for j in range(-(-int(new[s]) // BT), -(-int(old[s]) // BT)):
                self.refs[self.table[s, j]] -= 1
                self.table[s, j] = -1
        for (s, j, was), b in zip(want, free):
            if was is not None:
                self.refs[was] -= 1
                src[s], dst[s] = was, b
            self.refs[b] += 1
            self.table[s, j] = b
        self.lens[:] = new
        seq, pos, slot = [], [], []
        cu = [0]
        for s in range(S):
            for p in range(int(old[s]), int(new[s])):
                seq.append(s)
                pos.append(p)
                slot.append(int(self.table[s, p // BT]) * BT + p % BT)
            cu.append(len(seq))
        return True, src, dst, np.asarray(cu, np.int32), seq, pos, slot, flags

    def reorder(self, parents, per):
        S = len(self.lens)
        flags = 0
        table, lens = self.table.copy(), self.lens.copy()
        for s in range(S):
            p, base = int(parents[s]), s // per * per
            if p != -1 and not base <= p < base + per:
                p, flags = s, 1
            self.table[s] = -1 if p < 0 else table[p]
            self.lens[s] = 0 if p < 0 else lens[p]
        self.refs[:] = np.bincount(self.table[self.table >= 0], minlength=len(self.refs))
        shared = []
        for g in range(S // per):
            t, n = self.table[g * per:g * per + per], int(self.lens[g * per:g * per + per].min()) // BT
            same = (t == t[:1]).all(0)[:n]
            shared.append(n if same.all() else int(np.argmin(same)))
        return np.asarray(shared, np.int32), flags
