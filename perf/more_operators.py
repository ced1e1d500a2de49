"""Timed cases of sequences that share their first blocks: beams, samples of one prompt.

Kinds:

  shared   one query token per sequence; the sequences of a group hold the same
           first blocks, each its own ones behind them
  select   beam search's choice: the best of beams x vocabulary for every request
  reorder  block tables, lengths and holders follow the chosen parents, twice (to
           one choice, then to another, so that every pass moves rows)
  resize   blocks taken and given back by new lengths, with the map of the new
           rows, and back again
  step     reorder, then one more token for every live row: the partly filled block
           that it shares with its parent is replaced by one of its own

Lengths are spread evenly over a range, the same for every seed, and dealt in the
seed's order; blocks are scattered over the pool.
"""
import importlib.util
import math
import os
import sys

import numpy as np
import torch

own = False  # False: plain torch operations; True: the calls that a user makes of gkv.py

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
D = 64                # head dim
BT = 16               # tokens per block
EOS = 2               # the token that ends a sequence
BF16, FP8B = 0, 3     # cache formats: bf16; e4m3 with a scale per block and head

_gkv = None


def gkv():
    global _gkv
    if _gkv is None:
        path = os.path.join(ROOT, "optimize_inference_gpt-oss_amd", "gkv.py")
        spec = importlib.util.spec_from_file_location("gkv", path)
        _gkv = importlib.util.module_from_spec(spec)
        sys.modules["gkv"] = _gkv
        spec.loader.exec_module(_gkv)
        _gkv.lib()
    return _gkv


# ---- cases ------------------------------------------------------------------


def listed():
    return [
        # Four beams of one request: the smallest call, latency counts.
        dict(name="shared_beams_1x4", kind="shared", groups=1, per=4, plo=2048, phi=2048, lo=1, hi=64,
             fmt=BF16, Hq=64, Hkv=8, sinks=True, out="bfloat16"),
        # Beam search for a batch of requests, eight beams each.
        dict(name="shared_beams_64x8", kind="shared", groups=64, per=8, plo=256, phi=2048, lo=1, hi=256,
             fmt=FP8B, Hq=64, Hkv=8, sinks=True, out="bfloat16"),
        # A serving batch behind one system prompt.
        dict(name="shared_prompt_1x512", kind="shared", groups=1, per=512, plo=2048, phi=2048, lo=129,
             hi=1025, fmt=BF16, Hq=64, Hkv=8, sinks=True, out="bfloat16"),
        # Samples of two long documents' answers.
        dict(name="shared_long_2x16", kind="shared", groups=2, per=16, plo=24000, phi=30000, lo=10, hi=700,
             fmt=FP8B, Hq=64, Hkv=8, sinks=False, out="float32"),
        # One request's four beams, a small vocabulary.
        dict(name="select_1x4", kind="select", R=1, K=4, V=32001, n=4, dtype="float32", done=0.0),
        # A batch of requests in the middle of their search, a large vocabulary.
        dict(name="select_64x8", kind="select", R=64, K=8, V=131072, n=16, dtype="float32", done=0.1),
        # Logits as a bf16 product leaves them (many are equal), five beams.
        dict(name="select_24x5_bf16", kind="select", R=24, K=5, V=200000, n=10, dtype="bfloat16", done=0.2),
        # A request's beams after 100000 tokens, and the hypotheses that it keeps.
        dict(name="reorder_1x16_long", kind="reorder", groups=1, keep=8, live=8, pre=64, lo=60000, hi=100000,
             blocks=131072),
        # A batch of beam searches: as many kept rows as live ones.
        dict(name="reorder_64x16", kind="reorder", groups=64, keep=8, live=8, pre=64, lo=1500, hi=4000,
             blocks=262144),
        # The same batch's next token.
        dict(name="step_64x16", kind="step", groups=64, keep=8, live=8, pre=64, lo=1500, hi=4000,
             blocks=262144),
        # Eight drafted tokens for four chats, and back: the smallest call.
        dict(name="resize_draft_b4", kind="resize", S=4, lo=100, hi=5000, add_lo=8, add_hi=8, share=1.0,
             blocks=4096),
        # Prompts admitted to half of a serving batch's rows, and given up again.
        dict(name="resize_prompts_b512", kind="resize", S=512, lo=100, hi=3000, add_lo=64, add_hi=512,
             share=0.5, blocks=131072),
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    kind = rng.choice(["shared"] * 4 + ["select"] * 3 + ["reorder", "step", "resize", "resize"])
    if kind == "shared":
        Hq, Hkv = rng.choice([(64, 8)] * 4 + [(32, 4), (16, 2), (8, 1), (40, 8), (6, 3), (7, 7)])
        B = _log(rng, 2, 512)
        per = min(B, _log(rng, 2, 512))
        phi = _log(rng, 16, min(30000, 1200000 // B))
        hi = _log(rng, 1, max(2, min(2000, 1300000 // B - phi)))
        return dict(kind=kind, groups=B // per, per=per, plo=rng.randint(0, phi), phi=phi, lo=rng.randint(1, hi),
                    hi=hi, fmt=rng.choice([BF16, FP8B]), Hq=Hq, Hkv=Hkv, sinks=rng.random() < 0.7,
                    out=rng.choice(["bfloat16", "bfloat16", "float32"]))
    if kind == "select":
        V = _log(rng, 1000, 200000)
        K = _log(rng, 1, 16)
        R = _log(rng, 1, max(1, 67000000 // V // K))
        return dict(kind=kind, R=min(R, 256), K=K, V=V, n=rng.randint(1, 2 * K + 2),
                    dtype=rng.choice(["float32", "bfloat16"]), done=rng.choice([0.0, 0.2]))
    if kind == "resize":
        S = _log(rng, 1, 1024)
        hi = _log(rng, 20, min(20000, 1500000 // S))
        add = _log(rng, 1, max(2, min(4000, 100000 // S)))
        return dict(kind=kind, S=S, lo=rng.randint(1, hi), hi=hi, add_lo=rng.randint(1, add), add_hi=add,
                    share=rng.choice([0.25, 0.5, 1.0]),
                    blocks=int(S * ((hi + add) / BT + 2) * rng.uniform(1.05, 2)))
    live, keep = _log(rng, 1, 24), _log(rng, 1, 8)
    groups = _log(rng, 1, 1000 // (live + keep) + 1)
    hi = _log(rng, 40, min(100000, 2700000 // (groups * (live + keep))))
    return dict(kind=kind, groups=groups, keep=keep, live=live, pre=rng.randint(0, hi // BT), lo=rng.randint(1, hi),
                hi=hi, blocks=int(groups * (live + keep) * (hi / BT + 3) * rng.uniform(1.05, 1.5)))


def _spread(n, lo, hi):
    return [lo + int((i + 0.5) / n * (hi - lo + 1)) for i in range(n)]


# ---- inputs -----------------------------------------------------------------


def _pool(gen, nb, c):
    """A pool's K, V and scales: values of about unit size, scales that vary by block."""
    H = c["Hkv"]
    r = lambda: torch.randn((nb, H, BT * D), generator=gen, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    if c["fmt"] == BF16:
        return r(), r(), None
    codes = lambda: (r().float() * 100).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)  # noqa: E731
    e = torch.randint(-9, -4, (nb, H, 2), generator=gen, device="cuda")
    return codes(), codes(), torch.exp2(e.float())


def _angles(n):
    a = torch.arange(n, device="cuda", dtype=torch.float64)[:, None] * 150000.0 ** (
        -torch.arange(D // 2, device="cuda", dtype=torch.float64) / (D // 2))
    return a.cos().float(), a.sin().float()


def _dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def _prepare_shared(c, gen, rng):
    g, per = c["groups"], c["per"]
    B = g * per
    shared = rng.permutation(_spread(g, c["plo"], c["phi"])).astype(np.int64) // BT   # blocks
    mine = rng.permutation(_spread(B, c["lo"], c["hi"])).astype(np.int64)             # tokens behind them
    first = np.repeat(shared, per)
    lens = first * BT + mine
    stride = int((-(-lens // BT)).max())
    n_own = -(-mine // BT)
    nb = int(shared.sum() + n_own.sum())
    ids = rng.permutation(nb).astype(np.int32)
    s0 = np.concatenate([[0], np.cumsum(shared)])
    o0 = int(s0[-1]) + np.concatenate([[0], np.cumsum(n_own)])
    j = np.arange(stride)[None]
    f, grp = first[:, None], np.repeat(np.arange(g), per)
    at = np.where(j < f, s0[grp][:, None] + j, o0[:-1, None] + j - f)
    table = np.where(j < f + n_own[:, None], ids[np.clip(at, 0, nb - 1)], -1).astype(np.int32)
    k, v, sc = _pool(gen, nb, c)
    s = {"k": k, "v": v, "sc": sc, "table": _dev(table), "lens": _dev(lens.astype(np.int32)),
         "shared": _dev(shared.astype(np.int32)), "cu": _dev(np.arange(g + 1, dtype=np.int32) * per),
         "max_len": int(lens.max()), "max_shared": int(shared.max()), "max_own": int(mine.max())}
    s["cos"], s["sin"] = _angles(s["max_len"])
    s["q"] = torch.randn((B, (c["Hq"] + 2 * c["Hkv"]) * D), generator=gen, device="cuda")
    s["sinks"] = torch.randn(c["Hq"], generator=gen, device="cuda") if c["sinks"] else None
    return s


def _prepare_select(c, gen, rng):
    rows = c["R"] * c["K"]
    x = torch.randn((rows, c["V"]), generator=gen, device="cuda") * 2.5
    hot = torch.randint(0, c["V"] // 40, (rows, 40), generator=gen, device="cuda")
    hot += torch.arange(40, device="cuda") * (c["V"] // 40)
    x.scatter_(1, hot, torch.randn((rows, 40), generator=gen, device="cuda") * 3 + 12)  # likely tokens
    x[:, ::97] = -math.inf                                                              # forbidden ones
    x[:, EOS] = 11
    cum = torch.randn(rows, generator=gen, device="cuda") * 1.5 - 20
    done = torch.rand(rows, generator=gen, device="cuda") < c["done"]
    return {"x": x.to(getattr(torch, c["dtype"])), "cum": cum, "done": done.int()}


def _rows(lens, pre, groups, blocks, rng, stride):
    """A table over a scattered pool in which the rows of a group hold the same first blocks."""
    S = len(lens)
    per = S // groups
    n = -(-lens // BT)
    p = np.repeat(np.minimum(lens.reshape(groups, per).min(1) // BT, pre), per)
    ids = rng.permutation(blocks).astype(np.int64)
    grp = np.arange(S) // per
    s0 = np.concatenate([[0], np.cumsum(p[::per])])
    o0 = int(s0[-1]) + np.concatenate([[0], np.cumsum(n - p)])
    j = np.arange(stride)[None]
    at = np.where(j < p[:, None], s0[grp][:, None] + j, o0[:-1, None] + j - p[:, None])
    table = np.where(j < n[:, None], ids[np.clip(at, 0, blocks - 1)], -1).astype(np.int32)
    refs = np.bincount(table[table >= 0], minlength=blocks).astype(np.int32)
    return {"table": _dev(table), "lens": _dev(lens.astype(np.int32)), "refs": _dev(refs)}


def _prepare_tables(c, rng):
    if c["kind"] == "resize":
        S = c["S"]
        lens = rng.permutation(_spread(S, c["lo"], c["hi"])).astype(np.int64)
        n = max(1, int(S * c["share"]))
        more = np.zeros(S, np.int64)
        more[rng.permutation(S)[:n]] = _spread(n, c["add_lo"], c["add_hi"])
        if c["share"] < 1:  # (prompts: the rows that get tokens are empty before)
            lens[more > 0] = 0
        s = _rows(lens, 0, S, c["blocks"], rng, -(-(c["hi"] + c["add_hi"]) // BT) + 8)
        rows = int(more.sum())
        s.update(was=s["lens"].clone(), more=_dev((lens + more).astype(np.int32)))
    else:
        per = c["keep"] + c["live"]
        S = c["groups"] * per
        lens = rng.permutation(_spread(S, c["lo"], c["hi"])).astype(np.int64)
        s = _rows(lens, c["pre"], c["groups"], c["blocks"], rng, -(-c["hi"] // BT) + 8)
        at = np.arange(S).reshape(c["groups"], per)
        for name in ("p1", "p2"):
            p = at.copy()
            p[:, c["keep"]:] = at[:, :1] + rng.integers(0, c["keep"], (c["groups"], c["live"]))
            s[name] = _dev(p.reshape(-1).astype(np.int32))
        s["one"] = _dev(np.tile(np.arange(per) >= c["keep"], c["groups"]).astype(np.int32))
        s["shared"] = torch.zeros(c["groups"], dtype=torch.int32, device="cuda")
        rows = c["groups"] * c["live"]
    i32 = lambda n: torch.zeros(n, dtype=torch.int32, device="cuda")  # noqa: E731
    s.update(src=i32(S), dst=i32(S), cu=i32(S + 1), row_seq=i32(rows), row_pos=i32(rows),
             row_slot=torch.zeros(rows, dtype=torch.int64, device="cuda"))
    return s


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    if c["kind"] == "shared":
        s = _prepare_shared(c, gen, rng)
    elif c["kind"] == "select":
        s = _prepare_select(c, gen, rng)
    else:
        s = _prepare_tables(c, rng)
    s.update(c=c, err=torch.zeros(1, dtype=torch.int32, device="cuda"))
    return s


# ---- the plain form ------------------------------------------------------------


def _cells(s):
    """K and V of the pool by token and dimension, as views: [block, head, token..., dim...]."""
    n, H = s["k"].shape[:2]
    if s["c"]["fmt"] == BF16:
        return (s["k"].view(n, H, 2, 4, 16, 8).permute(0, 1, 4, 2, 3, 5),
                s["v"].view(n, H, 2, 4, 16, 2, 4).permute(0, 1, 3, 6, 2, 5, 4))
    return (s["k"].view(n, H, 4, 16, 2, 8).permute(0, 1, 3, 4, 2, 5),
            s["v"].view(n, H, 16, 4, 4, 4).permute(0, 1, 3, 5, 4, 2))


def _gather(s):
    """K and V of every position, fp32 [B, Hkv, T, 64]."""
    kc, vc = _cells(s)
    table = s["table"].clamp(min=0).long()
    B, n = table.shape
    at, off = table.repeat_interleave(BT, 1), torch.arange(n * BT, device="cuda").expand(B, -1) % BT
    kk, vv = kc[at, :, off].reshape(B, n * BT, -1, D), vc[at, :, off // 4, off % 4].reshape(B, n * BT, -1, D)
    if s["c"]["fmt"] == BF16:
        kk, vv = kk.float(), vv.float()
    else:
        sc = s["sc"][at]
        kk = kk.view(torch.float8_e4m3fn).float() * sc[..., 0, None]
        vv = vv.view(torch.float8_e4m3fn).float() * sc[..., 1, None]
    return kk.transpose(1, 2).contiguous(), vv.transpose(1, 2).contiguous()


def _plain_shared(s):
    c = s["c"]
    B, Hq, H = s["q"].shape[0], c["Hq"], c["Hkv"]
    at = (s["lens"] - 1).long()
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
    q = s["q"][:, :Hq * D].view(B, Hq, D)
    q = torch.cat([q[..., :32] * cos - q[..., 32:] * sin, q[..., 32:] * cos + q[..., :32] * sin], -1)
    k, v = _gather(s)
    z = torch.matmul(q.view(B, H, Hq // H, D), k.transpose(2, 3).contiguous()) * 0.125
    seen = torch.arange(k.shape[2], device="cuda") < s["lens"][:, None]
    z = z.masked_fill(~seen[:, None, None], -math.inf)
    m = z.amax(-1, keepdim=True)
    if c["sinks"]:
        sk = s["sinks"].view(1, H, Hq // H, 1)
        m = torch.maximum(m, sk)
    p = torch.exp(z - m)
    den = p.sum(-1, keepdim=True)
    if c["sinks"]:
        den = den + torch.exp(sk - m)
    return (torch.matmul(p, v) / den).view(B, Hq * D).to(getattr(torch, c["out"]))


def _plain_select(s):
    c = s["c"]
    R, K, V, n = c["R"], c["K"], c["V"], c["n"]
    x = s["x"].float()
    m = x.amax(1, keepdim=True)
    # (the logarithm's sum in 64 bits: a beam's choice hangs on it next to another beam's)
    lse = m[:, 0].double() + torch.log(torch.exp(x - m).sum(1, dtype=torch.float64))
    z = s["cum"].double()[:, None] + (x.double() - lse[:, None])
    done = s["done"] != 0
    z = z.masked_fill(done[:, None], -math.inf)
    z[:, EOS] = torch.where(done, s["cum"].double(), z[:, EOS])
    z = z.view(R, K * V)
    # the n largest, of equal ones those that come first
    low = torch.topk(z, n, 1).values[:, -1:]
    above, equal = z > low, z == low
    take = above | (equal & (equal.cumsum(1) <= n - above.sum(1, keepdim=True)))
    at = take.nonzero()[:, 1].view(R, n)
    val, order = torch.sort(z.gather(1, at), dim=1, descending=True, stable=True)
    at = at.gather(1, order)
    beam, token = at // V, at % V
    row = torch.arange(R, device="cuda")[:, None] * K + beam
    return {"scores": val.float(), "parents": row.int(), "tokens": token.int(),
            "done": ((token == EOS) | done[row]).int()}


def _plain_reorder(s, parents):
    per = parents.shape[0] // s["c"]["groups"]
    old = s["table"].clone()
    s["table"].copy_(old[parents.long()])
    s["lens"].copy_(s["lens"][parents.long()])
    moved = s["table"] != old
    for t, by in ((old, -1), (s["table"], 1)):  # what is held less, what more
        s["refs"].add_(torch.bincount(t[moved & (t >= 0)], minlength=s["refs"].shape[0]), alpha=by)
    t = s["table"].view(-1, per, old.shape[1])
    same = (t == t[:, :1]).all(1)
    full = s["lens"].view(-1, per).amin(1) // BT
    same &= torch.arange(old.shape[1], device="cuda") < full[:, None]
    s["shared"].copy_(same.int().cumprod(1).sum(1))


def _plain_resize(s, new, maps=True):
    lens, table, refs = s["lens"].clone(), s["table"], s["refs"]
    S, stride = table.shape
    nb = refs.shape[0]
    grow = new > lens
    have, want = (lens + BT - 1) // BT, (new + BT - 1) // BT
    last = table.gather(1, (lens // BT).clamp(max=stride - 1).long()[:, None])[:, 0]
    split = grow & (lens % BT != 0) & (refs[last.clamp(min=0).long()] > 1)
    take = split.int() + (want - have).clamp(min=0)
    before = take.cumsum(0).int() - take
    free = refs == 0
    rank = torch.where(free, free.cumsum(0) - 1, nb)
    ids = torch.zeros(nb + 1, dtype=torch.int32, device="cuda")
    ids[rank] = torch.arange(nb, dtype=torch.int32, device="cuda")
    # rows given back, blocks replaced, rows taken
    j = torch.arange(stride, device="cuda")[None]
    gone = (j >= want[:, None]) & (j < have[:, None])
    refs.sub_(torch.bincount(torch.cat([table[gone], last[split]]), minlength=nb))
    part = split[:, None] & (j == lens[:, None] // BT)
    come = part | ((j >= have[:, None]) & (j < want[:, None]))
    at = torch.where(part, before[:, None], (before + split)[:, None] + j - have[:, None])
    got = ids[at.clamp(0, nb).long()]
    table.copy_(torch.where(come, got, torch.where(gone, -1, table)))
    refs.add_(torch.bincount(got[come], minlength=nb))
    s["src"].copy_(torch.where(split, last, 0))
    s["dst"].copy_(torch.where(split, got.gather(1, (lens // BT).clamp(max=stride - 1).long()[:, None])[:, 0], 0))
    s["lens"].copy_(new)
    if not maps:
        return
    # the new rows
    cu = s["cu"]
    cu[1:] = (new - lens).clamp(min=0).cumsum(0)
    r = torch.arange(s["row_seq"].shape[0], dtype=torch.int32, device="cuda")
    seq = torch.searchsorted(cu, r, right=True).clamp(max=S) - 1
    pos = lens[seq] + r - cu[seq]
    slot = table[seq, (pos // BT).clamp(0, stride - 1).long()].long() * BT + pos % BT
    new_row = r < cu[-1]
    for name, x in (("row_seq", seq), ("row_pos", pos), ("row_slot", slot)):
        s[name].copy_(torch.where(new_row, x.to(s[name].dtype), s[name]))


# ---- one pass ------------------------------------------------------------------


def _tables_out(s):
    names = ["table", "lens", "refs", "src", "dst", "cu", "row_seq", "row_pos", "row_slot"]
    if s["c"]["kind"] == "reorder":
        names = ["table", "lens", "refs"]
    return {n: s[n] for n in names + (["shared"] if "shared" in s else [])}


def _own_shared(s):
    g, c = gkv(), s["c"]
    B = s["q"].shape[0]
    if "view" not in s:
        s["view"] = g.cache_view(s["k"], s["v"], s["table"], c["Hkv"], v_scale=s["sc"], v_format=c["fmt"])
        s["ws"] = torch.empty(max(1, g.shared_workspace_bytes(B, c["groups"], c["Hq"], c["Hkv"], s["max_shared"],
                                                              s["max_own"])), dtype=torch.uint8, device="cuda")
    out = torch.empty(B, c["Hq"] * D, dtype=getattr(torch, c["out"]), device="cuda")
    g.shared_decode(s["q"], c["Hq"], s["cu"], s["shared"], s["lens"], s["max_len"], s["view"], out,
                    max_shared_blocks=s["max_shared"], max_own=s["max_own"], sinks=s["sinks"], cos_tab=s["cos"],
                    sin_tab=s["sin"], workspace=s["ws"], dev_err=s["err"])
    return out


def _own_select(s):
    g, c = gkv(), s["c"]
    if "ws" not in s:
        s["ws"] = torch.empty(max(1, g.beam_workspace_bytes(c["R"], c["K"], c["V"], c["n"])), dtype=torch.uint8,
                              device="cuda")
    i32 = lambda: torch.empty(c["R"], c["n"], dtype=torch.int32, device="cuda")  # noqa: E731
    o = {"scores": torch.empty(c["R"], c["n"], device="cuda"), "parents": i32(), "tokens": i32(), "done": i32()}
    g.beam_select(s["x"], s["cum"], c["K"], o["scores"], o["parents"], o["tokens"], done=s["done"], eos=EOS,
                  done_out=o["done"], workspace=s["ws"], dev_err=s["err"])
    return o


def _own_tables(s):
    g, c = gkv(), s["c"]
    if "t" not in s:
        s["t"] = g.block_tables(s["table"], s["lens"], s["refs"])
        s["ws"] = torch.empty(max(1, g.tables_workspace_bytes(s["lens"].shape[0], c["blocks"])), dtype=torch.uint8,
                              device="cuda")
    t = s["t"]
    resize = lambda new: g.tables_resize(  # noqa: E731
        t, new, s["src"], s["dst"], cu_rows=s["cu"], row_seq=s["row_seq"], row_pos=s["row_pos"],
        row_slot=s["row_slot"], workspace=s["ws"], dev_err=s["err"])
    if c["kind"] == "resize":
        resize(s["more"])
        g.tables_resize(t, s["was"], s["src"], s["dst"], workspace=s["ws"], dev_err=s["err"])
        return _tables_out(s)
    per = c["keep"] + c["live"]
    g.tables_reorder(t, s["p1"], per, shared_blocks=s["shared"], dev_err=s["err"])
    if c["kind"] == "reorder":
        g.tables_reorder(t, s["p2"], per, shared_blocks=s["shared"], dev_err=s["err"])
    else:
        resize(s["lens"] + s["one"])
    return _tables_out(s)


def run(s):
    kind = s["c"]["kind"]
    if own:
        return _own_shared(s) if kind == "shared" else _own_select(s) if kind == "select" else _own_tables(s)
    if kind == "shared":
        return _plain_shared(s)
    if kind == "select":
        return _plain_select(s)
    if kind == "resize":
        _plain_resize(s, s["more"])
        _plain_resize(s, s["was"], maps=False)
        return _tables_out(s)
    _plain_reorder(s, s["p1"])
    if kind == "reorder":
        _plain_reorder(s, s["p2"])
    else:
        _plain_resize(s, s["lens"] + s["one"])
    return _tables_out(s)


def work(c):
    if c["kind"] == "shared":
        H, B = c["Hkv"], c["groups"] * c["per"]
        token = H * (256 if c["fmt"] == BF16 else 2056 / BT)
        first = [x // BT * BT for x in _spread(c["groups"], c["plo"], c["phi"])]
        mine = sum(_spread(B, c["lo"], c["hi"]))
        seen = sum(first) * c["per"] + mine
        return {"bytes": (sum(first) + mine) * token + B * c["Hq"] * D * (4 + (2 if c["out"] == "bfloat16" else 4)),
                "flops": 4 * seen * c["Hq"] * D}
    if c["kind"] == "select":
        rows = c["R"] * c["K"] * (1 - c["done"])
        return {"bytes": rows * c["V"] * (4 if c["dtype"] == "float32" else 2) + c["R"] * c["n"] * 16,
                "flops": 3 * rows * c["V"]}
    if c["kind"] == "resize":
        n = max(1, int(c["S"] * c["share"]))
        rows = sum(_spread(n, c["add_lo"], c["add_hi"]))
        taken = rows / BT + n / 2
        # the new rows' maps; per block its entry and holder, taken and given back; the holders
        # that have to be looked at to find as many free ones; the lengths
        return {"bytes": rows * 16 + taken * 16 + min(c["blocks"], 2 * taken) * 4 + c["S"] * 24, "flops": 0}
    S = c["groups"] * (c["keep"] + c["live"])
    entries = c["groups"] * c["live"] * ((c["lo"] + c["hi"]) / 2 / BT)
    if c["kind"] == "reorder":  # twice: a live row's entries read and written, its holders changed
        return {"bytes": 2 * (entries * 8 + 2 * max(0, entries - c["groups"] * c["live"] * c["pre"]) * 4 + S * 12),
                "flops": 0}
    return {"bytes": entries * 8 + c["groups"] * c["live"] * (24 + 16 + 16) + S * 24, "flops": 0}


# ---- the definition, in 64 bits --------------------------------------------------


def _e4m3_values():
    """The value of each of the 256 codes: sign, 4 exponent bits (bias 7), 3 mantissa bits."""
    v = np.empty(256)
    for i in range(256):
        e, m = (i >> 3) & 15, i & 7
        x = math.nan if (e, m) == (15, 7) else (8 + m) * 2.0 ** (e - 10) if e else m * 2.0 ** -9
        v[i] = -x if i & 128 else x
    return v


def _places(fmt):
    """Element of (token, dim) in a head's K block and in its V block, [16, 64]."""
    t, d = np.arange(BT)[:, None], np.arange(D)[None]
    if fmt == BF16:
        return (d // 32 * 512 + (d % 32 // 8 * 16 + t) * 8 + d % 8,
                d // 32 * 512 + (t // 4 * 16 + d % 16) * 8 + d // 16 % 2 * 4 + t % 4)
    return ((d % 32 // 8 * 16 + t) * 16 + d // 32 * 8 + d % 8,
            (d % 16 * 4 + t // 4) * 16 + d // 16 * 4 + t % 4)


def _exact_shared(s):
    c = s["c"]
    Hq, H = c["Hq"], c["Hkv"]
    values = torch.from_numpy(_e4m3_values()).cuda()
    lens = s["lens"].tolist()
    outs = []
    for b, n in enumerate(lens):
        ids = s["table"][b, :-(-n // BT)].long()
        kv = []
        for i, (pool, place) in enumerate(zip((s["k"], s["v"]), _places(c["fmt"]))):
            x = pool[ids][:, :, torch.from_numpy(place).cuda()]              # [blocks, H, 16, 64]
            x = x.double() if c["fmt"] == BF16 else values[x.long()] * s["sc"][ids, :, i].double()[..., None, None]
            kv.append(x.transpose(0, 1).reshape(H, -1, D)[:, :n])
        q = s["q"][b, :Hq * D].double().view(H, Hq // H, D)
        cos, sin = s["cos"][n - 1].double(), s["sin"][n - 1].double()
        q = torch.cat([q[..., :32] * cos - q[..., 32:] * sin, q[..., :32] * sin + q[..., 32:] * cos], -1)
        z = torch.bmm(q, kv[0].transpose(1, 2).contiguous()) / 8
        if c["sinks"]:
            z = torch.cat([z, s["sinks"].double().view(H, -1, 1)], 2)
        outs.append(torch.bmm(torch.softmax(z, 2)[..., :n].contiguous(), kv[1].contiguous()).reshape(-1))
    return torch.stack(outs)


def exact(case, seed):
    if case["kind"] not in ("shared", "select"):
        return None  # (whole numbers only)
    s = prepare(case, seed)
    if case["kind"] == "shared":
        return _exact_shared(s)
    R, K, V, n = (case[x] for x in "RKVn")
    best = []
    for r in range(R):
        got = []
        for b in range(r * K, r * K + K):
            if s["done"][b]:
                got.append(s["cum"][b:b + 1].double())
            else:
                top = torch.topk(torch.log_softmax(s["x"][b].double(), 0), min(n, V)).values
                got.append(top + s["cum"][b].double())
        got = torch.sort(torch.cat(got), descending=True).values[:n]
        best.append(torch.cat([got, got.new_full((n - len(got),), -math.inf)]))
    return {"scores": torch.stack(best), "parents": None, "tokens": None, "done": None}
