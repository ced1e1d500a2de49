"""Timed cases of the bounded, shared and block-scaled cache.

Kinds:

  copy     blocks of a paged cache copied inside it, in several layers at once
           (a fork's last blocks, a compaction)
  append   new tokens into a cache of whole blocks: RoPE on K, then bf16, or
           e4m3 codes with one scale per block of 16 tokens and head
  decode   one query token per sequence against such a cache
  prefill  prompts, or chunks that continue a cached history

The attention sees position t from position p iff t <= p and (t < kept or
t > p - window); window 0: every t <= p. A cache holds every position's block
in its table, or (windows here) the kept blocks and a ring of window + 16
slots. Lengths are spread evenly over [lo, hi], the same for every seed, and
dealt to the sequences in the seed's order; block tables are random
permutations of the pool's blocks.
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
        # Eight samples forked off one prompt: the last, partly filled block of
        # each in the full layers. Launch latency counts.
        dict(name="copy_fork8", kind="copy", layers=12, blocks=512, pairs=8, fmt=BF16, Hkv=8),
        # A pool compacted after many requests have ended.
        dict(name="copy_compact2048", kind="copy", layers=12, blocks=6144, pairs=2048, fmt=BF16,
             Hkv=8),
        # One decode step's new tokens of a serving batch.
        dict(name="append_step_b512", kind="append", B=512, lo=1, hi=1, start=1056, kept=0, window=0,
             fmt=FP8B, Hq=64, Hkv=8, pack=False),
        # A batch of prompts into an empty cache, with the packed rows that the
        # prefill attention reads.
        dict(name="append_prompts_b64", kind="append", B=64, lo=64, hi=512, start=0, kept=0, window=0,
             fmt=FP8B, Hq=64, Hkv=8, pack=True),
        # Two chats with bounded memory: the smallest call.
        dict(name="decode_kept_b2", kind="decode", B=2, lo=100, hi=5000, kept=64, window=256, fmt=FP8B,
             Hq=64, Hkv=8, sinks=False, out="float32"),
        # A full layer of a serving batch.
        dict(name="decode_full_b512", kind="decode", B=512, lo=129, hi=2049, kept=0, window=0,
             fmt=FP8B, Hq=64, Hkv=8, sinks=True, out="bfloat16"),
        # Three long documents: few sequences, a long axis.
        dict(name="decode_full_b3", kind="decode", B=3, lo=20001, hi=60001, kept=0, window=0, fmt=FP8B,
             Hq=64, Hkv=8, sinks=True, out="float32"),
        # A window layer of a serving batch, the first block kept.
        dict(name="decode_kept_b512", kind="decode", B=512, lo=1, hi=100000, kept=16, window=128,
             fmt=BF16, Hq=64, Hkv=8, sinks=True, out="bfloat16"),
        # Endless chats over a wide window.
        dict(name="decode_kept_w4096", kind="decode", B=97, lo=2000, hi=40000, kept=64, window=4096,
             fmt=FP8B, Hq=64, Hkv=8, sinks=False, out="bfloat16"),
        # Whole prompts of a window layer with its first block kept.
        dict(name="prefill_kept_b12", kind="prefill", B=12, lo=200, hi=1500, start=0, kept=16,
             window=128, fmt=BF16, Hq=64, Hkv=8, sinks=True),
        # Chunks of long prompts after a history in the block format.
        dict(name="prefill_full_chunk_b8", kind="prefill", B=8, lo=100, hi=700, start=1536, kept=0,
             window=0, fmt=FP8B, Hq=64, Hkv=8, sinks=True),
        # The same over a bounded cache, a few rows each.
        dict(name="prefill_kept_chunk_b5", kind="prefill", B=5, lo=20, hi=300, start=2048, kept=64,
             window=256, fmt=FP8B, Hq=64, Hkv=8, sinks=False),
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    kind = rng.choice(["copy", "append", "append", "decode", "decode", "decode", "prefill", "prefill"])
    Hq, Hkv = rng.choice([(64, 8)] * 4 + [(32, 4), (16, 2), (8, 1), (40, 8), (6, 3), (7, 7)])
    fmt = rng.choice([BF16, FP8B, FP8B])
    window = rng.choice([0, 0, 128, 16 * rng.randint(2, 64)])
    kept = 16 * rng.choice([0, 1, rng.randint(0, 8)])
    if kind == "copy":
        layers = rng.randint(1, 36)
        pairs = _log(rng, 1, 24576 // layers)
        return dict(kind=kind, layers=layers, blocks=2 * pairs + rng.randint(0, pairs), pairs=pairs,
                    fmt=fmt, Hkv=Hkv)
    if kind == "append":
        if rng.random() < 0.5:
            return dict(kind=kind, B=_log(rng, 1, 512), lo=1, hi=1, start=rng.randint(0, 1056),
                        kept=kept, window=window, fmt=fmt, Hq=Hq, Hkv=Hkv, pack=False)
        hi = _log(rng, 3, 1024)
        return dict(kind=kind, B=_log(rng, 1, min(64, 18000 // hi)), lo=rng.randint(1, hi), hi=hi,
                    start=rng.choice([0, rng.randint(0, 700)]), kept=kept, window=window, fmt=fmt,
                    Hq=Hq, Hkv=Hkv, pack=rng.random() < 0.5)
    if kind == "decode":
        B = _log(rng, 1, 512)
        hi = _log(rng, 16, min(60000, 700000 // B))
        if window:
            hi = _log(rng, 16, 100000)
        return dict(kind=kind, B=B, lo=rng.randint(1, hi), hi=hi, kept=kept, window=window, fmt=fmt,
                    Hq=Hq, Hkv=Hkv, sinks=rng.random() < 0.5, out=rng.choice(["bfloat16", "float32"]))
    hi = _log(rng, 32, 700)
    return dict(kind=kind, B=rng.randint(1, 8), lo=rng.randint(1, hi), hi=hi,
                start=16 * rng.choice([0, rng.randint(1, 96)]), kept=kept, window=window, fmt=fmt,
                Hq=Hq, Hkv=Hkv, sinks=rng.random() < 0.5)


def _spread(n, lo, hi):
    return [lo + int((i + 0.5) / n * (hi - lo + 1)) for i in range(n)]


def _slots(c):
    """Blocks of a sequence's table row: every position's, or the kept ones and the ring."""
    last = c["hi"] + c.get("start", 0)
    return (c["kept"] + c["window"]) // BT + 1 if c["window"] else -(-last // BT)


def _seen(c, p):
    """How many positions position p sees."""
    if not c["window"]:
        return p + 1
    return p + 1 if p < c["kept"] + c["window"] else c["kept"] + c["window"]


# ---- inputs -----------------------------------------------------------------


def _pool(gen, nb, c):
    """A pool's K, V and scales: values of about unit size, scales that vary by block."""
    dev, H = "cuda", c["Hkv"]
    if c["fmt"] == BF16:
        r = lambda: torch.randn((nb, H, BT * D), generator=gen, device=dev, dtype=torch.bfloat16)  # noqa: E731
        return r(), r(), None
    r = lambda: (torch.randn((nb, H, BT * D), generator=gen, device=dev, dtype=torch.bfloat16).float() * 100  # noqa: E731
                 ).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    e = torch.randint(-9, -4, (nb, H, 2), generator=gen, device=dev)
    return r(), r(), torch.exp2(e.float())


def _angles(n):
    a = torch.arange(n, device="cuda", dtype=torch.float64)[:, None] * 150000.0 ** (
        -torch.arange(D // 2, device="cuda", dtype=torch.float64) / (D // 2))
    return a.cos().float(), a.sin().float()


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    t = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()  # noqa: E731
    s = {"c": c, "err": torch.zeros(1, dtype=torch.int32, device="cuda")}
    if c["kind"] == "copy":
        # one tensor per array, the layers along its first axis
        k, v, sc = _pool(gen, c["layers"] * c["blocks"], c)
        cut = lambda x: None if x is None else x.view(c["layers"], c["blocks"], *x.shape[1:])  # noqa: E731
        ids = rng.permutation(c["blocks"]).astype(np.int32)
        s.update(k=cut(k), v=cut(v), sc=cut(sc), src=t(ids[:c["pairs"]]),
                 dst=t(ids[c["pairs"]:2 * c["pairs"]]))
        return s
    B, H = c["B"], c["Hkv"]
    lens = rng.permutation(_spread(B, c["lo"], c["hi"])).astype(np.int32)
    start = c.get("start", 0)
    n_blk = _slots(c)
    nb = B * n_blk
    k, v, sc = _pool(gen, nb, c)
    s.update(k=k, v=v, sc=sc, table=t(rng.permutation(nb).astype(np.int32).reshape(B, n_blk)))
    s["cos"], s["sin"] = _angles(c["hi"] + start)
    width = (c["Hq"] + 2 * H) * D
    if c.get("sinks"):
        s["sinks"] = torch.randn(c["Hq"], generator=gen, device="cuda")
    if c["kind"] == "decode":
        s["lens"] = t(lens)
        s["qkv"] = torch.randn((B, width), generator=gen, device="cuda")
        return s
    s["qkv"] = torch.randn((int(lens.sum()), width), generator=gen, device="cuda")
    s["cu"] = t(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32))
    if c["kind"] == "append":
        # (sequences of a step stand anywhere inside a block)
        s["start"] = t((start + rng.integers(-min(start, 15), 1, B)).astype(np.int32))
        s["lens"] = s["start"] + t(lens)
        return s
    s["start"] = torch.full((B,), start, dtype=torch.int32, device="cuda")
    s["kp"], s["vp"] = (torch.randn((s["qkv"].shape[0], H * D), generator=gen, device="cuda",
                                    dtype=torch.bfloat16) for _ in "kv")
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


def _block_of(s, blk):
    """Pool block of each sequence's logical block blk [B, n] (clamped into the table)."""
    c = s["c"]
    if c["window"]:
        kb, ring = c["kept"] // BT, c["window"] // BT + 1
        blk = torch.where(blk < kb, blk, kb + (blk - kb) % ring)
    return s["table"].gather(1, blk.clamp(0, s["table"].shape[1] - 1).long()).long()


def _codes(x):
    return x.view(torch.float8_e4m3fn).float()


def _gather(s, pos):
    """K and V of the positions pos [B, T], fp32 [B, Hkv, T, 64]."""
    kc, vc = _cells(s)
    pos = pos.clamp(min=0)
    ids, off = _block_of(s, pos // BT), pos % BT
    B, T = pos.shape
    kk, vv = kc[ids, :, off].reshape(B, T, -1, D), vc[ids, :, off // 4, off % 4].reshape(B, T, -1, D)
    if s["c"]["fmt"] == BF16:
        kk, vv = kk.float(), vv.float()
    else:
        sc = s["sc"][ids]
        kk, vv = _codes(kk) * sc[..., 0, None], _codes(vv) * sc[..., 1, None]
    return kk.transpose(1, 2), vv.transpose(1, 2)


def _rotate(x, cos, sin):
    """RoPE of [..., heads, 64] at the rows' angles [..., 32]. The framework's rounding, so that
    codes next to a border fall alike: second product rounded, first product fused (done in 64 bits)."""
    x1, x2 = x[..., :32], x[..., 32:]
    c, sn = cos[..., None, :], sin[..., None, :]
    a = x1.double() * c.double() - (x2 * sn).double()
    b = x2.double() * c.double() + (x1 * sn).double()
    return torch.cat([a, b], -1).float()


def _attend(q, k, v, mask, sinks, G):
    """q [B, L, Hq, 64], k and v [B, Hkv, T, 64], mask [B, L, T] -> [B, L, Hq, 64]."""
    B, L, Hq, _ = q.shape
    H = Hq // G
    q = q.view(B, L, H, G, D).permute(0, 2, 1, 3, 4).reshape(B, H, L * G, D)
    sc = (torch.matmul(q, k.transpose(2, 3).contiguous()) * 0.125).view(B, H, L, G, -1)
    sc = sc.masked_fill(~mask[:, None, :, None], -math.inf)
    m = sc.amax(-1, keepdim=True)
    if sinks is not None:
        sk = sinks.view(1, H, 1, G, 1)
        m = torch.maximum(m, sk)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = torch.exp(sc - m)
    den = p.sum(-1, keepdim=True)
    if sinks is not None:
        den = den + torch.exp(sk - m)
    o = torch.matmul(p.view(B, H, L * G, -1), v).view(B, H, L, G, D) / den.clamp(min=1e-30)
    return o.permute(0, 2, 1, 3, 4).reshape(B, L, Hq * D)


def _plain_decode(s):
    c = s["c"]
    lens = s["lens"][:, None]
    if c["window"]:
        first = torch.arange(c["kept"], device="cuda")[None].expand(c["B"], -1)
        last = lens - c["window"] + torch.arange(c["window"], device="cuda")
        pos = torch.cat([first, last], 1)
        ok = torch.cat([first < lens, last >= c["kept"]], 1)
    else:
        pos = torch.arange(c["hi"], device="cuda")[None].expand(c["B"], -1)
        ok = pos < lens
    k, v = _gather(s, pos)
    at = (s["lens"] - 1).long()
    q = _rotate(s["qkv"][:, :c["Hq"] * D].view(c["B"], c["Hq"], D), s["cos"][at], s["sin"][at])
    o = _attend(q[:, None], k, v, ok[:, None], s.get("sinks"), c["Hq"] // c["Hkv"])
    return o[:, 0].to(getattr(torch, c["out"]))


def _plain_prefill(s):
    c = s["c"]
    B, H, Lm, h = c["B"], c["Hkv"], c["hi"], c["start"]
    cu, j = s["cu"].long(), torch.arange(c["hi"], device="cuda")
    row = (cu[:-1, None] + j).clamp(max=s["qkv"].shape[0] - 1)
    new = j[None] < (cu[1:] - cu[:-1])[:, None]
    pos = h + j
    q = _rotate(s["qkv"][:, :c["Hq"] * D].view(-1, c["Hq"], D)[row], s["cos"][pos], s["sin"][pos])
    k, v = (x.float().view(-1, H, D)[row].transpose(1, 2) for x in (s["kp"], s["vp"]))
    if h:
        hk, hv = _gather(s, torch.arange(h, device="cuda")[None].expand(B, -1))
        k, v = torch.cat([hk, k], 2), torch.cat([hv, v], 2)
    t = torch.arange(h + Lm, device="cuda")
    ok = t[None] <= pos[:, None]
    if c["window"]:
        ok &= (t[None] < c["kept"]) | (t[None] > pos[:, None] - c["window"])
    out = torch.empty(s["qkv"].shape[0], c["Hq"] * D, dtype=torch.bfloat16, device="cuda")
    o = _attend(q, k, v, ok[None].expand(B, -1, -1), s.get("sinks"), c["Hq"] // H)
    out[row[new]] = o[new].to(torch.bfloat16)
    return out


def _scale_of(amax):
    """The smallest power of two s with amax <= 448 s (0 for amax 0)."""
    m, e = torch.frexp(amax / 448.0)
    s = torch.exp2((e - (m == 0.5).int()).clamp(min=-126).float())
    return torch.where(amax > 0, s, torch.zeros_like(s))


def _to_codes(x, sc):
    inv = torch.where(sc > 0, 1.0 / sc, torch.zeros_like(sc))
    return (x * inv).clamp(-448, 448).to(torch.float8_e4m3fn)


def _plain_append(s):
    c = s["c"]
    B, H = c["B"], c["Hkv"]
    n = -(-c["hi"] // BT) + 1
    first = s["start"].long() // BT
    blk = first[:, None] + torch.arange(n, device="cuda")
    pos = (first * BT)[:, None] + torch.arange(n * BT, device="cuda")
    start, lens = s["start"].long()[:, None], s["lens"].long()[:, None]
    new, old = (pos >= start) & (pos < lens), pos < start
    row = (s["cu"][:-1].long()[:, None] + pos - start).clamp(0, s["qkv"].shape[0] - 1)
    qkv = s["qkv"].view(-1, c["Hq"] + 2 * H, D)
    at = pos.clamp(max=s["cos"].shape[0] - 1)
    xs = (_rotate(qkv[row, c["Hq"]:c["Hq"] + H], s["cos"][at], s["sin"][at]),
          qkv[row, c["Hq"] + H:])
    keep = new.view(B, n, BT).any(-1)
    if c["window"]:  # blocks that later ones of the same call replace in the ring
        last = (lens - 1) // BT
        keep &= (blk < c["kept"] // BT) | (blk + c["window"] // BT + 1 > last)
    ids = _block_of(s, blk)[keep]
    outs = []
    for i, (cells, x) in enumerate(zip(_cells(s), xs)):
        x = x.view(B, n, BT, H, D).permute(0, 1, 3, 2, 4)[keep]         # [blocks, H, 16, 64]
        isnew = new.view(B, n, 1, BT, 1)[keep]
        isold = old.view(B, n, 1, BT, 1)[keep]
        begun = isold.any(2, keepdim=True)  # (slots behind the last token: left as they were)
        was = cells[ids].reshape(x.shape)
        if c["fmt"] == BF16:
            y = torch.where(isnew, x.to(torch.bfloat16), torch.where(begun, was, torch.zeros_like(was)))
            cells[ids] = y.view(cells[ids].shape)
            continue
        so = torch.where(begun[..., 0, 0], s["sc"][ids, :, i], torch.zeros_like(s["sc"][ids, :, i]))
        sn = torch.maximum(so, _scale_of((x.abs() * isnew).amax((2, 3))))
        ratio = torch.where(sn > 0, so / sn, torch.zeros_like(sn))[..., None, None]
        moved = (_codes(was) * ratio).to(torch.float8_e4m3fn).view(torch.uint8)
        y = torch.where(isnew, _to_codes(x, sn[..., None, None]).view(torch.uint8),
                        torch.where(isold, moved, torch.where(begun, was, torch.zeros_like(was))))
        cells[ids] = y.view(cells[ids].shape)
        s["sc"][ids, :, i] = sn
    if c["pack"]:
        at = s["start"].repeat_interleave(s["cu"][1:] - s["cu"][:-1], output_size=qkv.shape[0]).long()
        at = at + torch.arange(qkv.shape[0], device="cuda") - s["cu"][:-1].repeat_interleave(
            s["cu"][1:] - s["cu"][:-1], output_size=qkv.shape[0])
        outs = [_rotate(qkv[:, c["Hq"]:c["Hq"] + H], s["cos"][at], s["sin"][at]).to(torch.bfloat16),
                qkv[:, c["Hq"] + H:].to(torch.bfloat16)]
    return outs


# ---- one pass ------------------------------------------------------------------


def _cache_out(s):
    """The cache after a pass, as the values it holds."""
    f8 = lambda x: x.view(torch.float8_e4m3fn) if s["c"]["fmt"] == FP8B else x  # noqa: E731
    return {"k": f8(s["k"]), "v": f8(s["v"]), **({} if s["sc"] is None else {"sc": s["sc"]})}


def _view(g, s):
    c = s["c"]
    return g.cache_view(s["k"], s["v"], s["table"], c["Hkv"], ring=c["window"] + BT if c["window"] else 0,
                        v_scale=s["sc"], v_format=c["fmt"])


def _run_own(s):
    g, c = gkv(), s["c"]
    if c["kind"] == "copy":
        if "views" not in s:  # a program makes its layers' views once
            s["views"] = g.cache_views([
                g.CacheView(s["k"][i].data_ptr(), s["v"][i].data_ptr(), None, 0, c["blocks"], c["Hkv"], 0,
                            None if s["sc"] is None else s["sc"][i].data_ptr(), c["fmt"])
                for i in range(c["layers"])])
        g.copy_blocks(s["views"], s["src"], s["dst"], dev_err=s["err"])
        return _cache_out(s)
    if "view" not in s:
        s["view"] = _view(g, s)
    kw = dict(kept=c["kept"], window=c["window"], dev_err=s["err"])
    if c["kind"] == "append":
        kp = vp = None
        if c["pack"]:
            kp, vp = (torch.empty(s["qkv"].shape[0], c["Hkv"], D, dtype=torch.bfloat16, device="cuda")
                      for _ in "kv")
        g.kept_append(s["qkv"], c["Hq"], s["cos"], s["sin"], s["lens"], s["view"],
                      cu_seqlens=None if c["hi"] == 1 else s["cu"], max_rows=c["hi"], k_pack=kp,
                      v_pack=vp, **kw)
        return {**_cache_out(s), **({"kp": kp, "vp": vp} if c["pack"] else {})}
    if c["kind"] == "decode":
        if "ws" not in s:
            s["ws"] = torch.empty(max(1, g.kept_workspace_bytes(c["B"], c["Hkv"], c["hi"], c["kept"],
                                                                c["window"])),
                                  dtype=torch.uint8, device="cuda")
        out = torch.empty(c["B"], c["Hq"] * D, dtype=getattr(torch, c["out"]), device="cuda")
        g.kept_decode(s["qkv"], c["Hq"], s["lens"], c["hi"], s["view"], out, sinks=s.get("sinks"),
                      cos_tab=s["cos"], sin_tab=s["sin"], workspace=s["ws"], **kw)
        return out
    out = torch.empty(s["qkv"].shape[0], c["Hq"] * D, dtype=torch.bfloat16, device="cuda")
    g.kept_prefill(s["cu"], c["hi"], s["qkv"], c["Hq"], s["view"], out, start_pos=s["start"],
                   k=s["kp"], v=s["vp"], sinks=s.get("sinks"), cos_tab=s["cos"], sin_tab=s["sin"], **kw)
    return out


def run(s):
    if own:
        return _run_own(s)
    kind = s["c"]["kind"]
    if kind == "copy":
        src, dst = s["src"].long(), s["dst"].long()
        for x in (s["k"], s["v"], s["sc"]):
            if x is not None:
                x[:, dst] = x[:, src]
        return _cache_out(s)
    if kind == "append":
        packs = _plain_append(s)
        return {**_cache_out(s), **({"kp": packs[0], "vp": packs[1]} if packs else {})}
    return _plain_decode(s) if kind == "decode" else _plain_prefill(s)


def work(c):
    H = c["Hkv"]
    block = H * (4096 if c["fmt"] == BF16 else 2056)  # bytes of one block, K and V
    if c["kind"] == "copy":
        return {"bytes": 2 * c["layers"] * c["pairs"] * block, "flops": 0}
    lens = _spread(c["B"], c["lo"], c["hi"])
    if c["kind"] == "append":
        rows = sum(lens)
        return {"bytes": rows * H * (512 + block / H / BT + (256 if c["pack"] else 0)), "flops": 0}
    if c["kind"] == "decode":
        n = sum(_seen(c, x - 1) for x in lens)
        out = 2 if c["out"] == "bfloat16" else 4
        return {"bytes": n * block / BT + c["B"] * c["Hq"] * D * (4 + out), "flops": 4 * n * c["Hq"] * D}
    h = c["start"]
    n = sum(_seen(c, h + j) for x in lens for j in range(x))
    hist = min(h, c["kept"] + c["window"] - 1) if c["window"] else h
    return {"bytes": sum(lens) * (c["Hq"] * D * 6 + H * 256) + c["B"] * hist * block / BT,
            "flops": 4 * n * c["Hq"] * D}


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


def _turn(x, cos, sin):
    """[n, heads, 64] in 64 bits, turned by the rows' angles [n, 32]."""
    a, b = x[..., :32], x[..., 32:]
    c, s = cos.double()[:, None], sin.double()[:, None]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def _exact_rows(s, b, positions):
    """K and V of sequence b at the positions (a host array), in 64 bits [n, Hkv, 64]."""
    c = s["c"]
    blk = positions // BT
    if c["window"]:
        kb, r = c["kept"] // BT, c["window"] // BT + 1
        blk = np.where(blk < kb, blk, kb + (blk - kb) % r)
    ids = s["table"][b][torch.from_numpy(blk).cuda()].long()
    off = positions % BT
    got = []
    for i, (pool, at) in enumerate(zip((s["k"], s["v"]), _places(c["fmt"]))):
        cell = torch.from_numpy(at[off]).cuda()[:, None].expand(-1, c["Hkv"], -1)
        x = pool[ids].gather(2, cell)
        if c["fmt"] == BF16:
            got.append(x.double())
        else:
            got.append(torch.from_numpy(_e4m3_values()).cuda()[x.long()] * s["sc"][ids, :, i].double()[..., None])
    return got


def _exact_attention(q, k, v, ok, sinks):
    """q [L, Hq, 64], k and v [T, Hkv, 64], ok [L, T]."""
    L, Hq, _ = q.shape
    H = k.shape[1]
    out = torch.empty(L, Hq, D, dtype=torch.float64, device="cuda")
    for h in range(Hq):
        g = h // (Hq // H)
        z = (q[:, h] @ k[:, g].T.contiguous() / 8).masked_fill(~ok, -math.inf)
        if sinks is not None:
            z = torch.cat([z, sinks[h].double().expand(L, 1)], 1)
        w = torch.softmax(z, 1)[:, :k.shape[0]]
        out[:, h] = w @ v[:, g].contiguous()
    return out.reshape(L, Hq * D)


def exact(case, seed):
    s = prepare(case, seed)
    c = s["c"]
    if c["kind"] == "copy":
        want = {n: x.clone() for n, x in _cache_out(s).items()}
        for n, x in want.items():
            raw = x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x
            for l in range(c["layers"]):
                raw[l].index_copy_(0, s["dst"].long(), raw[l].index_select(0, s["src"].long()))
        return {n: x.float() if x.dtype == torch.float8_e4m3fn else x for n, x in want.items()}
    Hq, H = c["Hq"], c["Hkv"]
    qkv = s["qkv"].double().view(-1, Hq + 2 * H, D)
    if c["kind"] == "decode":
        lens, outs = s["lens"].cpu().numpy(), []
        for b in range(c["B"]):
            n = int(lens[b])
            p = np.arange(n)
            if c["window"]:
                p = p[(p < c["kept"]) | (p >= n - c["window"])]
            k, v = _exact_rows(s, b, p)
            q = _turn(qkv[b:b + 1, :Hq], s["cos"][n - 1:n], s["sin"][n - 1:n])
            G = Hq // H
            z = torch.matmul(q.view(H, G, D), k.permute(1, 2, 0).contiguous()) / 8
            if s.get("sinks") is not None:
                z = torch.cat([z, s["sinks"].double().view(H, G, 1)], 2)
            w = torch.softmax(z, 2)[..., :len(p)]
            outs.append(torch.matmul(w, v.transpose(0, 1).contiguous()).reshape(Hq * D))
        return torch.stack(outs)
    cu = s["cu"].cpu().numpy()
    if c["kind"] == "prefill":
        outs, h = [], c["start"]
        for b in range(c["B"]):
            r = slice(int(cu[b]), int(cu[b + 1]))
            L = r.stop - r.start
            p = np.arange(h)
            if c["window"]:
                p = p[(p < c["kept"]) | (p > h - c["window"])]
            k, v = _exact_rows(s, b, p)
            k, v = (torch.cat([x, y[r].double().view(L, H, D)]) for x, y in ((k, s["kp"]), (v, s["vp"])))
            t = torch.from_numpy(np.concatenate([p, h + np.arange(L)])).cuda()
            at = torch.arange(h, h + L, device="cuda")
            ok = t[None] <= at[:, None]
            if c["window"]:
                ok &= (t[None] < c["kept"]) | (at[:, None] - t[None] < c["window"])
            q = _turn(qkv[r, :Hq], s["cos"][at], s["sin"][at])
            outs.append(_exact_attention(q, k, v, ok, s.get("sinks")))
        return torch.cat(outs)
    # append: sequence by sequence, block by block
    start, lens = s["start"].cpu().numpy(), s["lens"].cpu().numpy()
    f8 = c["fmt"] == FP8B
    vals = torch.from_numpy(_e4m3_values()).cuda()
    pools = [vals[x.long()] if f8 else x.double() for x in (s["k"], s["v"])]
    sc = s["sc"].double() if f8 else None
    table = s["table"].cpu().numpy()
    order = torch.tensor(sorted(x for x in _e4m3_values() if x == x and (x != 0 or math.copysign(1, x) > 0)),
                         dtype=torch.float64, device="cuda")

    def nearest(x):
        """The e4m3 value nearest to x, ties to the even mantissa."""
        hi = torch.searchsorted(order, x.contiguous()).clamp(1, len(order) - 1)
        lo_v, hi_v = order[hi - 1], order[hi]
        low = (x - lo_v < hi_v - x)
        tie = (x - lo_v) == (hi_v - x)
        _, e = torch.frexp(lo_v.abs().clamp(min=2.0 ** -6))
        even = torch.remainder(lo_v / torch.exp2((e - 4).double()), 2) == 0
        return torch.where(low | (tie & even), lo_v, hi_v)

    packs = []
    for b in range(c["B"]):
        r = slice(int(cu[b]), int(cu[b + 1]))
        at = torch.arange(int(start[b]), int(lens[b]), device="cuda")
        kn = _turn(qkv[r, Hq:Hq + H], s["cos"][at], s["sin"][at])
        vn = qkv[r, Hq + H:]
        packs.append((kn.reshape(-1, H, D), vn.reshape(-1, H, D)))
        kb, ring = c["kept"] // BT, c["window"] // BT + 1
        for j in range(int(start[b]) // BT, (int(lens[b]) - 1) // BT + 1):
            slot = j
            if c["window"]:
                if j >= kb and j + ring <= (int(lens[b]) - 1) // BT:
                    continue
                slot = j if j < kb else kb + (j - kb) % ring
            phys = int(table[b, slot])
            lo, hi = max(int(start[b]), j * BT), min(int(lens[b]), j * BT + BT)
            for i, (pool, xs, place) in enumerate(zip(pools, (kn, vn), _places(c["fmt"]))):
                cell = torch.from_numpy(place).cuda()
                was = pool[phys][:, cell]                                 # [H, 16, 64]
                x = xs[lo - int(start[b]):hi - int(start[b])].transpose(0, 1)
                n_old = lo - j * BT
                now = was.clone() if n_old else torch.zeros_like(was)
                if not f8:
                    now[:, n_old:n_old + x.shape[1]] = x
                else:
                    a = x.abs().amax((1, 2))
                    sn = torch.where(a > 0, torch.exp2(torch.ceil(torch.log2(a / 448))), torch.zeros_like(a))
                    if n_old:
                        sn = torch.maximum(sn, sc[phys, :, i])
                        now[:, :n_old] = nearest(was[:, :n_old] * (sc[phys, :, i] / sn)[:, None, None])
                    now[:, n_old:n_old + x.shape[1]] = nearest(x / sn[:, None, None])
                    sc[phys, :, i] = sn
                pool[phys, :, cell.reshape(-1)] = now.reshape(H, -1)
    out = {"k": pools[0], "v": pools[1]}
    if f8:
        out["sc"] = sc
    if c["pack"]:
        out.update(kp=torch.cat([p[0] for p in packs]), vp=torch.cat([p[1] for p in packs]))
    return out
