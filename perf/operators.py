"""Measured cases of the paged-cache operators beside plain decode.

Four operators of a paged KV cache, each in its plain form (elementary torch
operations in 32 bits, rounded once at the end) and as the package's call:

  append   new K/V rows into a cache held in 8 bits (e4m3) with one scale for each
           block of tokens and KV head
  attend   paged attention over such a cache, or over a 16/32-bit one with changed
           scores: a tanh cap, a distance bias, a sliding window, a document mask,
           a prefix mask
  copy, beam, compact
           pages of a cache: copied, freed / forked / reserved in one step of a
           beam search, and moved together to the low end of the pool

Scores: s = scale * q.k; capped c * tanh(s / c); minus slope_h * |i - j| for the
query at position i and the key at j; key j is visible to i when
first_i <= j, i - j < window, and j <= i or j < prefix.  A row that sees nothing is 0.

Eight-bit cache: value = code * scale, scale[block, head] = 2^e with the smallest
e >= -100 for which the block's largest finite |value| is at most 448 * 2^e.  A write
at offset 0 of a block starts it anew; a later write raises the scale where its
values need it, and the block's other codes are rounded again to the new scale.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

F8 = torch.float8_e4m3fn
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ---------------------------------------------------------------- the cases

def _append(name, dtype, B, q, Hkv, D, bs, lo, hi):
    return {"name": name, "op": "append", "dtype": dtype, "B": B, "q": q, "Hkv": Hkv, "D": D, "bs": bs, "lo": lo,
            "hi": hi}


def _attend(name, dtype, B, q, Hq, Hkv, D, bs, lo, hi, cache="fp8", append=False, softcap=0.0, window=0, alibi=False,
            document=0, prefix=0):
    return {"name": name, "op": "attend", "dtype": dtype, "B": B, "q": q, "Hq": Hq, "Hkv": Hkv, "D": D, "bs": bs,
            "lo": lo, "hi": hi, "cache": cache, "append": append, "softcap": softcap, "window": window, "alibi": alibi,
            "document": document, "prefix": prefix}


def _pages(name, op, pages, layers, Hkv, D, bs, n):
    return {"name": name, "op": op, "pages": pages, "layers": layers, "Hkv": Hkv, "D": D, "bs": bs, "n": n}


def listed():
    return [
        # one token for each of 64 sequences of a small model: all latency
        _append("append8 64 rows", "fp16", 64, 1, 2, 64, 16, 128, 2048),
        # a prefill chunk of eight prompts, of odd length, starting inside blocks
        _append("append8 chunk 8x509", "bf16", 8, 509, 8, 128, 16, 1, 4096),
        # one long-context sequence: split over the whole GPU or slow
        _attend("attend8 1 row 32k", "bf16", 1, 1, 32, 8, 128, 16, 32701, 32701),
        # a decode step of a small model, the new token appended in the same call
        _attend("attend8+append 64 rows", "fp16", 64, 1, 14, 2, 64, 16, 128, 2048, append=True),
        # a full decode batch of an 8B-shaped model, ragged
        _attend("attend8 192 rows", "bf16", 192, 1, 32, 8, 128, 16, 256, 8192),
        # speculative verification, four tokens a row
        _attend("attend8 verify 96x4", "bf16", 96, 4, 32, 8, 128, 16, 16, 2048),
        # sliding-window decode with capped scores
        _attend("window+cap 128 rows", "bf16", 128, 1, 32, 8, 128, 16, 256, 8192, cache="same", softcap=50.0,
                window=1024),
        # distance bias with a prefix, 32 bits, short rows down to one token
        _attend("bias fp32 4 rows", "fp32", 4, 1, 8, 2, 64, 16, 1, 512, cache="same", alibi=True, prefix=5),
        # packed documents and a bidirectional prefix in a prefill chunk
        _attend("documents chunk 4x1021", "bf16", 4, 1021, 32, 8, 128, 16, 64, 2048, cache="same", document=700,
                prefix=96),
        # copy-on-write of a few pages of a 4-layer pool (K and V)
        _pages("copy 48 pages", "copy", 512, 4, 8, 128, 16, 48),
        # one beam-search step: dead beams freed, live ones forked, a token reserved
        _pages("beam 64 forks", "beam", 6000, 2, 8, 128, 16, 64),
        # a fragmented pool moved together
        _pages("compact 4096 pages", "compact", 4096, 4, 8, 128, 16, 2458),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    heads = [(14, 2, 64), (32, 8, 128), (16, 4, 128), (8, 8, 64), (12, 4, 96), (16, 1, 128), (8, 2, 32)]
    op = rng.choice(["append", "attend", "attend", "scored", "scored", "copy", "beam", "compact"])
    Hq, Hkv, D = rng.choice(heads)
    bs = rng.choice([8, 16, 16, 32, 64])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "append":
        B, q = rng.choice([(_log(rng, 1, 300), 1), (_log(rng, 1, 64), rng.randint(2, 9)),
                           (rng.randint(1, 8), _log(rng, 17, 512))])
        c = _append("", dtype, B, q, Hkv, D, bs, 1, _log(rng, 16, 4096))
    elif op == "attend":
        B, q, hi = rng.choice([(1, 1, _log(rng, 16, 32768)), (_log(rng, 2, 160), 1, _log(rng, 64, 6000)),
                               (_log(rng, 2, 64), rng.randint(2, 8), _log(rng, 64, 2048))])
        c = _attend("", dtype, B, q, Hq, Hkv, D, bs, max(1, hi // 32), hi, append=rng.random() < 0.3 and B * hi < 2e5)
    elif op == "scored":
        B, q, hi = rng.choice([(_log(rng, 1, 128), 1, _log(rng, 64, 6000)), (_log(rng, 1, 32), rng.randint(2, 8), 2048),
                               (rng.randint(1, 3), _log(rng, 32, 800), 1500)])
        # any mixture of the five is allowed
        c = _attend("", rng.choice(["bf16", "fp16", "fp32"]), B, q, Hq, Hkv, D, bs, max(1, hi // 32), hi, cache="same",
                    softcap=rng.choice([0.0, 20.0, 50.0]), window=rng.choice([0, 0, _log(rng, 1, 2048)]),
                    alibi=rng.random() < 0.4, document=rng.choice([0, 0, _log(rng, 30, 900)]),
                    prefix=rng.choice([0, 0, _log(rng, 1, 300)]))
        if c["dtype"] == "fp32":  # long rows and chunks are a 16-bit path
            c["hi"] = min(c["hi"], 1500)
            c["lo"] = min(c["lo"], c["hi"])
            if c["q"] > 8:
                c["dtype"] = "bf16"
        if c["dtype"] != "fp32" and c["D"] % 16 == 0 and rng.random() < 0.3:
            c["cache"] = "fp8"
    else:
        layers = rng.randint(1, 4)
        pages = min(_log(rng, 64, 4096), int(1.2e9 / (4 * layers * Hkv * bs * D)))
        n = {"copy": rng.randint(1, pages // 4), "beam": rng.randint(1, max(1, min(96, pages // 48))),
             "compact": rng.randint(1, pages - 1)}[op]
        c = _pages("", op, pages, layers, Hkv, D, bs, n)
    del c["name"]
    return c


# ---------------------------------------------------------------- lengths and masks of a case

def _lens(c):
    """Tokens cached before the step, one row each: the quantiles of a log-uniform
    distribution (the same for every seed, which only permutes them)."""
    u = (np.arange(c["B"]) + 0.5) / c["B"]
    return np.clip(np.round(np.exp(np.log(c["lo"]) + u * (np.log(c["hi"]) - np.log(c["lo"])))), c["lo"],
                   c["hi"]).astype(np.int64)


def _interval(c, lens):
    """First and one past the last visible key of every query token [B, q] (numpy)."""
    pos = lens[:, None] + np.arange(c["q"])[None, :]
    first = np.zeros_like(pos)
    if c["document"]:
        first = pos // c["document"] * c["document"]
    if c["window"]:
        first = np.maximum(first, pos - c["window"] + 1)
    end = pos + 1
    if c["prefix"]:
        end = np.maximum(end, np.minimum(c["prefix"], lens[:, None] + c["q"]))
    return first, end


def work(c):
    if c["op"] == "append":
        n = c["B"] * c["q"] * c["Hkv"] * c["D"]
        blocks = sum((l + c["q"] - 1) // c["bs"] - l // c["bs"] + 1 for l in _lens(c).tolist())
        return {"bytes": 2 * n * (BYTES[c["dtype"]] + 1) + 2 * blocks * c["Hkv"] * 4 + c["B"] * 8, "flops": 4 * n}
    if c["op"] == "attend":
        lens = _lens(c)
        first, end = _interval(c, lens)
        pairs = int(np.maximum(end - first, 0).sum())
        seen = int((end.max(1) - first.min(1)).sum())
        e = 1 if c["cache"] == "fp8" else BYTES[c["dtype"]]
        b = 2 * seen * c["Hkv"] * c["D"] * e + 2 * c["B"] * c["q"] * c["Hq"] * c["D"] * BYTES[c["dtype"]]
        b += seen // c["bs"] * (4 + (2 * 4 * c["Hkv"] if c["cache"] == "fp8" else 0)) + c["B"] * 4
        if c["append"]:
            b += 2 * c["B"] * c["q"] * c["Hkv"] * c["D"] * (BYTES[c["dtype"]] + e)
        return {"bytes": b, "flops": 4 * pairs * c["Hq"] * c["D"]}
    page = 2 * c["layers"] * c["Hkv"] * c["bs"] * c["D"] * 2
    if c["op"] == "copy":
        moved = c["n"]
    elif c["op"] == "beam":
        moved = sum(int(l) % c["bs"] != 0 for l in _beam_lens(c))
    else:
        live = _live(c, np.random.default_rng(c["pages"] * 7 + c["n"]))
        moved = int((live >= c["n"]).sum())
    return {"bytes": 2 * moved * page + c["pages"] * 4, "flops": 0}


def _beam_lens(c):
    """Tokens of each live beam: short to long, within the pool."""
    most = c["pages"] * c["bs"] // (2 * c["n"])
    return np.maximum(1, np.round(np.linspace(1, max(1, most), c["n"]))).astype(np.int64)


def _live(c, rng):
    return np.sort(rng.permutation(c["pages"])[: c["n"]])


# ---------------------------------------------------------------- inputs

def _quantise(x):
    """[nb, H, bs, D] float values -> codes and power-of-two scales [nb, H]."""
    amax = x.abs().amax(dim=(2, 3)).clamp_min(2.0**-90)
    m, e = torch.frexp(amax)  # amax = m * 2^e, 0.5 <= m < 1; 448 = 0.875 * 2^9
    e = (e - 9 + (m > 0.875).to(e.dtype)).to(torch.float32)
    scale = torch.exp2(e)
    return (x / scale[:, :, None, None]).to(F8), scale


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    dev = "cuda"
    if c["op"] in ("copy", "beam", "compact"):
        return _prepare_pages(c, g, rng)
    B, q, Hkv, D, bs = c["B"], c["q"], c["Hkv"], c["D"], c["bs"]
    dt = TYPES[c["dtype"]]
    lens = rng.permutation(_lens(c))
    counts = (lens + q + bs - 1) // bs
    M = int(counts.max())
    nb = int(counts.sum()) + 3
    perm = rng.permutation(nb).astype(np.int32)
    bt = np.zeros((B, M), dtype=np.int32)
    ends = np.cumsum(counts)
    for b in range(B):
        bt[b, : counts[b]] = perm[ends[b] - counts[b]: ends[b]]
    st = {"case": c, "bt": torch.from_numpy(bt).to(dev), "lens": torch.from_numpy(lens.astype(np.int32)).to(dev)}
    if c["op"] == "append" or c["append"]:
        # rows of different size: some raise their block's scale, most do not
        size = torch.exp2(torch.randint(-2, 3, (B, 1, q, 1), generator=g, device=dev).float())
        st["key"] = (torch.randn(B, Hkv, q, D, generator=g, device=dev) * 0.5 * size).to(dt)
        st["value"] = (torch.randn(B, Hkv, q, D, generator=g, device=dev) * 0.5 * size).to(dt)
    eight = c["op"] == "append" or c["cache"] == "fp8"
    for name in ("k", "v"):
        x = torch.randn(nb, Hkv, bs, D, generator=g, device=dev) * 0.5
        if eight:
            x *= torch.exp2(torch.randint(-2, 2, (nb, Hkv, 1, 1), generator=g, device=dev).float())
            st[name + "c"], st[name + "s"] = _quantise(x)
        else:
            st[name + "c"] = x.to(dt)
    if c["op"] == "append":
        return st
    st["q"] = (torch.randn(B, c["Hq"], q, D, generator=g, device=dev)).to(dt)
    st["scale"] = D**-0.5
    pos = lens[:, None] + np.arange(q)[None, :]
    st["first"] = (torch.from_numpy((pos // c["document"] * c["document"]).astype(np.int32)).to(dev)
                   if c["document"] else None)
    st["prefix"] = torch.full((B,), c["prefix"], dtype=torch.int32, device=dev) if c["prefix"] else None
    st["slopes"] = (torch.exp2(-8.0 * torch.arange(1, c["Hq"] + 1, device=dev, dtype=torch.float32) / c["Hq"])
                    if c["alibi"] else None)
    if own and (c["softcap"] or c["window"] or c["alibi"] or c["document"] or c["prefix"]):
        from llm_serving_runtime_b200 import ScoreModifiers

        st["mods"] = ScoreModifiers(softcap=c["softcap"], window=c["window"], alibi_slopes=st["slopes"],
                                    key_starts=st["first"], prefix_lens=st["prefix"])
    return st


def _prepare_pages(c, g, rng):
    P, n, bs = c["pages"], c["n"], c["bs"]
    shape = (P, c["layers"], c["Hkv"], bs, c["D"])
    st = {"case": c, "caches": [torch.randn(shape, generator=g, device="cuda", dtype=torch.bfloat16)
                                for _ in range(2)]}
    if c["op"] == "copy":
        ids = rng.permutation(P)
        st["src"] = torch.from_numpy(ids[:n].astype(np.int32)).cuda()
        st["dst"] = torch.from_numpy(ids[n: 2 * n].astype(np.int32)).cuda()
        return st
    if c["op"] == "beam":
        # slots 0..n-1: live beams; n..2n-1: their children of the step before (dead now)
        lens = rng.permutation(_beam_lens(c))
        counts = (lens + bs - 1) // bs
        M = int(counts.max()) + 1
        tables = np.full((2 * n, M), -1, dtype=np.int32)
        refs = np.zeros(P, dtype=np.int32)
        order = rng.permutation(P)
        at = 0
        for b in range(n):
            tables[b, : counts[b]] = order[at: at + counts[b]]
            at += counts[b]
            shared = lens[b] // bs  # the dead child still holds its parent's full pages
            tables[n + b, :shared] = tables[b, :shared]
        held = tables[tables >= 0]
        np.add.at(refs, held, 1)
        all_lens = np.concatenate([lens, lens // bs * bs])
        st["parents"] = torch.arange(n, dtype=torch.int32, device="cuda")
        st["children"] = torch.arange(n, 2 * n, dtype=torch.int32, device="cuda")
        st["all"] = torch.arange(2 * n, dtype=torch.int32, device="cuda")
        st["one"] = torch.ones(2 * n, dtype=torch.int32, device="cuda")
    else:
        fixed = np.random.default_rng(P * 7 + n)
        live = rng.permutation(_live(c, fixed))
        S = max(1, n // 40)
        cuts = np.sort(fixed.integers(0, n + 1, S - 1))
        counts = np.diff(np.concatenate([[0], cuts, [n]]))
        M = max(1, int(counts.max()))
        tables = np.full((S, M), -1, dtype=np.int32)
        at = 0
        for b in range(S):
            tables[b, : counts[b]] = live[at: at + counts[b]]
            at += counts[b]
        refs = np.zeros(P, dtype=np.int32)
        refs[live] = 1
        all_lens = counts * bs
    st["start"] = [torch.from_numpy(x).cuda() for x in (tables, all_lens.astype(np.int32), refs)]
    st["now"] = [x.clone() for x in st["start"]]
    if own:
        from llm_serving_runtime_b200 import DevicePages

        st["pages"] = DevicePages.from_tensors(*st["now"], block_size=bs)
    return st


# ---------------------------------------------------------------- one pass

def run(st):
    c = st["case"]
    return {"append": _run_append, "attend": _run_attend, "copy": _run_copy, "beam": _run_beam,
            "compact": _run_compact}[c["op"]](st, c)


def _run_append(st, c):
    if own:
        from llm_serving_runtime_b200 import kv_append

        kv_append(st["key"], st["value"], st["kc"], st["vc"], block_tables=st["bt"], positions=st["lens"],
                  key_scales=st["ks"], value_scales=st["vs"])
    else:
        _plain_append(st, c)
    return [st["kc"], st["vc"], st["ks"], st["vs"]]


def _plain_append(st, c):
    B, q, Hkv, D, bs = c["B"], c["q"], c["Hkv"], c["D"], c["bs"]
    nl = (q + bs - 2) // bs + 1  # blocks a row's tokens can touch
    lens, bt = st["lens"].long(), st["bt"].long()
    first = lens // bs
    logical = first[:, None] + torch.arange(nl, device=lens.device)
    touched = logical <= ((lens + q - 1) // bs)[:, None]
    blocks = torch.gather(bt, 1, logical.clamp_max(bt.shape[1] - 1))  # [B, nl]
    # token of each (row, touched block, offset): t = position - length
    pos = logical[:, :, None] * bs + torch.arange(bs, device=lens.device)
    t = pos - lens[:, None, None]
    new = (t >= 0) & (t < q) & touched[:, :, None]  # [B, nl, bs]
    fresh = (logical * bs >= lens[:, None]) & touched  # offset 0 is written: the block starts anew
    for rows, codes, scales in ((st["key"], st["kc"], st["ks"]), (st["value"], st["vc"], st["vs"])):
        x = rows.float().transpose(1, 2)  # [B, q, Hkv, D]
        at = t.clamp(0, q - 1).reshape(B, nl * bs, 1, 1).expand(-1, -1, Hkv, D)
        x = torch.gather(x, 1, at).reshape(B, nl, bs, Hkv, D).permute(0, 1, 3, 2, 4)  # [B, nl, Hkv, bs, D]
        mine = new[:, :, None, :, None]
        size = torch.where(mine & torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(dim=(3, 4))
        m, e = torch.frexp(size.clamp_min(2.0**-95))
        need = torch.exp2((e - 9 + (m > 0.875).to(e.dtype)).clamp_min(-100).float())
        need = torch.where(size > 448 * 2.0**-100, need, torch.full_like(need, 2.0**-100))
        old = scales[blocks]  # [B, nl, Hkv]
        old = torch.where(fresh[:, :, None], torch.zeros_like(old), old)
        scale = torch.maximum(old, need)
        held = codes[blocks].float()  # [B, nl, Hkv, bs, D]
        ratio = torch.where(fresh[:, :, None], torch.ones_like(old), old / scale)
        held = (held * ratio[..., None, None]).to(F8)
        fits = (x / scale[..., None, None]).clamp(-448, 448).to(F8)
        put = torch.where(mine, fits.float(), held.float()).to(F8)
        # rows that touch fewer blocks write their last one again: the same values
        last = touched.long().sum(1, keepdim=True) - 1
        pick = torch.minimum(torch.arange(nl, device=lens.device)[None, :].expand(B, nl), last)
        ids = torch.gather(blocks, 1, pick)
        put = torch.gather(put.view(torch.uint8), 1, pick[:, :, None, None, None].expand_as(put)).view(F8)
        scale = torch.gather(scale, 1, pick[:, :, None].expand_as(scale))
        codes.view(torch.uint8)[ids] = put.view(torch.uint8)
        scales[ids] = scale


def _run_attend(st, c):
    eight = c["cache"] == "fp8"
    if own:
        from llm_serving_runtime_b200 import paged_attention_decode

        more = {}
        if eight:
            more.update(key_scales=st["ks"], value_scales=st["vs"])
        if "mods" in st:
            more.update(score_modifiers=st["mods"])
        if c["append"]:
            more.update(key=st["key"], value=st["value"])
        out = paged_attention_decode(st["q"], st["kc"], st["vc"], st["bt"], st["lens"], st["scale"], **more)
        return [out, st["kc"], st["vc"], st["ks"], st["vs"]] if c["append"] else out
    if c["append"]:
        _plain_append(st, c)
    out = _plain_attend(st, c)
    return [out, st["kc"], st["vc"], st["ks"], st["vs"]] if c["append"] else out


def _plain_attend(st, c):
    B, q, Hq, Hkv, D, bs = c["B"], c["q"], c["Hq"], c["Hkv"], c["D"], c["bs"]
    G, bt = Hq // Hkv, st["bt"].long()
    T = bt.shape[1] * bs
    kv = []
    for name in ("k", "v"):
        x = st[name + "c"][bt].float()  # [B, M, Hkv, bs, D]
        if c["cache"] == "fp8":
            x *= st[name + "s"][bt][..., None, None]
        kv.append(x.permute(0, 2, 1, 3, 4).reshape(B, Hkv, T, D))
    j = torch.arange(T, device=bt.device)
    L = st["lens"].long() + q
    i = st["lens"].long()[:, None] + torch.arange(q, device=bt.device)  # [B, q]
    kv[1].masked_fill_((j[None, :] >= L[:, None])[:, None, :, None], 0)
    s = torch.matmul(st["q"].float().reshape(B, Hkv, G * q, D), kv[0].transpose(2, 3)).mul_(st["scale"])
    s = s.reshape(B, Hkv, G, q, T)
    if c["softcap"]:
        s = torch.tanh(s / c["softcap"]).mul_(c["softcap"])
    far = i[:, :, None] - j  # [B, q, T]
    if st["slopes"] is not None:
        s -= st["slopes"].reshape(1, Hkv, G, 1, 1) * far.abs().float()[:, None, None]
    seen = far >= 0
    if st["prefix"] is not None:
        seen = seen | (j < torch.minimum(st["prefix"].long(), L)[:, None])[:, None, :]
    if st["first"] is not None:
        seen = seen & (j >= st["first"].long()[:, :, None])
    if c["window"]:
        seen = seen & (far < c["window"])
    s.masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True).clamp_min(-3e38)
    p = torch.exp_(s.sub_(top))
    total = p.sum(-1)
    o = torch.matmul(p.reshape(B, Hkv, G * q, T), kv[1]).reshape(B, Hkv, G, q, D)
    o = o / torch.where(total > 0, total, torch.ones_like(total))[..., None]
    return o.reshape(B, Hq, q, D).to(TYPES[c["dtype"]])


def _run_copy(st, c):
    if own:
        from llm_serving_runtime_b200 import copy_pages

        copy_pages(st["caches"], st["src"], st["dst"])
    else:
        src, dst = st["src"].long(), st["dst"].long()
        for x in st["caches"]:
            x[dst] = x[src]
    return _bits(st["caches"])


def _bits(caches):
    """The caches' bits: pages are moved, not computed."""
    return [x.view(torch.int16) for x in caches]


def _restore(st):
    for x, x0 in zip(st["now"], st["start"]):
        x.copy_(x0)


def _run_beam(st, c):
    _restore(st)
    if own:
        pages = st["pages"]
        pages.free(st["children"])
        pages.fork(st["parents"], st["children"], st["caches"])
        pages.reserve(st["all"], st["one"])
        return [*st["now"], *_bits(st["caches"])]
    tables, lens, refs = st["now"]
    bs, M = c["bs"], tables.shape[1]
    j = torch.arange(M, device="cuda")
    parents, children = st["parents"].long(), st["children"].long()
    # freed: one holder fewer for every page of the rows
    rows = tables[children].reshape(-1).long()
    refs.index_add_(0, rows.clamp_min(0), -(rows >= 0).to(torch.int32))
    tables[children] = -1
    lens[children] = 0
    # forked: full pages shared, the page in use copied to the lowest free one
    have, full = lens[parents], lens[parents] // bs
    tail = have % bs != 0
    free = torch.argsort((refs != 0).to(torch.int8), stable=True)
    mine = free[(torch.cumsum(tail, 0) - 1).clamp_min(0)]
    row = tables[parents]
    shared = (j[None, :] < full[:, None])
    at_tail = tail[:, None] & (j[None, :] == full[:, None])
    held = torch.where(shared, row, torch.zeros_like(row)).reshape(-1).long()
    refs.index_add_(0, held, shared.reshape(-1).to(torch.int32))
    refs.index_add_(0, mine, tail.to(torch.int32))
    tables[children] = torch.where(shared, row, torch.where(at_tail, mine[:, None].to(torch.int32),
                                                            torch.full_like(row, -1)))
    lens[children] = have
    old = torch.gather(row, 1, full.long().clamp_max(M - 1)[:, None])[:, 0].long()
    src, dst = old[tail], mine[tail]
    for x in st["caches"]:
        x[dst] = x[src]
    # reserved: room for one more token of every row
    rows = st["all"].long()
    have = lens[rows]
    more = (have + st["one"] + bs - 1) // bs - (have + bs - 1) // bs
    free = torch.argsort((refs != 0).to(torch.int8), stable=True)
    at = torch.cumsum(more, 0) - more
    mine = free[at.clamp_max(free.numel() - 1)]
    put = (j[None, :] == ((have + bs - 1) // bs)[:, None]) & (more > 0)[:, None]
    tables[rows] = torch.where(put, mine[:, None].to(torch.int32), tables[rows])
    refs.index_add_(0, mine, (more > 0).to(torch.int32))
    lens[rows] = have + st["one"]
    return [*st["now"], *_bits(st["caches"])]


def _run_compact(st, c):
    _restore(st)
    if own:
        live = st["pages"].compact(st["caches"])
        return [live, *st["now"], *_bits(st["caches"])]
    tables, _, refs = st["now"]
    held = refs > 0
    live = held.sum(dtype=torch.int32).reshape(1)
    ids = torch.arange(refs.numel(), device="cuda")
    src = torch.nonzero(held & (ids >= live)).reshape(-1)
    dst = torch.nonzero(~held & (ids < live)).reshape(-1)
    for x in st["caches"]:
        x[dst] = x[src]
    to = ids.clone()
    to[src] = dst
    tables.copy_(torch.where(tables >= 0, to[tables.clamp_min(0).long()].to(torch.int32), tables))
    refs[dst] = refs[src]
    refs[src] = 0
    return [live, *st["now"], *_bits(st["caches"])]


# ---------------------------------------------------------------- the definitions, in 64 bits

def exact(c, seed):
    """From the definitions, row by row in 64 bits; moved pages are whole values and have none."""
    global own
    before, own = own, False
    try:
        st = prepare(c, seed)
    finally:
        own = before
    if c["op"] not in ("append", "attend"):
        return None
    rows = [int(x) for x in st["lens"].cpu()]
    tables = st["bt"].cpu().numpy()
    state = []
    if c["op"] == "append" or c["append"]:
        state = _exact_append(st, c, rows, tables)
        if c["op"] == "append":
            return state
        for name, x in zip(("kc", "vc", "ks", "vs"), state):
            st[name] = torch.from_numpy(x).cuda()
    out = torch.zeros(c["B"], c["Hq"], c["q"], c["D"], dtype=torch.float64)
    G, bs = c["Hq"] // c["Hkv"], c["bs"]
    first, end = _interval(c, np.array(rows))
    slopes = st["slopes"].double() if st["slopes"] is not None else torch.zeros(c["Hq"], device="cuda").double()
    for b, before_b in enumerate(rows):
        n = before_b + c["q"]
        ids = torch.from_numpy(tables[b, : (n + bs - 1) // bs].astype(np.int64)).cuda()
        k, v = (st[x + "c"][ids].double() for x in "kv")
        if c["cache"] == "fp8":
            k, v = k * st["ks"][ids].double()[:, :, None, None], v * st["vs"][ids].double()[:, :, None, None]
        k, v = (x.transpose(0, 1).reshape(c["Hkv"], -1, c["D"])[:, :n] for x in (k, v))
        query = st["q"][b].double()
        keys = torch.arange(n, device="cuda").double()
        lo = torch.from_numpy(first[b]).cuda()[:, None]
        hi = torch.from_numpy(end[b]).cuda()[:, None]
        hidden = (keys < lo) | (keys >= hi)  # [q, n]
        far = (before_b + torch.arange(c["q"], device="cuda").double()[:, None] - keys).abs()
        for h in range(c["Hq"]):
            s = query[h] @ k[h // G].T * st["scale"]
            if c["softcap"]:
                s = c["softcap"] * torch.tanh(s / c["softcap"])
            w = torch.softmax((s - slopes[h] * far).masked_fill(hidden, -math.inf), -1)
            out[b, h] = torch.nan_to_num(w @ v[h // G], nan=0.0).cpu()
    return [out, *state] if c["append"] else out


def _e4m3(x):
    """The nearest e4m3 value (ties to even) of each float64, saturating."""
    a = np.minimum(np.abs(x), 448.0)
    _, e = np.frexp(a)
    step = np.exp2(np.maximum(e - 1, -6) - 3.0)  # 3 bits behind the leading one, least normal 2^-6
    return np.copysign(np.minimum(np.rint(a / step) * step, 448.0), x)


def _exact_append(st, c, rows, tables):
    got = []
    for new, codes, scales in ((st["key"], st["kc"], st["ks"]), (st["value"], st["vc"], st["vs"])):
        new = new.double().cpu().numpy()
        codes, scales = codes.double().cpu().numpy().copy(), scales.double().cpu().numpy().copy()
        for b, at in enumerate(rows):
            for lb in range(at // c["bs"], (at + c["q"] - 1) // c["bs"] + 1):
                blk = tables[b, lb]
                o0, o1 = max(0, at - lb * c["bs"]), min(c["bs"], at + c["q"] - lb * c["bs"])
                x = new[b, :, lb * c["bs"] + o0 - at: lb * c["bs"] + o1 - at]  # [Hkv, tokens, D]
                need = np.array([max(-100, math.ceil(math.log2(a / 448))) if a else -100
                                 for a in np.abs(x).max(axis=(1, 2))])
                need = np.exp2(need.astype(np.float64))
                if o0 > 0:
                    scale = np.maximum(scales[blk], need)
                    codes[blk] = _e4m3(codes[blk] * (scales[blk] / scale)[:, None, None])
                else:
                    scale = need
                scales[blk] = scale
                codes[blk, :, o0:o1] = _e4m3(x / scale[:, None, None])
        got += [codes, scales]
    return [got[0], got[2], got[1], got[3]]
