"""Plain 64-bit forms of the extended cache operators, and the error bars the
kernels' arithmetic allows against them.

``attend64`` is the definition of changed-score attention over a cache of values;
``append8`` the definition of the 8-bit append, on numpy arrays; ``Pages`` the
sequence table in plain Python.
"""

from __future__ import annotations

import math

import numpy as np
import torch

F8 = torch.float8_e4m3fn


# ---- attention -------------------------------------------------------------------

def visible(lens, q_len, window=0, key_starts=None, prefix_lens=None):
    """Per row a bool [q_len, L] of the keys each query token sees (L = lens + q_len)."""
    out = []
    for b, n in enumerate(lens):
        L = int(n) + q_len
        i = (L - q_len + np.arange(q_len))[:, None]
        j = np.arange(max(L, 0))[None, :]
        see = j <= i
        if prefix_lens is not None:
            see = see | (j < int(prefix_lens[b]))
        if key_starts is not None:
            ks = np.asarray(key_starts[b]).reshape(-1)
            see = see & (j >= (np.full(q_len, ks[0]) if ks.size == 1 else ks)[:, None])
        if window:
            see = see & (i - j < window)
        out.append(see & (i >= 0))
    return out


def attend64(query, key_cache, value_cache, tables, lens, scale, *, key_scales=None, value_scales=None, softcap=0.0,
             window=0, alibi_slopes=None, key_starts=None, prefix_lens=None):
    """(output, bar) in float64, CPU.  The bar is what the kernels' roundings allow:

    * the output's own rounding, eps/2 of the value (none beyond fp32 arithmetic for fp32);
    * weights rounded before P.V: 2^-11 (fp16, and every 8-bit cache), 2^-16 (bf16
      keeps a second part), of sum_j w_j |v_j|; 8-bit caches: the largest weighted
      scale w_j vs_j is at 2^14 there, fp16's least step is 2^-24, so a weight far
      below is off by at most 2^-25, 2^-39 of the largest, times its code;
    * scores: products of D terms summed in fp32 (tensor cores may truncate: 2^-23 a
      step), the cap (2^-21 of it), the exponent's argument and ex2 (2^-21): an
      error d of a score moves its weight by d, and weights enter twice (sum, norm);
    * P.V summed in fp32 over n / 16 steps of 16.
    """
    query, tables, lens = query.cpu(), tables.cpu().long(), lens.cpu().long()
    dt = query.dtype
    q = query.double()
    k, v = key_cache.cpu().to(torch.float64), value_cache.cpu().to(torch.float64)
    if key_scales is not None:
        k = k * key_scales.cpu().double()[:, :, None, None]
        v = v * value_scales.cpu().double()[:, :, None, None]
    B, Hq, q_len, D = q.shape
    _, Hkv, bs, _ = k.shape
    G = Hq // Hkv
    sees = visible(lens.tolist(), q_len, window, None if key_starts is None else key_starts.cpu().numpy(),
                   None if prefix_lens is None else prefix_lens.cpu().numpy())
    out = torch.zeros(B, Hq, q_len, D, dtype=torch.float64)
    bar = torch.zeros_like(out)
    weight_eps = {torch.float32: 0.0, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-16}[dt]
    if key_scales is not None:
        weight_eps = 2.0**-11
    out_eps = 2.0**-23 if dt == torch.float32 else torch.finfo(dt).eps / 2
    for b in range(B):
        L = int(lens[b]) + q_len
        see = torch.from_numpy(sees[b])
        cols = torch.nonzero(see.any(0)).reshape(-1)
        if cols.numel() == 0:
            continue
        # only keys that some token sees are looked at: tables may hold anything elsewhere
        kb = k[tables[b, cols // bs], :, cols % bs]  # [n, Hkv, D]
        vb = v[tables[b, cols // bs], :, cols % bs]
        see = see[:, cols]
        far = ((L - q_len + torch.arange(q_len))[:, None] - cols[None, :]).abs().double()
        for h in range(Hq):
            kk, vv = kb[:, h // G], vb[:, h // G]
            s = q[b, h] @ kk.T * scale
            size = q[b, h].abs() @ kk.abs().T * abs(scale)
            d = (D + 16) * 2.0**-23 * size + 2.0**-20
            if softcap:
                s = softcap * torch.tanh(s / softcap)
                d = d + softcap * 2.0**-21
            if alibi_slopes is not None:
                bias = float(alibi_slopes[h]) * far
                s = s - bias
                d = d + bias * 2.0**-22
            for t in range(q_len):
                on = see[t]
                if not bool(on.any()):
                    continue
                st, vt = s[t][on], vv[on]
                w = torch.softmax(st, 0)
                out[b, h, t] = w @ vt
                n = int(on.sum())
                slack = weight_eps + 2 * float(d[t][on].max()) + (n / 16 + 32) * 2.0**-23
                if key_scales is not None:
                    vs = value_scales.cpu().double()[tables[b, cols // bs], h // G][on]
                    codes = value_cache.cpu().to(torch.float64)[tables[b, cols // bs], h // G, cols % bs][on].abs()
                    bar[b, h, t] = 2.0**-39 * (w * vs).max() * codes.sum(0)
                bar[b, h, t] += (w @ vt.abs()) * slack + out[b, h, t].abs() * out_eps
    # results below the type's normal range are rounded to its least step
    bar += 2.0**-24 if dt == torch.float16 else 1e-38
    return out, bar


def check(out, ref, bar):
    o = out.detach().double().cpu()
    assert torch.equal(torch.isnan(o), torch.isnan(ref)), "NaN in the wrong rows"
    bad = (o - ref).abs() > bar
    bad &= ~torch.isnan(ref)
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} beyond the bar, worst {((o - ref).abs() / bar).nan_to_num().max():.3g} bars"


# ---- the 8-bit append --------------------------------------------------------------

def e4m3(x):
    """The nearest e4m3 value (ties to even) of each float; infinities saturate, NaN stays."""
    x = np.asarray(x, dtype=np.float64)
    a = np.minimum(np.abs(x), 448.0)
    _, e = np.frexp(np.where(np.isnan(a), 0, a))
    step = np.exp2(np.maximum(e - 1, -6) - 3.0)
    return np.copysign(np.minimum(np.rint(a / step) * step, 448.0), x)


def needed_scale(x):
    a = np.abs(x)[np.isfinite(x)]
    top = float(a.max()) if a.size else 0.0
    e = -100
    while top > 448 * 2.0**e:
        e += 1
    return np.float32(2.0**e)


def append8(rows, codes, scales, slots, q_len, bs):
    """rows [B, H, q, D] (float32), codes [nb, H, bs, D] (values), scales [nb, H],
    slots [B * q] (-1: padding): in place.  Returns the error flags of conflicts."""
    B, H, _, D = rows.shape
    nb = codes.shape[0]
    done, flags = set(), 0
    for b in range(B):
        runs = []
        for t in range(q_len):
            s = int(slots[b * q_len + t])
            if s < 0:
                continue
            if not runs or runs[-1][0] != s // bs:
                runs.append((s // bs, {}))
            runs[-1][1][s % bs] = t
        for blk, at in runs:
            if blk in done:
                flags |= 0x40
                continue
            done.add(blk)
            if blk >= nb:
                flags |= 0x4
                continue
            for h in range(H):
                new = np.stack([rows[b, h, t] for t in at.values()])
                need = needed_scale(new)
                held = np.float32(scales[blk, h])
                if 0 in at or not (held > 0 and np.isfinite(held)):
                    held = np.float32(0)
                scale = max(held, need)
                if 0 not in at and scale != held:
                    ratio = np.float32(held / scale)
                    codes[blk, h] = e4m3((codes[blk, h].astype(np.float32) * ratio))
                for o, t in at.items():
                    codes[blk, h, o] = e4m3(rows[b, h, t].astype(np.float32) / scale)
                scales[blk, h] = scale
    return flags


# ---- the sequence table ---------------------------------------------------------------

class Pages:
    """Plain Python form of DevicePages; ``moves`` collects (src, dst) page copies."""

    def __init__(self, tables, lens, refs, bs):
        self.tables = [list(r) for r in tables]
        self.lens, self.refs, self.bs = list(lens), list(refs), bs
        self.flags, self.moves = 0, []

    def pages(self, n):
        return math.ceil(n / self.bs)

    def lowest(self, n):
        return [p for p, r in enumerate(self.refs) if r == 0][:n]

    def free(self, slots):
        for s in dict.fromkeys(slots):
            if s < 0:
                continue
            if s >= len(self.lens):
                self.flags |= 0x80
                continue
            for j, p in enumerate(self.tables[s]):
                if p >= 0:
                    self.refs[p] -= 1
                self.tables[s][j] = -1
            self.lens[s] = 0

    def fork(self, parents, children):
        S = len(self.lens)
        plan, seen = [], set()
        for p, c in zip(parents, children):
            if p < 0 or c < 0:
                continue
            if p >= S or c >= S or c in seen or self.lens[c] or self.tables[c][0] >= 0:
                self.flags |= 0x80
            else:
                plan.append((p, c, self.lens[p]))
            seen.add(c)
        free = self.lowest(len(plan))
        rows = {p: list(self.tables[p]) for p, _, _ in plan}
        for p, c, n in plan:
            full, tail = n // self.bs, n % self.bs
            if tail and not free:
                self.flags |= 0x100
                continue
            for j in range(full):
                self.tables[c][j] = rows[p][j]
                self.refs[rows[p][j]] += 1
            if tail:
                f = free.pop(0)
                self.tables[c][full] = f
                self.refs[f] = 1
                self.moves.append((rows[p][full], f))
            self.lens[c] = n

    def reserve(self, slots, tokens):
        seen, plan, rank = set(), [], 0
        for s, n in zip(slots, tokens):
            if s < 0:
                continue
            if s >= len(self.lens) or s in seen or n < 0:
                self.flags |= 0x80
            elif self.pages(self.lens[s] + n) > len(self.tables[s]):
                self.flags |= 0x2
            else:
                need = self.pages(self.lens[s] + n) - self.pages(self.lens[s])
                plan.append((s, n, rank, need))
                rank += need
            seen.add(s)
        free = self.lowest(rank)
        for s, n, k, need in plan:
            if need and k + need > len(free):
                self.flags |= 0x100
                continue
            old = self.pages(self.lens[s])
            for j in range(need):
                self.tables[s][old + j] = free[k + j]
                self.refs[free[k + j]] = 1
            self.lens[s] += n

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        src = [p for p in range(live, len(self.refs)) if self.refs[p] > 0]
        dst = [p for p in range(live) if self.refs[p] <= 0]
        to = dict(zip(src, dst))
        for s, d in to.items():
            self.refs[d], self.refs[s] = self.refs[s], 0
            self.moves.append((s, d))
        self.tables = [[to.get(p, p) for p in row] for row in self.tables]
        return live
