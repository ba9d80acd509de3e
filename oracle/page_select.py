"""Page means, the choice of pages, attention over chosen pages and rotary positions in
64 bits, on the CPU: the definition that pool_pages, select_pages, selected_attention
and rotary are tested against.  Sums of codes and scores are Python's whole numbers."""
from __future__ import annotations

import math
from fractions import Fraction

import torch

from oracle.paged_kv import PAGE, rows_of


def whole(top: Fraction) -> int:
    """Least e with top <= 127 * 2^e (top > 0)."""
    e = math.floor(math.log2(top)) - 8
    while top > 127 * Fraction(2) ** e:
        e += 1
    return e


def nearest(x: Fraction) -> int:
    return round(x)  # ties to even


def mean_of(codes, scale_byte: int):
    """codes [128, D] (float64 e4m3 values) of a page and head -> (D integers, scale byte)."""
    D = codes.shape[1]
    if scale_byte == 255 or not bool(torch.isfinite(codes).all()):
        return [0] * D, 255
    unit = Fraction(2) ** (scale_byte - 127) / PAGE
    mean = [Fraction(float(x)) * unit for x in codes.sum(0)]  # exact: multiples of 2^-9 below 2^16
    top = max(abs(x) for x in mean)
    e = -127 if top == 0 else min(max(whole(top), -127), 127)
    return [min(max(nearest(x / Fraction(2) ** e), -127), 127) for x in mean], e + 127


def pooled(mean, scale, cache, k_scale, table, lengths, tokens, cu=None):
    """mean [N, H, D] int8 and scale [N, H] bytes after pool_pages (in place); cache as
    paged_kv.from_pages, k_scale bytes; tokens None: every full page."""
    N, H, _ = mean.shape
    B = len(lengths)
    for b, (_, n) in enumerate(rows_of(tokens or 0, B, cu) if B else []):
        L = max(int(lengths[b]), 0)
        held = 0 if tokens is None else max(L - n, 0)
        for j in range(held // PAGE, min(L // PAGE, table.shape[1])):
            page = int(table[b, j])
            if not 0 <= page < N:
                continue
            for h in range(H):
                m, s = mean_of(cache["k"][page, h], int(k_scale[page, h]))
                mean[page, h] = torch.tensor(m, dtype=torch.int8)
                scale[page, h] = s


def integers(q):
    """A group's queries [G, D] as integers of at most 127 times a power of two."""
    if not bool(torch.isfinite(q).all()):
        return torch.zeros(q.shape, dtype=torch.int64)
    top = Fraction(float(q.abs().max()))
    if top == 0:
        return torch.zeros(q.shape, dtype=torch.int64)
    return torch.round(q * 2.0 ** -whole(top)).long()


def selected(q, mean, scale, table, lengths, top, first, recent, cu=None):
    """[T, H, top] int32: the columns of select_pages; q [T, Hq, D] float64."""
    T, Hq, _ = q.shape
    N, H, _ = mean.shape
    G = Hq // H
    out = torch.full((T, H, top), -1, dtype=torch.int32)
    for b, (lo, n) in enumerate(rows_of(T, len(lengths), cu)):
        for i in range(n):
            p = int(lengths[b]) - n + i
            seen = min(p // PAGE + 1, table.shape[1]) if p >= 0 else 0
            if seen <= top:
                for h in range(H):
                    out[lo + i, h, :seen] = torch.arange(seen, dtype=torch.int32)
                continue
            sure = [j for j in range(seen) if j < first or j >= seen - recent]
            rest = [j for j in range(seen) if j not in set(sure)]
            ids = [int(table[b, j]) for j in rest]
            for h in range(H):
                x = integers(q[lo + i, h * G:(h + 1) * G])

                def score(page):
                    if not 0 <= page < N or int(scale[page, h]) == 255:
                        return -math.inf
                    dot = int((x @ mean[page, h].long()).max())
                    return Fraction(dot) * Fraction(2) ** int(scale[page, h])
                best = sorted(zip(rest, map(score, ids)), key=lambda e: (-e[1], e[0]))
                cols = sorted(sure + [j for j, _ in best[:top - first - recent]])
                out[lo + i, h] = torch.tensor(cols, dtype=torch.int32)
    return out


def power(e) -> float:
    """A scale of exponent e; 128 is the byte 255, NaN."""
    return math.nan if int(e) == 128 else 2.0 ** int(e)


def attended(q, cache, table, lengths, columns, cu=None, sm_scale=None):
    """(o, size, logit) as paged_kv.attention gives them, over the listed columns alone."""
    T, Hq, D = q.shape
    N, H = cache["k"].shape[:2]
    scale = sm_scale if sm_scale is not None else 1 / math.sqrt(D)
    o, size, logit = (torch.zeros(T, Hq, D).double(), torch.zeros(T, Hq, D).double(),
                      torch.zeros(T, Hq).double())
    q = q.double()
    for b, (lo, n) in enumerate(rows_of(T, len(lengths), cu)):
        for i in range(n):
            limit = min(int(lengths[b]) - n + i + 1, table.shape[1] * PAGE)
            for c in range(Hq):
                h = c // (Hq // H)
                cols = [j for j in columns[lo + i, h].tolist() if 0 <= j and j * PAGE < limit]
                if not cols:
                    continue
                ks, vs = [], []
                for j in cols:
                    page, m = int(table[b, j]), min(PAGE, limit - j * PAGE)
                    if not 0 <= page < N:
                        ks.append(torch.full((m, D), math.nan).double())
                        vs.append(torch.zeros(m, D).double())
                        continue
                    ks.append(cache["k"][page, h, :m] * power(cache["ke"][page, h]))
                    vs.append(cache["v"][page, h, :, :m].T * power(cache["ve"][page, h]))
                k, v = torch.cat(ks), torch.cat(vs)
                p = torch.softmax(k @ q[lo + i, c] * scale, 0)
                o[lo + i, c] = p @ v
                size[lo + i, c] = p @ v.abs()
                logit[lo + i, c] = (k.abs() @ q[lo + i, c].abs()).max() * scale
    return o, size, logit


def counted(T, Hq, H, D, table, lengths, columns, cu=None, most=0):
    """[T, Hq, D]: what attention over the listed columns of a paged_kv.counting_pool gives."""
    from oracle.paged_kv import lift
    want = torch.zeros(T, Hq, D).double()
    for b, (lo, n) in enumerate(rows_of(T, len(lengths), cu)):
        for i in range(n):
            limit = min(int(lengths[b]) - n + i + 1, table.shape[1] * PAGE)
            for h in range(H):
                w = torch.zeros(D).double()
                for j in columns[lo + i, h].tolist():
                    if 0 <= j and j * PAGE < limit:
                        w[(j + 5 * h) % D] += min(PAGE, limit - j * PAGE) * 2.0 ** lift(j, h, most)
                if w.sum() > 0:
                    want[lo + i, h * (Hq // H):(h + 1) * (Hq // H)] = w / w.sum()
    return want


def rotated(x, turns, gain, positions, pairs, back=False):
    """x [B, S, H, D] turned, float64; turns [R / 2] float64, positions [S] or [B, S] or None."""
    B, S, _, D = x.shape
    R = 2 * len(turns)
    pos = torch.arange(S) if positions is None else positions
    pos = pos.expand(B, S).tolist()
    # Products of whole numbers and doubles as fractions: no rounding before the sine.
    ang = torch.tensor([[[float((p * Fraction(t)) % 1) for t in turns.tolist()] for p in row]
                        for row in pos], dtype=torch.float64).reshape(B, S, 1, R // 2)
    ang = 2 * math.pi * ang * (-1 if back else 1)
    c, s = gain * torch.cos(ang), gain * torch.sin(ang)
    x = x.double()
    y = x.clone()
    ia = torch.arange(R // 2) if pairs == "half" else torch.arange(0, R, 2)
    ib = ia + R // 2 if pairs == "half" else ia + 1
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
    return y
