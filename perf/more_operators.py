"""Sparse attention over the 8-bit paged cache, and rotary positions.

A long sequence's next tokens need few of its pages.  Three operators choose and read
them; the cache is that of perf/operators.py (pages of 128 tokens, e4m3 codes, a power of
two for each page and head):

  pool     pool_pages: each page that is full gets a mean key, 8-bit integers with a power
           of two of its own for each page and head:
             mean   [pages, heads, dim] int8     scale  [pages, heads] e8m0
           scale is the least 2**e (e >= -127) with |mean of the page's keys| <= 127 * 2**e,
           the codes are rounded to the nearest integer, ties to even.
  select   select_pages: for each row and key/value head the `top` columns of the page
           table that its queries read, rising, -1 behind the last.  The first `first`
           and the last `recent` of those that the row sees are always there; the others
           are those of the highest score max over the group's queries q' . mean * scale, q' the
           group's queries rounded to integers of at most 127 times one power of two.  Ties
           go to the lower column.  The products are of whole numbers: a score is exact.
  attend   selected_attention: softmax(q k^T / sqrt(dim)) v of a row over the tokens up to its
           own position in the pages of its columns.

And before the cache, where keys and queries get their positions:

  rotary   rotary: the first `turned` channels of each head are rotated in pairs (2i, 2i + 1) or
           (i, i + turned / 2) by position * frequency_i; frequencies may be stretched for
           long contexts ("parts": those that turn often over the old context stay, those that do
           not turn once are divided by the factor, linear between, and all is scaled by
           0.1 ln(factor) + 1).  Its gradient is the rotation back.

Sizes: 12 heads x 128 is this repository's DiT (chunks of 16896 tokens at 1408x768); 32 query
heads over 8 key/value heads and heads of 64 are generic.
"""
from __future__ import annotations

import functools
import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"
PAGE = 128
TOP = 448.0     # the largest e4m3 value
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # A serving step in which a page or two of 192 sequences fill up.
        {"name": "pool_step_192", "kind": "pool", "batch": 192, "new": 1, "held": 1535, "ragged": True,
         "hq": 32, "hk": 8, "dim": 128, "layout": 1},
        # Prompts of odd lengths behind earlier turns, packed, heads of 64.
        {"name": "pool_prompts_ragged", "kind": "pool", "batch": 24, "new": 2100, "held": 900,
         "ragged": True, "hq": 16, "hk": 4, "dim": 64, "layout": 2},
        # A 4-frame chunk at 1408x768 behind another.
        {"name": "pool_chunk_16896", "kind": "pool", "batch": 1, "new": 16896, "held": 16896,
         "ragged": False, "hq": 12, "hk": 12, "dim": 128, "layout": 3},
        # The next token of one stream: the smallest selection, all latency.
        {"name": "select_token", "kind": "select", "batch": 1, "new": 1, "held": 20000, "ragged": False,
         "hq": 12, "hk": 12, "dim": 128, "dtype": "bf16", "top": 24, "first": 1, "recent": 2, "layout": 4},
        # The next token of 64 long ragged sequences, shared heads.
        {"name": "select_tokens_64_ragged", "kind": "select", "batch": 64, "new": 1, "held": 130000,
         "ragged": True, "hq": 32, "hk": 8, "dim": 128, "dtype": "fp16", "top": 64, "first": 1,
         "recent": 2, "layout": 5},
        # A chunk of a prompt: every row chooses for itself among some 500 pages.
        {"name": "select_prompt_4096", "kind": "select", "batch": 1, "new": 4096, "held": 60000,
         "ragged": False, "hq": 32, "hk": 8, "dim": 128, "dtype": "bf16", "top": 16, "first": 1,
         "recent": 2, "layout": 6},
        # The next token of one sequence of 262 thousand: 64 of its 2047 pages.
        {"name": "attend_token_262k", "kind": "attend", "batch": 1, "new": 1, "held": 262000,
         "ragged": False, "hq": 32, "hk": 8, "dim": 128, "dtype": "bf16", "top": 64, "first": 1,
         "recent": 2, "layout": 7},
        # The next token of 128 ragged sequences.
        {"name": "attend_tokens_128", "kind": "attend", "batch": 128, "new": 1, "held": 16000,
         "ragged": True, "hq": 32, "hk": 8, "dim": 128, "dtype": "bf16", "top": 32, "first": 1,
         "recent": 2, "layout": 8},
        # A chunk of a prompt, heads of 64 in fp16: every row reads pages of its own choice.
        {"name": "attend_prompt_2048", "kind": "attend", "batch": 1, "new": 2048, "held": 30000,
         "ragged": False, "hq": 16, "hk": 4, "dim": 64, "dtype": "fp16", "top": 16, "first": 1,
         "recent": 2, "layout": 9},
        # One new token's q and k.
        {"name": "rotary_token", "kind": "rotary", "batch": 1, "new": 1, "hq": 32, "hk": 8, "dim": 128,
         "turned": 128, "pairs": "half", "scaling": "none", "dtype": "bf16", "back": False,
         "far": 100000},
        # A training step's q and k, forward and backward.
        {"name": "rotary_train_4x4096", "kind": "rotary", "batch": 4, "new": 4096, "hq": 32, "hk": 8,
         "dim": 128, "turned": 128, "pairs": "half", "scaling": "none", "dtype": "bf16", "back": True,
         "far": 0},
        # A chunk far into a stretched context, half of each head turned, in fp32.
        {"name": "rotary_far_fp32", "kind": "rotary", "batch": 1, "new": 16896, "hq": 12, "hk": 12,
         "dim": 128, "turned": 64, "pairs": "interleaved", "scaling": "parts", "dtype": "fp32",
         "back": False, "far": 900000},
    ]


HEADS = [(12, 12, 128), (32, 8, 128), (8, 2, 128), (16, 16, 64), (16, 4, 64), (6, 2, 128), (16, 2, 128)]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    hq, hk, dim = rng.choice(HEADS)
    kind = rng.choice(["pool", "select", "attend", "rotary"])
    if kind == "rotary":
        back = rng.random() < 0.5
        new = _log(rng, 1, 8000)
        return {"kind": kind, "batch": rng.randint(1, max(1, min(4, 16000 // new))), "new": new,
                "hq": hq, "hk": hk, "dim": dim, "turned": rng.choice([dim, dim, dim // 2, dim // 4]),
                "pairs": rng.choice(["half", "interleaved"]), "scaling": rng.choice(["none", "parts"]),
                "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "back": back,
                "far": rng.choice([0, _log(rng, 1, 1000000)])}
    c = {"kind": kind, "hq": hq, "hk": hk, "dim": dim, "ragged": rng.random() < 0.6,
         "layout": rng.randrange(1 << 20)}
    if kind == "pool":
        c["new"] = 1 if rng.random() < 0.4 else _log(rng, 2, 8000)
        c["batch"] = _log(rng, 1, max(1, min(192, 16000 // c["new"])))
        c["held"] = _log(rng, 1, max(2, min(9000, 120000 // c["batch"])))
        return c
    c["dtype"] = rng.choice(["bf16", "bf16", "fp16"])
    c["first"], c["recent"] = rng.randint(0, 4), rng.randint(1, 4)
    form = rng.choice(["token", "token", "few", "prompt"])
    if form == "token":
        c["new"], c["batch"], c["top"] = 1, _log(rng, 1, 64), rng.randint(8, 64)
        most = 130000 if kind == "select" else min(130000, 1000000 // c["batch"])
        c["held"] = _log(rng, 1, most)
    elif form == "few":
        c["new"], c["batch"], c["top"] = rng.randint(2, 24), _log(rng, 1, 16), rng.randint(8, 40)
        c["held"] = _log(rng, 1, 40000)
    else:
        c["new"], c["batch"], c["top"] = _log(rng, 25, 700), rng.randint(1, 2), rng.randint(8, 16)
        c["held"] = _log(rng, 1, 30000)
    if kind == "select":  # one sequence at least has more pages than are chosen
        c["held"] = max(c["held"], PAGE * (c["top"] + 8))
    return c


def _counts(case):
    """New and held tokens of each sequence: the case's own, the largest first."""
    rng = random.Random(case["layout"])
    new, held = [case["new"]], [case["held"]]
    for _ in range(case["batch"] - 1):
        new.append(_log(rng, 1, case["new"]) if case["ragged"] else case["new"])
        held.append(rng.randint(0, case["held"]) if case["ragged"] else case["held"])
    return new, held


def _turns(case):
    """Turns of each pair per position, and what results are scaled by."""
    R = case["turned"]
    inv = 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    gain = 1.0
    if case["scaling"] == "parts":
        factor, context, fast, slow = 16.0, 65536, 32.0, 1.0
        keep = ((context * inv / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1)
        inv = keep * inv + (1 - keep) * inv / factor
        gain = 0.1 * math.log(factor) + 1
    return inv / (2 * math.pi), gain


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, device=DEV, generator=g)

    hq, hk, D = case["hq"], case["hk"], case["dim"]
    if case["kind"] == "rotary":
        B, S, dtype = case["batch"], case["new"], DTYPES[case["dtype"]]
        turns, gain = _turns(case)
        # The columns of one fused projection, as the linear before writes them.
        qkv = randn(B, S, hq + 2 * hk, D).to(dtype)
        s = {"case": case, "q": qkv[:, :, :hq], "k": qkv[:, :, hq:hq + hk], "turns": turns.to(DEV),
             "gain": gain, "positions": torch.arange(case["far"], case["far"] + S, device=DEV,
                                                     dtype=torch.int32)}
        if case["back"]:
            s["q"], s["k"] = s["q"].detach().requires_grad_(), s["k"].detach().requires_grad_()
            s["dq"], s["dk"] = randn(B, S, hq, D).to(dtype), randn(B, S, hk, D).to(dtype)
        return s
    new, held = _counts(case)
    B, T = case["batch"], sum(new)
    need = [-(-(n + h) // PAGE) for n, h in zip(new, held)]
    N = sum(need) + 3
    # The pages that sequences hold lie anywhere in the pool.
    order = torch.randperm(N, device=DEV, generator=g)[:sum(need)].to(torch.int32).cpu()
    table = torch.zeros(B, max(need), dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    lengths = torch.tensor([n + h for n, h in zip(new, held)], dtype=torch.int32)
    cu = torch.tensor([0] + new, dtype=torch.int32).cumsum(0).to(torch.int32)
    s = {"case": case, "T": T, "most": max(new), "table": table.to(DEV), "lengths": lengths.to(DEV),
         "cu": None if min(new) == max(new) else cu.to(DEV), "scale": D ** -0.5}

    def codes(*shape):
        return (64 * randn(*shape)).clamp_(-TOP, TOP).to(torch.float8_e4m3fn)

    def means():
        return (45 * randn(N, hk, D)).round_().clamp_(-127, 127).to(torch.int8)

    def scales(lo, hi):
        return torch.randint(lo, hi, (N, hk), device=DEV, generator=g, dtype=torch.uint8).view(
            torch.float8_e8m0fnu)
    if case["kind"] != "select":
        # Values of about one, half or a quarter.
        s["k"], s["k_scale"], s["v_scale"] = codes(N, hk, PAGE, D), scales(119, 122), scales(119, 122)
    if case["kind"] == "pool":
        s["v"] = torch.zeros(N, hk, D, PAGE, device=DEV, dtype=torch.uint8).view(torch.float8_e4m3fn)
        s["mean"], s["mean_scale"] = means(), scales(118, 121)  # of what the pages held before
        return s
    s["q"] = (1.5 * randn(T, hq, D)).to(DTYPES[case["dtype"]])
    if case["kind"] == "select":
        s["mean"], s["mean_scale"] = means(), scales(118, 121)
        return s
    s["v"] = codes(N, hk, D, PAGE)
    # Columns as a selection gives them: neighbouring rows want much the same pages.
    seq, last = _places(s)
    P = table.shape[1]
    want = randn(B, hk, P)[seq] + randn(T // 32 + 1, hk, P)[torch.arange(T, device=DEV) // 32]
    want += 0.5 * randn(T, hk, P)
    j, last = torch.arange(P, device=DEV), last[:, None, None]
    always = (j < case["first"]) | (j > last - case["recent"])
    want = want.masked_fill_(always, math.inf).masked_fill_(j > last, -math.inf)
    best, cols = want.topk(min(case["top"], P), dim=-1)
    cols = torch.where(best > -math.inf, cols, P).sort(dim=-1).values
    s["columns"] = torch.full((T, hk, case["top"]), -1, dtype=torch.int32, device=DEV)
    s["columns"][..., :cols.shape[-1]] = torch.where(cols < P, cols, -1)
    return s


def _starts(s):
    """First packed row of each sequence, and the end."""
    if s["cu"] is not None:
        return s["cu"].long()
    B = s["lengths"].shape[0]
    return torch.arange(B + 1, device=DEV) * (s["T"] // B)


def _places(s):
    """Each row's sequence, and the column of its own position."""
    starts = _starts(s)
    t = torch.arange(s["T"], device=DEV)
    seq = torch.searchsorted(starts[1:].contiguous(), t, right=True)
    pos = s["lengths"].long()[seq] - starts[seq + 1] + t
    return seq, pos // PAGE


@functools.lru_cache(maxsize=1)
def _ops():
    package = os.path.join(os.getcwd(), "flashvsr-sm89-ops_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import flashvsr_sm89_ops
    return flashvsr_sm89_ops


def run(s):
    kind = s["case"]["kind"]
    if kind == "rotary":
        return _rotary_own(s) if own else _rotary_plain(s)
    if kind == "select":
        return _select_own(s) if own else _select_plain(s)
    if kind == "attend":
        return _attend_own(s) if own else _attend_plain(s)
    if own:
        _pool_own(s)
    else:
        _pool_plain(s)
    return {"mean": s["mean"], "scale": s["mean_scale"]}


def _pool_own(s):
    f = _ops()
    f.pool_pages(f.PageMeans(s["mean"], s["mean_scale"]),
                 f.KVPages(s["k"], s["v"], s["k_scale"], s["v_scale"]), s["table"], s["lengths"],
                 s["cu"], tokens=s["T"])


def _select_own(s):
    f, case = _ops(), s["case"]
    return f.select_pages(s["q"], f.PageMeans(s["mean"], s["mean_scale"]), s["table"], s["lengths"],
                          s["cu"], top=case["top"], first=case["first"], recent=case["recent"])


def _attend_own(s):
    f = _ops()
    return f.selected_attention(s["q"], f.KVPages(s["k"], s["v"], s["k_scale"], s["v_scale"]),
                                s["table"], s["lengths"], s["columns"], s["cu"])


def _rotary_own(s):
    f = _ops()
    q, k = f.rotary(s["q"], s["k"], f.RotaryFrequencies(s["turns"], s["gain"]), s["positions"],
                    pairs=s["case"]["pairs"])
    if not s["case"]["back"]:
        return {"q": q, "k": k}
    dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
    return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk}


def _pool_plain(s):
    starts = _starts(s)
    before = s["lengths"].long() - (starts[1:] - starts[:-1])
    j = torch.arange(s["table"].shape[1], device=DEV)
    filled = (j >= before[:, None] // PAGE) & (j < s["lengths"].long()[:, None] // PAGE)
    page = s["table"][filled].long()
    # Codes are multiples of 2**-9 and the mean of 128 of 2**-16: whole numbers of 26 bits.
    total = (s["k"][page].float() * 512).to(torch.int32).sum(2, dtype=torch.int32).double()
    e = s["k_scale"].view(torch.uint8)[page].int() - 127 - 16
    m, x = torch.frexp(total.abs().amax(-1))
    least = torch.where(m > 127 / 128, x - 6, x - 7)
    least = torch.where(m > 0, torch.clamp(least, min=-127 - e), -127 - e)
    s["mean"][page] = torch.round(total * torch.exp2(-least.double())[..., None]).to(torch.int8)
    s["mean_scale"].view(torch.uint8)[page] = (least + e + 127).to(torch.uint8)


def _select_plain(s):
    case, table = s["case"], s["table"].long()
    (B, P), hq, hk, D, n = table.shape, case["hq"], case["hk"], case["dim"], s["most"]
    G, top, first, recent = hq // hk, case["top"], case["first"], case["recent"]
    starts = _starts(s)
    i = torch.arange(n, device=DEV)
    row = torch.where(i < (starts[1:] - starts[:-1])[:, None], starts[:-1, None] + i, s["T"])
    q = torch.cat([s["q"].float(), torch.zeros(1, hq, D, device=DEV)])[row]      # [B, n, hq, D]
    q = q.reshape(B, n, hk, G * D)
    m, e = torch.frexp(q.abs().amax(-1, keepdim=True))
    e = torch.where(m > 127 / 128, e - 6, e - 7)
    q = torch.round(q * torch.exp2(-e.float())).reshape(B, n, hk, G, D)
    means = s["mean"][table].float().permute(0, 2, 3, 1).contiguous()            # [B, hk, D, P]
    # Whole numbers below 2**24: fp32's products and sums are exact in any order.
    x = torch.matmul(q.permute(0, 2, 3, 1, 4).reshape(B, hk, G * n, D), means)
    x = x.reshape(B, hk, G, n, P).amax(2).double()
    x = x * s["mean_scale"].double()[table].permute(0, 2, 1)[:, :, None]         # [B, hk, n, P]
    j = torch.arange(P, device=DEV)
    last = (s["lengths"].long() - (starts[1:] - starts[:-1]))[:, None] + i       # [B, n] positions
    last = (last // PAGE)[:, None, :, None]
    x = torch.where((j < first) | (j > last - recent), math.inf, x)
    x = torch.where(j > last, -math.inf, x)
    best, cols = torch.sort(x, dim=-1, descending=True, stable=True)
    cols = torch.where(best[..., :top] > -math.inf, cols[..., :top], P).sort(dim=-1).values
    cols = torch.where(cols < P, cols, -1).to(torch.int32).permute(0, 2, 1, 3)
    out = torch.full((s["T"] + 1, hk, top), -1, dtype=torch.int32, device=DEV)
    out[row, :, :cols.shape[-1]] = cols
    return out[:-1].contiguous()


def _attend_plain(s):
    case, cols = s["case"], s["columns"].long()
    hq, hk, D, T, S = case["hq"], case["hk"], case["dim"], s["T"], s["columns"].shape[-1]
    seq, _ = _places(s)
    pos = s["lengths"].long()[seq] - _starts(s)[seq + 1] + torch.arange(T, device=DEV)
    page = s["table"].long()[seq[:, None, None], cols.clamp(min=0)]              # [T, hk, S]
    h = torch.arange(hk, device=DEV)[None, :, None]
    k = (s["k"][page, h].float() * s["k_scale"].float()[page, h][..., None, None])
    k = k.reshape(T, hk, S * PAGE, D)
    q = s["q"].float().reshape(T, hk, hq // hk, D)
    x = torch.matmul(q, k.transpose(2, 3)) * s["scale"]
    del k
    at = cols[..., None] * PAGE + torch.arange(PAGE, device=DEV)
    sees = (cols[..., None] >= 0) & (at <= pos[:, None, None, None])
    x = x.masked_fill_(~sees.reshape(T, hk, 1, S * PAGE), -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True).clamp_(min=-1e30))
    total = x.sum(-1, keepdim=True)
    v = (s["v"][page, h].float() * s["v_scale"].float()[page, h][..., None, None])
    v = v.transpose(3, 4).reshape(T, hk, S * PAGE, D)
    o = torch.matmul(x, v)
    o = torch.where(total > 0, o / total, 0.0)
    return o.reshape(T, hq, D).to(s["q"].dtype)


def _turned_plain(x, cos, sin, pairs):
    """The first channels of each head of x [B, S, H, D] rotated, in 32 bits."""
    R = 2 * cos.shape[-1]
    y, rest = x[..., :R].float(), x[..., R:]
    half = pairs == "half"
    a, b = (y[..., :R // 2], y[..., R // 2:]) if half else (y[..., 0::2], y[..., 1::2])
    a, b = a * cos - b * sin, a * sin + b * cos
    y = torch.cat([a, b], -1) if half else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([y.to(x.dtype), rest], -1)


def _rotary_plain(s):
    case = s["case"]
    # Angles of far positions: whole turns are taken off in 64 bits.
    turns = s["positions"].double()[:, None] * s["turns"]
    angle = (2 * math.pi * (turns - torch.round(turns)))[:, None]                # [S, 1, R / 2]
    cos, sin = (torch.cos(angle) * s["gain"]).float(), (torch.sin(angle) * s["gain"]).float()
    with torch.no_grad():
        out = {n: _turned_plain(s[n], cos, sin, case["pairs"]) for n in ("q", "k")}
        if case["back"]:
            out |= {n: _turned_plain(s[n], cos, -sin, case["pairs"]) for n in ("dq", "dk")}
    return out


def work(case):
    hq, hk, D = case["hq"], case["hk"], case["dim"]
    if case["kind"] == "rotary":
        size, n = 4 if case["dtype"] == "fp32" else 2, case["batch"] * case["new"] * (hq + hk)
        ways = 2 if case["back"] else 1
        return {"bytes": 2 * ways * n * D * size + 4 * case["new"], "flops": 3 * ways * n * case["turned"]}
    new, held = _counts(case)
    T = sum(new)
    if case["kind"] == "pool":
        # The keys of the pages that fill up, their scales and table entries; the means.
        filled = sum((n + h) // PAGE - h // PAGE for n, h in zip(new, held))
        return {"bytes": filled * (hk * (PAGE * D + D + 2) + 4) + 4 * len(new),
                "flops": filled * hk * PAGE * D}
    top = case["top"]
    pages = [-(-(n + h) // PAGE) for n, h in zip(new, held)]
    if case["kind"] == "select":
        # Each sequence's means once, q, the columns; a product and sum for each query and channel.
        return {"bytes": sum(pages) * (hk * (D + 1) + 4) + T * (2 * hq * D + 4 * hk * top),
                "flops": 2 * hq * D * sum(n * p for n, p in zip(new, pages))}
    # q, the output and the columns; each page that some row reads once.
    read = sum(min(p, n * min(top, p)) for n, p in zip(new, pages))
    seen = sum(n * min(top * PAGE, n + h) for n, h in zip(new, held))
    return {"bytes": T * (4 * hq * D + 4 * hk * top) + read * hk * (2 * PAGE * D + 2),
            "flops": 4 * hq * D * seen}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rotary":
        return _rotary_exact(s)
    new, held = _counts(case)
    if case["kind"] == "pool":
        return _pool_exact(s, new, held)
    if case["kind"] == "select":
        return _select_exact(s, new, held)
    return _attend_exact(s, new, held)


def _pool_exact(s, new, held):
    mean, scale = s["mean"].clone(), s["mean_scale"].double()
    for b, (n, h) in enumerate(zip(new, held)):
        ids = s["table"][b, h // PAGE:(n + h) // PAGE].long()
        if len(ids) == 0:
            continue
        m = s["k"][ids].double().mean(2) * s["k_scale"][ids].double()[..., None]  # exact
        f = torch.exp2(torch.ceil(torch.log2(m.abs().amax(-1) / 127)).clamp(min=-127))
        mean[ids] = torch.round(m / f[..., None]).to(torch.int8)
        scale[ids] = f
    return {"mean": mean, "scale": scale}


def _select_exact(s, new, held):
    case, t, out = s["case"], 0, []
    G, top = case["hq"] // case["hk"], case["top"]
    for b, (n, h) in enumerate(zip(new, held)):
        P = -(-(n + h) // PAGE)
        ids = s["table"][b, :P].long()
        m = s["mean"][ids].double() * s["mean_scale"][ids].double()[..., None]
        last = (h + torch.arange(n, device=DEV)) // PAGE
        j = torch.arange(P, device=DEV)
        sure = (j < case["first"]) | (j[None] > last[:, None] - case["recent"])
        seen = j[None] <= last[:, None]
        rows = torch.full((n, case["hk"], top), -1, dtype=torch.int32, device=DEV)
        for c in range(case["hk"]):
            q = s["q"][t:t + n, c * G:(c + 1) * G].double()
            f = torch.exp2(torch.ceil(torch.log2(q.abs().amax((1, 2), keepdim=True) / 127)))
            x = (torch.round(q / f) * f @ m[:, c].T.contiguous()).amax(1)
            x = x.masked_fill(sure, math.inf).masked_fill(~seen, -math.inf)
            # Ranks: how many pages stand before each one, ties by column.
            order = x.sort(dim=1, descending=True, stable=True).indices
            kept = torch.zeros(n, P, dtype=torch.bool, device=DEV).scatter_(1, order[:, :top], True)
            kept &= seen
            i, col = kept.nonzero(as_tuple=True)
            rows[i, c, kept.cumsum(1)[i, col] - 1] = col.to(torch.int32)
        out.append(rows)
        t += n
    return torch.cat(out)


def _attend_exact(s, new, held):
    case, t, out = s["case"], 0, []
    G = case["hq"] // case["hk"]
    at = torch.arange(PAGE, device=DEV)
    for b, (n, h) in enumerate(zip(new, held)):
        for lo in range(0, n, 256):
            hi, heads = min(n, lo + 256), []
            cols = s["columns"][t + lo:t + hi].long()
            pos = h + torch.arange(lo, hi, device=DEV)
            for c in range(case["hk"]):
                col = cols[:, c]
                ids = s["table"][b, col.clamp(min=0)].long()                       # [r, S]
                k = s["k"][ids, c].double() * s["k_scale"][ids, c].double()[..., None, None]
                v = s["v"][ids, c].double() * s["v_scale"][ids, c].double()[..., None, None]
                q = s["q"][t + lo:t + hi, c * G:(c + 1) * G].double()
                x = torch.einsum("rgd,rstd->rgst", q, k) / math.sqrt(case["dim"])
                sees = (col[..., None] >= 0) & (col[..., None] * PAGE + at <= pos[:, None, None])
                x = x.masked_fill(~sees[:, None], -math.inf).flatten(2)
                w = torch.softmax(x, -1).reshape(hi - lo, G, *col.shape[1:], PAGE)
                heads.append(torch.einsum("rgst,rsdt->rgd", w, v))
            out.append(torch.cat(heads, 1))
        t += n
    return torch.cat(out)


def _rotary_exact(s):
    case = s["case"]
    angle = 2 * math.pi * torch.remainder(s["positions"].double()[:, None] * s["turns"], 1.0)
    z = torch.polar(torch.full_like(angle, s["gain"]), angle)[:, None]

    def turned(x, z):
        R = case["turned"]
        y = x.detach().double()
        a = y[..., :R]
        if case["pairs"] == "half":
            w = torch.complex(a[..., :R // 2].contiguous(), a[..., R // 2:].contiguous()) * z
            a = torch.cat([w.real, w.imag], -1)
        else:
            w = torch.view_as_complex(a.reshape(*a.shape[:-1], R // 2, 2).contiguous()) * z
            a = torch.view_as_real(w).flatten(-2)
        return torch.cat([a, y[..., R:]], -1)

    out = {"q": turned(s["q"], z), "k": turned(s["k"], z)}
    if case["back"]:
        out |= {"dq": turned(s["dq"], z.conj()), "dk": turned(s["dk"], z.conj())}
    return out
