"""An 8-bit key/value cache in pages, and the attention that reads it.

A streaming or autoregressive run keeps the keys and values of what it has
computed.  The cache here is a pool of pages of 128 tokens (the attention's key
block); a page table says which pages hold a sequence's tokens.  Per page and
key/value head the codes are e4m3 and share one power-of-two scale:

  k        [pages, heads, 128, dim] e4m3    k_scale  [pages, heads] e8m0
  v        [pages, heads, dim, 128] e4m3    v_scale  [pages, heads] e8m0

``lengths[b]`` counts the tokens of sequence b with the tokens of this call; its
n new ones stand at positions lengths[b] - n and on.  Two operators:

  append   append_kv: RMSNorm (over the whole row or each head) and the rotation of
           interleaved pairs on k (and on q, which comes back in its own type), then
           k and v into their pages.  A page's scale is the least 2**e with every
           finite magnitude at most 448 * 2**e; if the page already holds tokens, it is
           never below the old one and their codes are rounded again to a larger one.
  attend   paged_attention: softmax(q k^T / sqrt(dim)) v over a sequence's tokens; causal
           (a query sees the positions up to its own), or every token, or the pages
           that a block mask keeps.  Rows that see nothing are zeros.

Sizes: 12 heads x 128 is this repository's DiT (chunks of 8448 or 16896 tokens at
1408x768); 32 query heads over 8 key/value heads and heads of 64 are generic.
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
EPS = 1e-6
TOP = 448.0     # the largest e4m3 value
LEAST = -126    # the least scale exponent
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # One new token of one stream: the smallest call, all latency.
        {"name": "append_token", "kind": "append", "batch": 1, "new": 1, "held": 700, "ragged": False,
         "hq": 12, "hk": 12, "dim": 128, "dtype": "bf16", "norm": "row", "layout": 1},
        # A serving step: one token for each of 192 sequences of any length, shared heads.
        {"name": "append_tokens_192", "kind": "append", "batch": 192, "new": 1, "held": 1500,
         "ragged": True, "hq": 32, "hk": 8, "dim": 128, "dtype": "bf16", "norm": "none", "layout": 2},
        # Prompts of odd lengths behind earlier turns, packed, heads of 64 with a norm each.
        {"name": "append_prompts_ragged", "kind": "append", "batch": 24, "new": 2100, "held": 900,
         "ragged": True, "hq": 16, "hk": 4, "dim": 64, "dtype": "fp16", "norm": "head", "layout": 3},
        # A 4-frame chunk at 1408x768: RMSNorm over the 1536-wide row, q and k rotated.
        {"name": "append_chunk_16896", "kind": "append", "batch": 1, "new": 16896, "held": 16896,
         "ragged": False, "hq": 12, "hk": 12, "dim": 128, "dtype": "bf16", "norm": "row", "layout": 4},
        # The next token of one short stream.
        {"name": "token_short", "kind": "attend", "batch": 1, "new": 1, "held": 500, "ragged": False,
         "hq": 12, "hk": 12, "dim": 128, "dtype": "bf16", "causal": True, "keep": 0.0, "layout": 5},
        # The next token of 32 ragged sequences, a key/value head for each query head of 64.
        {"name": "tokens_32_ragged", "kind": "attend", "batch": 32, "new": 1, "held": 9000,
         "ragged": True, "hq": 16, "hk": 16, "dim": 64, "dtype": "fp16", "causal": True, "keep": 0.0,
         "layout": 6},
        # The next token of 128 long ragged sequences, shared heads: the cache's bandwidth.
        {"name": "tokens_128_long", "kind": "attend", "batch": 128, "new": 1, "held": 16000,
         "ragged": True, "hq": 32, "hk": 8, "dim": 128, "dtype": "bf16", "causal": True, "keep": 0.0,
         "layout": 7},
        # The next token of one sequence of 262 thousand: one row over a long axis.
        {"name": "token_262k", "kind": "attend", "batch": 1, "new": 1, "held": 262000, "ragged": False,
         "hq": 32, "hk": 8, "dim": 128, "dtype": "bf16", "causal": True, "keep": 0.0, "layout": 8},
        # Five proposed tokens checked at once for each of 16 sequences.
        {"name": "verify_5x16", "kind": "attend", "batch": 16, "new": 5, "held": 6000, "ragged": False,
         "hq": 32, "hk": 8, "dim": 128, "dtype": "bf16", "causal": True, "keep": 0.0, "layout": 9},
        # Prompts packed behind what their sequences hold.
        {"name": "prompts_ragged", "kind": "attend", "batch": 5, "new": 4001, "held": 5000,
         "ragged": True, "hq": 32, "hk": 8, "dim": 128, "dtype": "bf16", "causal": True, "keep": 0.0,
         "layout": 10},
        # One streaming step at 1408x768 over itself and two cached ones, every page.
        {"name": "step_8448", "kind": "attend", "batch": 1, "new": 8448, "held": 16896, "ragged": False,
         "hq": 12, "hk": 12, "dim": 128, "dtype": "bf16", "causal": False, "keep": 0.0, "layout": 11},
        # A 4-frame chunk at 1408x768 and a cached one: 30% of the pages kept for each query block.
        {"name": "chunk_16896_kept", "kind": "attend", "batch": 1, "new": 16896, "held": 16896,
         "ragged": False, "hq": 12, "hk": 12, "dim": 128, "dtype": "bf16", "causal": False,
         "keep": 0.3, "layout": 12},
    ]


HEADS = [(12, 12, 128), (32, 8, 128), (8, 2, 128), (16, 16, 64), (16, 4, 64), (6, 2, 128), (16, 2, 128)]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    hq, hk, dim = rng.choice(HEADS)
    c = {"kind": rng.choice(["append", "attend"]), "hq": hq, "hk": hk, "dim": dim,
         "dtype": rng.choice(["bf16", "bf16", "fp16"]), "ragged": rng.random() < 0.6,
         "layout": rng.randrange(1 << 20)}
    if c["kind"] == "append":
        c["norm"] = rng.choice(["none", "head", "row"])
        if rng.random() < 0.2:
            c["dtype"] = "fp32"
        c["new"] = 1 if rng.random() < 0.4 else _log(rng, 2, 8000)
        c["batch"] = _log(rng, 1, max(1, min(192, 16000 // c["new"])))
        c["held"] = _log(rng, 1, max(2, min(9000, 120000 // c["batch"])))
        return c
    form = rng.choice(["token", "token", "few", "prompt", "kept"])
    c["causal"], c["keep"] = True, 0.0
    if form == "token":
        c["new"], c["batch"] = 1, _log(rng, 1, 128)
        c["held"] = _log(rng, 1, min(100000, 1500000 // c["batch"]))
    elif form == "few":
        c["new"], c["batch"] = rng.randint(2, 40), _log(rng, 1, 32)
        c["held"] = _log(rng, 1, min(20000, 300000 // c["batch"]))
    elif form == "prompt":
        c["new"], c["batch"] = _log(rng, 41, 6000), rng.randint(1, 4)
        c["held"], c["causal"] = _log(rng, 1, 5000), rng.random() < 0.8
    else:
        c["new"], c["batch"] = _log(rng, 41, 9000), 1
        c["held"], c["causal"] = _log(rng, 1, 9000), rng.random() < 0.3
        c["keep"] = round(rng.uniform(0.2, 0.9), 2)
    return c


def _counts(case):
    """New and held tokens of each sequence: the case's own, the largest first."""
    rng = random.Random(case["layout"])
    new, held = [case["new"]], [case["held"]]
    for _ in range(case["batch"] - 1):
        new.append(_log(rng, 1, case["new"]) if case["ragged"] else case["new"])
        held.append(rng.randint(0, case["held"]) if case["ragged"] else case["held"])
    return new, held


def _kept(case, pages):
    """Pages that each row of the block mask keeps."""
    return max(1, round(case["keep"] * pages))


def prepare(case, seed):
    new, held = _counts(case)
    B, hq, hk, D = case["batch"], case["hq"], case["hk"], case["dim"]
    T, dtype = sum(new), DTYPES[case["dtype"]]
    g = torch.Generator(device=DEV).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, device=DEV, generator=g)

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
         "cu": None if min(new) == max(new) else cu.to(DEV), "scale": D ** -0.5,
         "k": (64 * randn(N, hk, PAGE, D)).clamp_(-TOP, TOP).to(torch.float8_e4m3fn),
         "v": (64 * randn(N, hk, D, PAGE)).clamp_(-TOP, TOP).to(torch.float8_e4m3fn),
         # Values of about one, half or a quarter.
         "k_scale": torch.randint(119, 122, (N, hk), device=DEV, generator=g, dtype=torch.uint8)
         .view(torch.float8_e8m0fnu),
         "v_scale": torch.randint(119, 122, (N, hk), device=DEV, generator=g, dtype=torch.uint8)
         .view(torch.float8_e8m0fnu)}
    if case["kind"] == "attend":
        s["q"] = (1.5 * randn(T, hq, D)).to(dtype)
        s["keep"] = None
        if case["keep"]:
            nq, nk = -(-T // PAGE), max(need)
            r = torch.rand(hq, nq, nk, device=DEV, generator=g)
            s["keep"] = r >= r.sort(dim=-1, descending=True).values[..., _kept(case, nk) - 1, None]
        return s
    # The columns of one fused projection, as the linear before writes them; a few channels of k
    # are several times the others.
    qkv = randn(T, hq + 2 * hk, D)
    qkv[:, hq:hq + hk, 7::32] *= 6.0
    qkv = qkv.to(dtype).view(T, hq + 2 * hk, D)
    s["q"], s["new_k"], s["new_v"] = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
    s["wq"] = s["wk"] = None
    if case["norm"] != "none":
        wide = case["norm"] == "row"
        s["wq"] = (1 + 0.1 * randn(hq * D if wide else D)).to(dtype)
        s["wk"] = (1 + 0.1 * randn(hk * D if wide else D)).to(dtype)
    # Rotations of the positions that the new tokens have.
    pos = torch.cat([torch.arange(h, h + n) for n, h in zip(new, held)])
    inv = 10000.0 ** (-torch.arange(0, D, 2, device=DEV, dtype=torch.float64) / D)
    ang = torch.arange(int(lengths.max()), device=DEV, dtype=torch.float64)[:, None] * inv
    s["freqs"] = torch.polar(torch.ones_like(ang), ang).to(torch.complex64)
    s["positions"] = pos.to(torch.int32).to(DEV)
    return s


@functools.lru_cache(maxsize=1)
def _ops():
    package = os.path.join(os.getcwd(), "flashvsr-sm89-ops_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import flashvsr_sm89_ops
    return flashvsr_sm89_ops


def run(s):
    if s["case"]["kind"] == "append":
        q = _append_own(s) if own else _append_plain(s)
        return {"q": q, "k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    return _attend_own(s) if own else _attend_plain(s)


def _append_own(s):
    f = _ops()
    pages = f.KVPages(s["k"], s["v"], s["k_scale"], s["v_scale"])
    return f.append_kv(pages, s["new_k"], s["new_v"], s["table"], s["lengths"], s["cu"],
                       freqs_cis=s["freqs"], positions=s["positions"], k_weight=s["wk"], q=s["q"],
                       q_weight=s["wq"], eps=EPS)


def _attend_own(s):
    f = _ops()
    pages = f.KVPages(s["k"], s["v"], s["k_scale"], s["v_scale"])
    return f.paged_attention(s["q"], pages, s["table"], s["lengths"], s["cu"],
                             causal=s["case"]["causal"], keep=s["keep"])


def _starts(s):
    """First packed row of each sequence, and the end."""
    if s["cu"] is not None:
        return s["cu"].long()
    B = s["lengths"].shape[0]
    return torch.arange(B + 1, device=DEV) * (s["T"] // B)


def _turned_plain(x, w, wide, freqs, positions):
    """RMSNorm over the row or each head, and the rotation, in 32 bits."""
    T, H, D = x.shape
    x = x.float()
    if w is not None:
        r = x.reshape(T, 1, H * D) if wide else x
        r = r * torch.rsqrt(r.square().mean(-1, keepdim=True) + EPS) * w.float()
        x = r.reshape(T, H, D)
    cs = torch.view_as_real(freqs)[positions.long()][:, None]  # [T, 1, D/2, 2]
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cs[..., 0] - b * cs[..., 1], a * cs[..., 1] + b * cs[..., 0]],
                       -1).reshape(T, H, D)


def _bits(x):
    return x.to(torch.float8_e4m3fn).view(torch.uint8)


def _store_plain(x, codes, scale, table, pos, seq, first, held, live):
    """Tokens x [T, H, D] at positions pos of sequences seq into codes [N, H, 128, D] (a view);
    first and held [B]: the page that a sequence's first new token goes to and the tokens that it
    holds before; live [B]: whether there is one."""
    N, H = scale.shape
    page = table[seq, pos // PAGE].long()
    top = torch.zeros(N, H, device=DEV).scatter_reduce_(
        0, page[:, None].expand(-1, H), x.abs().amax(-1), "amax")
    m, e = torch.frexp(top)
    e = torch.where(m > 0.875, e - 8, e - 9).clamp(min=LEAST)  # 448 = 0.875 * 2**9
    e = torch.where(top > 0, e, LEAST)
    old = scale.view(torch.uint8).int() - 127
    touched = torch.zeros(N, dtype=torch.bool, device=DEV).index_fill_(0, page, True)
    has = torch.zeros(N, dtype=torch.int32, device=DEV).scatter_reduce_(
        0, first, torch.where(live, held, 0).int(), "amax")
    e = torch.where((has > 0)[:, None], torch.maximum(e, old), e)
    e = torch.where(touched[:, None], e, old)
    # Codes that stood there, to the scale as it is now.
    was = codes[first]
    now = _bits(was.float() * torch.exp2((old - e)[first].float())[..., None, None])
    mine = (live[:, None] & (torch.arange(PAGE, device=DEV) < held[:, None]))[:, None, :, None]
    raw = codes.view(torch.uint8)
    raw[first] = torch.where(mine, now, raw[first])
    raw[page, :, pos % PAGE] = _bits(x * torch.exp2(-e[page].float())[..., None])
    scale.view(torch.uint8).copy_(e + 127)


def _append_plain(s):
    wide = s["case"]["norm"] == "row"
    starts = _starts(s)
    n = starts[1:] - starts[:-1]
    t = torch.arange(s["T"], device=DEV)
    seq = torch.searchsorted(starts[1:].contiguous(), t, right=True)
    before = s["lengths"].long() - n
    pos = before[seq] + t - starts[seq]
    rows = torch.arange(n.shape[0], device=DEV)
    first = s["table"][rows, before // PAGE].long()
    place = (s["table"], pos, seq, first, before % PAGE, n > 0)
    _store_plain(_turned_plain(s["new_k"], s["wk"], wide, s["freqs"], s["positions"]), s["k"],
                 s["k_scale"], *place)
    _store_plain(s["new_v"].float(), s["v"].transpose(2, 3), s["v_scale"], *place)
    return _turned_plain(s["q"], s["wq"], wide, s["freqs"], s["positions"]).to(s["q"].dtype)


def _attend_plain(s):
    case, table = s["case"], s["table"].long()
    (B, P), hq, hk, D = table.shape, case["hq"], case["hk"], case["dim"]
    G, L, n = hq // hk, P * PAGE, s["most"]
    k = (s["k"].float() * s["k_scale"].float()[..., None, None])[table]      # [B, P, hk, 128, D]
    v = (s["v"].float() * s["v_scale"].float()[..., None, None])[table]      # [B, P, hk, D, 128]
    k = k.permute(0, 2, 4, 1, 3).reshape(B, hk, D, L)
    v = v.permute(0, 2, 1, 4, 3).reshape(B, hk, L, D)
    starts = _starts(s)
    count = starts[1:] - starts[:-1]
    i = torch.arange(n, device=DEV)
    row = torch.where(i < count[:, None], starts[:-1, None] + i, s["T"])     # [B, n]; T: nobody's
    q = torch.cat([s["q"].float(), torch.zeros(1, hq, D, device=DEV)])[row]  # [B, n, hq, D]
    q = q.reshape(B, n, hk, G, D).permute(0, 2, 3, 1, 4).reshape(B, hk, G * n, D)
    x = torch.matmul(q, k).reshape(B, hk, G, n, L)
    j = torch.arange(L, device=DEV)
    sees = j < s["lengths"][:, None, None]                                   # [B, 1, L]
    if case["causal"]:
        sees = sees & (j <= (s["lengths"][:, None] - count[:, None] + i)[..., None])
    sees = sees[:, None, None]
    if s["keep"] is not None:
        sees = sees & s["keep"][:, i // PAGE][..., j // PAGE].reshape(1, hk, G, n, L)
    x = (x * s["scale"]).masked_fill_(~sees, -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True).clamp_(min=-1e30))
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.reshape(B, hk, G * n, L), v).reshape(B, hk, G, n, D)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 3, 1, 2, 4).reshape(B, n, hq, D)
    out = torch.zeros(s["T"] + 1, hq, D, dtype=s["q"].dtype, device=DEV)
    out[row] = o.to(out.dtype)
    return out[:-1]


def work(case):
    new, held = _counts(case)
    hq, hk, D, T = case["hq"], case["hk"], case["dim"], sum(_counts(case)[0])
    size = 4 if case["dtype"] == "fp32" else 2
    need = [-(-(n + h) // PAGE) for n, h in zip(new, held)]
    if case["kind"] == "append":
        # q read and written, k and v read, their codes written, the rotations, a scale byte each.
        touched = sum(-(-(n + h) // PAGE) - h // PAGE for n, h in zip(new, held))
        return {"bytes": T * D * (2 * hq * size + 2 * hk * size + 2 * hk) + T * (4 * D + 4) +
                4 * (2 * len(new) + touched) + 2 * touched * hk,
                "flops": T * D * (hq * 7 + hk * 9)}
    pairs = sum(n * h + n * (n + 1) // 2 if case["causal"] else n * (n + h) for n, h in zip(new, held))
    if case["keep"]:
        pairs = int(pairs * _kept(case, max(need)) / max(need))
    # q and the output; each sequence's codes and scales once; the table.
    return {"bytes": 2 * T * hq * D * size + 2 * hk * D * sum(n + h for n, h in zip(new, held)) +
            sum(need) * (2 * hk + 4) + (hq * -(-T // PAGE) * max(need) if case["keep"] else 0),
            "flops": 4 * pairs * hq * D}


def _e4m3(x):
    """The e4m3 value nearest to x (ties to even), |x| <= 448, in 64 bits."""
    step = torch.exp2((torch.frexp(x)[1] - 4).clamp(min=-9).double())  # three bits behind the first
    return torch.round(x / step) * step


def exact(case, seed):
    new, held = _counts(case)
    if case["kind"] == "attend" and case["hq"] * sum(n * (n + h) for n, h in zip(new, held)) > 8e10:
        return None
    s = prepare(case, seed)
    return _append_exact(s, new, held) if case["kind"] == "append" else _attend_exact(s, new, held)


def _append_exact(s, new, held):
    case = s["case"]
    wide = case["norm"] == "row"

    def turned(x, w):
        T, H, D = x.shape
        x = x.double()
        if w is not None:
            axes = (1, 2) if wide else (2,)
            x = x / torch.sqrt((x ** 2).mean(axes, keepdim=True) + EPS)
            x = x * w.double().view(1, -1, D)
        z = torch.view_as_complex(x.reshape(T, H, D // 2, 2))
        z = z * s["freqs"][s["positions"].long()].to(torch.complex128)[:, None]
        return torch.view_as_real(z).reshape(T, H, D)

    out = {"q": turned(s["q"], s["wq"])}
    for name, x in (("k", turned(s["new_k"], s["wk"])), ("v", s["new_v"].double())):
        codes, scale = s[name].double(), s[name + "_scale"].double()
        if name == "v":
            codes = codes.transpose(2, 3).contiguous()
        t = 0
        for b, (n, h) in enumerate(zip(new, held)):
            for j in range(h // PAGE, -(-(n + h) // PAGE)):
                lo, hi = max(h, j * PAGE), min(n + h, (j + 1) * PAGE)
                p, there = int(s["table"][b, j]), lo - j * PAGE
                y = x[t + lo - h:t + hi - h].transpose(0, 1)                 # [H, tokens, D]
                e = torch.ceil(torch.log2(y.abs().amax((1, 2)) / TOP)).clamp(min=LEAST)
                f = torch.exp2(e)
                if there:
                    f = torch.maximum(f, scale[p])
                    codes[p, :, :there] = _e4m3(codes[p, :, :there] * (scale[p] / f)[:, None, None])
                codes[p, :, there:there + hi - lo] = _e4m3(y / f[:, None, None])
                scale[p] = f
            t += n
        out[name] = codes.transpose(2, 3).contiguous() if name == "v" else codes
        out[name + "_scale"] = scale
    return out


def _attend_exact(s, new, held):
    case, t, out = s["case"], 0, []
    G = case["hq"] // case["hk"]
    for b, (n, h) in enumerate(zip(new, held)):
        ids = s["table"][b, :-(-(n + h) // PAGE)].long()
        heads = []
        for c in range(case["hq"]):
            k = (s["k"][ids, c // G].double() * s["k_scale"][ids, c // G].double()[:, None, None])
            v = (s["v"][ids, c // G].double() * s["v_scale"][ids, c // G].double()[:, None, None])
            k = k.reshape(-1, case["dim"])[:n + h]
            v = v.transpose(1, 2).reshape(-1, case["dim"])[:n + h]
            x = s["q"][t:t + n, c].double() @ k.T.contiguous() / math.sqrt(case["dim"])
            sees = torch.ones(n, n + h, dtype=torch.bool, device=DEV)
            if case["causal"]:
                sees = sees.tril(h)
            if s["keep"] is not None:
                m = s["keep"][c].repeat_interleave(PAGE, 0)[:n].repeat_interleave(PAGE, 1)
                sees = sees & m[:, :n + h]
            x = x.masked_fill(~sees, -math.inf)
            w = torch.where(sees.any(1, keepdim=True), torch.softmax(x, 1), 0.0)
            heads.append(w @ v)
        out.append(torch.stack(heads, 1))
        t += n
    return torch.cat(out)
