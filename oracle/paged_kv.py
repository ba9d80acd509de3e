"""The paged 8-bit K/V cache and its attention in 64 bits, token by token and
page by page, on the CPU: the definition that append_kv and paged_attention are
tested against.  Tensors are torch CPU tensors; a cache is a dict of e4m3 codes
as float64 values (``k`` [N, H, 128, D], ``v`` [N, H, D, 128]) and scale
exponents (``ke``, ``ve`` [N, H] int)."""
from __future__ import annotations

import math

import torch

PAGE = 128
TOP = 448.0


def e4m3(x: torch.Tensor) -> torch.Tensor:
    """x (float64, |x| <= 448 or not finite) rounded to e4m3, ties to even; what is
    not finite becomes NaN."""
    step = torch.exp2((torch.frexp(x)[1] - 4).clamp(min=-9).double())
    return torch.where(torch.isfinite(x), torch.round(x / step) * step, math.nan)


def half_step(y: torch.Tensor) -> torch.Tensor:
    """Half the distance between e4m3 neighbours at y."""
    return torch.exp2((torch.frexp(y)[1] - 4).clamp(min=-9).double()) / 2


def exponent(top: float) -> int:
    """Least e >= -126 with top <= 448 * 2^e."""
    if top == 0:
        return -126
    m, e = math.frexp(top)
    return max(e - 9 if m <= 0.875 else e - 8, -126)


def from_pages(k, v, k_scale, v_scale):
    """The cache dict of a pool."""
    def exps(s):
        return s.cpu().view(torch.uint8).int() - 127
    return {"k": k.cpu().float().double(), "v": v.cpu().float().double(), "ke": exps(k_scale),
            "ve": exps(v_scale)}


def turned(x, weight, freqs, positions, eps):
    """RMSNorm (weight over a head or the row, or None) and rotation of x
    [T, H, D] by rows `positions` of freqs (or None)."""
    T, H, D = x.shape
    x = x.double()
    if weight is not None:
        w = weight.double()
        axes = (2,) if w.numel() == D else (1, 2)
        x = x / torch.sqrt((x ** 2).mean(axes, keepdim=True) + eps) * w.reshape(-1, D)
    if freqs is None:
        return x
    f = freqs.to(torch.complex128).reshape(-1, D // 2)
    inside = (positions >= 0) & (positions < f.shape[0])
    f = f[torch.where(inside, positions, 0).long()]
    c, s = f.real[:, None], f.imag[:, None]
    c = torch.where(inside[:, None, None], c, math.nan)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * c - b * s, a * s + b * c], -1).reshape(T, H, D)


def rows_of(T, B, cu):
    if cu is None:
        return [(b * (T // B), T // B) for b in range(B)]
    return [(int(cu[b]), int(cu[b + 1] - cu[b])) for b in range(B)]


def store(codes, exps, x, table, lengths, cu):
    """x [T, H, D] (float64) into codes [N, H, 128, D], exps [N, H], in place."""
    N, H = exps.shape
    for b, (lo, n) in enumerate(rows_of(x.shape[0], len(lengths), cu)):
        at = int(lengths[b]) - n
        spots = [(at + i, lo + i) for i in range(n) if at + i >= 0]
        for j in sorted({p // PAGE for p, _ in spots}):
            if j >= table.shape[1] or not 0 <= int(table[b, j]) < N:
                continue
            page = int(table[b, j])
            mine = [(p % PAGE, t) for p, t in spots if p // PAGE == j]
            held = mine[0][0]
            for h in range(H):
                y = x[[t for _, t in mine], h]
                e = exponent(float(torch.where(torch.isfinite(y), y, 0.0).abs().max()))
                if held:
                    old = int(exps[page, h])
                    e = max(e, old)
                    codes[page, h, :held] = e4m3(codes[page, h, :held] * 2.0 ** (old - e))
                codes[page, h, [s for s, _ in mine]] = e4m3(y * 2.0 ** -e)
                exps[page, h] = e


def attention(q, cache, table, lengths, cu=None, causal=True, keep=None, sm_scale=None):
    """(o, size, logit) [T, Hq, D], [T, Hq, D], [T, Hq]: the attention, the mean of |v| under
    the same weights, and the largest sum of |q k| * sm_scale, for error bounds.
    Rows that see nothing and rows of no sequence are zeros."""
    T, Hq, D = q.shape
    H, N = cache["k"].shape[1], cache["k"].shape[0]
    scale = sm_scale if sm_scale is not None else 1 / math.sqrt(D)
    out, size, logit = (torch.zeros(T, Hq, D).double(), torch.zeros(T, Hq, D).double(),
                        torch.zeros(T, Hq).double())
    q = q.double()
    for b, (lo, n) in enumerate(rows_of(T, len(lengths), cu)):
        L = min(int(lengths[b]), table.shape[1] * PAGE)
        if L <= 0 or n == 0:
            continue
        ids = table[b, :-(-L // PAGE)].long()
        bad = (ids < 0) | (ids >= N)
        ids = torch.where(bad, 0, ids)
        wrong = bad.repeat_interleave(PAGE)[:L]
        pos = torch.arange(L)
        for c in range(Hq):
            h = c // (Hq // H)
            k = (cache["k"][ids, h] * torch.exp2(cache["ke"][ids, h].double())[:, None, None])
            v = (cache["v"][ids, h] * torch.exp2(cache["ve"][ids, h].double())[:, None, None])
            k = k.reshape(-1, D)[:L]
            v = v.transpose(1, 2).reshape(-1, D)[:L]
            k = torch.where(wrong[:, None], math.nan, k)
            for i in range(n):
                sees = torch.ones(L, dtype=torch.bool)
                if causal:
                    sees &= pos <= int(lengths[b]) - n + i
                if keep is not None:
                    m = keep[b, c]
                    row = torch.zeros(L, dtype=torch.bool)
                    if i // PAGE < m.shape[0]:
                        w = m[i // PAGE].repeat_interleave(PAGE)[:L]
                        row[:len(w)] = w
                    sees &= row
                if not sees.any():
                    continue
                x = k[sees] @ q[lo + i, c] * scale
                p = torch.softmax(x, 0)
                out[lo + i, c] = p @ v[sees]
                size[lo + i, c] = p @ v[sees].abs()
                logit[lo + i, c] = (k[sees].abs() @ q[lo + i, c].abs()).max() * scale
    return out, size, logit


def lift(j, h, most):
    """Log2 of the weight of page j's tokens for head h in a lifted counting_pool: a whole number
    of e4m3, at most `most` either way."""
    steps = [x for x in (0, 1, 2, 3, 4, 5, 6, 7, 8, 10, 12, 14, 16, 20) if x <= most]
    x = steps[(5 * j + 3 * h) % len(steps)]
    return x if (j + h) % 3 else -x


def counting_pool(N, H, D, table, seed=0, most=0):
    """A pool in which attention counts tokens: every key is 0, so that what a row sees weighs the
    same (most > 0: lift() in dim 0, for queries of 1 there and sm_scale = ln 2), and every
    value of a sequence's page j is 1 in dim (j + 5 h) % D of head h and 0 in the others, as a
    power of two and a scale that differ from page to page.  An output is then a dim's share
    of the tokens seen, in which one page, or a token, more or less shows.  Codes and scales
    as bytes: (k, v, k_scale, v_scale)."""
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.zeros(s, dtype=torch.uint8) for s in ((N, H, PAGE, D), (N, H, D, PAGE)))
    # (The largest lift at the least scale, 20 * 2^4, is below 448.)
    ke, ve = torch.randint(123, 130, (2, N, H), generator=g, dtype=torch.uint8)
    for row in table.tolist():
        for j, page in enumerate(row):
            if 0 <= page < N:
                for h in range(H):
                    v[page, h, (j + 5 * h) % D] = (7 - (int(ve[page, h]) - 127)) << 3
                    x = torch.tensor(lift(j, h, most) * 2.0 ** (127 - int(ke[page, h])))
                    k[page, h, :, 0] = x.to(torch.float8_e4m3fn).view(torch.uint8)
    return k, v, ke, ve


def counted(T, Hq, H, D, columns, lengths, cu=None, causal=True, keep=None, most=0):
    """[T, Hq, D]: what attention over a counting_pool gives."""
    want = torch.zeros(T, Hq, D).double()
    j = torch.arange(columns)
    for b, (lo, n) in enumerate(rows_of(T, len(lengths), cu)):
        i = torch.arange(n)
        last = int(lengths[b]) - n + i + 1 if causal else torch.full((n,), int(lengths[b]))
        sees = (last[:, None] - PAGE * j).clamp(0, PAGE).double()  # [n, columns]
        for c in range(Hq):
            s = sees
            if keep is not None:
                m = torch.zeros(-(-n // PAGE) + 1, columns).double()
                a = keep[b, c][:m.shape[0], :columns].double()
                m[:a.shape[0], :a.shape[1]] = a
                s = sees * m[i // PAGE]
            h = c // (Hq // H)
            s = s * torch.tensor([2.0 ** lift(x, h, most) for x in range(columns)]).double()
            total = s.sum(1, keepdim=True)
            dims = torch.zeros(columns, D).double()
            dims[j, (j + 5 * h) % D] = 1
            want[lo:lo + n, c] = torch.where(total > 0, s @ dims / total, 0.0)
    return want


def counts_agree(got, want):
    """Whether outputs in a type of 16 bits are `want` from a counting_pool: one rounding to the
    type (or half of its least step), 2^-12 for the matrix cores' sums and 2^-17 for those of up
    to 64 pieces and the fp32 steps of a weight."""
    t = torch.finfo(got.dtype)
    tol = (t.eps / 2 + 2.0 ** -12 + 2.0 ** -17) * want + t.smallest_normal * t.eps / 2
    return bool(((got.double() - want).abs() <= torch.where(want > 0, tol, 0.0)).all())
