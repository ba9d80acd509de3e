"""append_kv and paged_attention against their 64-bit definition.

Bounds.  A stored value is off by half an e4m3 step and the fp32 steps before it:
norm and rotation are eight roundings of terms below |a| + |b| (the pair), so
2^-21 of that covers them; the returned q by half a step of its type and the same.
Attention: q's terms are exact for bf16 and within 2^-12 for fp16; a weight's terms
leave 2^-8 (two of four bits) or 2^-12 (three) of it; the matrix cores keep a sum of
products to 2^-12 of the sum of their magnitudes (measured: 1.6e-4), which moves a
logit by 2^-12 * logit, and a weight by twice that; the output is rounded once."""
import math

import pytest
import torch

from oracle import paged_kv as O

DEV = "cuda"
pytestmark = pytest.mark.gpu
FP32_STEPS = 2.0 ** -21


def gen(seed):
    return torch.Generator().manual_seed(seed)


def pool(N, H, D, seed=0, bad=False):
    """A pool with codes in every slot (bad: NaN codes), as pages that held other
    sequences before have."""
    from flashvsr_sm89_ops import KVPages
    g = gen(seed)
    k = (64 * torch.randn(N, H, 128, D, generator=g)).clamp(-448, 448).to(torch.float8_e4m3fn)
    v = (64 * torch.randn(N, H, D, 128, generator=g)).clamp(-448, 448).to(torch.float8_e4m3fn)
    if bad:
        k.view(torch.uint8).fill_(0x7f)
        v.view(torch.uint8).fill_(0xff)
    s = torch.randint(119, 123, (2, N, H), generator=g, dtype=torch.uint8)
    e8 = torch.float8_e8m0fnu
    return KVPages(k.to(DEV), v.to(DEV), s[0].to(DEV).view(e8), s[1].to(DEV).view(e8))


def tables(lengths, spare=2, seed=0, width=None):
    """Page tables over a shuffled pool; unused columns hold -1."""
    need = [-(-n // 128) for n in lengths]
    N = sum(need) + spare
    ids = torch.randperm(N, generator=gen(seed))
    t = torch.full((len(lengths), width or max(need + [1])), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        t[b, :n] = ids[at:at + n].int()
        at += n
    return t, N


def i32(x):
    return torch.tensor(x, dtype=torch.int32)


def starts(counts):
    return i32([0] + counts).cumsum(0).int()


def freqs_of(rows, D):
    ang = torch.arange(rows).double()[:, None] * 10000.0 ** (-torch.arange(0, D, 2).double() / D)
    return torch.polar(torch.ones_like(ang), ang).to(torch.complex64)


def nearly(stored, exact, exps, size):
    """stored codes (float64 values) [.., D] of exact values x at scale 2^exps: off by
    half a step and fp32 steps of `size`."""
    s = torch.exp2(exps.double())
    y = exact / s
    ok = (stored - y).abs() <= O.half_step(y) * (1 + 2.0 ** -20) + FP32_STEPS * size / s
    return ok | (torch.isnan(stored) & ~torch.isfinite(y))


def pair_size(x, w, eps):
    """|a| + |b| of the normed pairs, for each of both."""
    y = O.turned(x, w, None, None, eps).abs()
    s = y[..., 0::2] + y[..., 1::2]
    return s.repeat_interleave(2, -1)


def check_append(pages, before, k, v, table, lengths, cu, freqs, pos, kw, eps=1e-6):
    """pages after append_kv of k, v against the definition from `before`."""
    after = O.from_pages(*pages)
    want = {n: before[n].clone() for n in before}
    x = O.turned(k, kw, freqs, pos if freqs is not None else None, eps)
    O.store(want["k"], want["ke"], x, table, lengths, cu)
    vt = want["v"].transpose(2, 3).contiguous()
    O.store(vt, want["ve"], v.double(), table, lengths, cu)
    want["v"] = vt.transpose(2, 3)
    assert torch.equal(after["ke"], want["ke"]) and torch.equal(after["ve"], want["ve"])
    assert torch.equal(after["v"].nan_to_num(nan=999.0), want["v"].nan_to_num(nan=999.0))
    if freqs is None and kw is None:
        assert torch.equal(after["k"].nan_to_num(nan=999.0), want["k"].nan_to_num(nan=999.0))
        return
    # k: the same but where fp32 falls on the other side of a rounding border
    exact, size = torch.full_like(want["k"], math.inf), torch.zeros_like(want["k"])
    ps = pair_size(k, kw, eps)
    for b, (lo, n) in enumerate(O.rows_of(k.shape[0], len(lengths), cu)):
        for i in range(n):
            p = int(lengths[b]) - n + i
            if p < 0 or p // 128 >= table.shape[1]:
                continue
            page = int(table[b, p // 128])
            if 0 <= page < exact.shape[0]:
                exact[page, :, p % 128] = x[lo + i]
                size[page, :, p % 128] = ps[lo + i]
    new = ~torch.isinf(exact)
    same = (after["k"] == want["k"]) | (torch.isnan(after["k"]) & torch.isnan(want["k"]))
    assert bool(same[~new].all())
    e = want["ke"][..., None, None].expand_as(exact)
    assert bool(nearly(after["k"], exact, e, size)[new].all())
    assert float((~same[new]).double().mean()) < 1e-3


def check_q(out, q, freqs, pos, qw, eps=1e-6):
    want = O.turned(q, qw, freqs, pos, eps)
    tol = torch.finfo(q.dtype).eps / 2 * want.abs() + FP32_STEPS * pair_size(q, qw, eps)
    tol = tol + torch.finfo(q.dtype).smallest_normal * 2.0 ** -8  # fp16's subnormal steps
    err = (out.cpu().double() - want).abs()
    assert bool(((err <= tol) | (torch.isnan(out.cpu()) & torch.isnan(want))).all())


NEW = [(0, 5, 1, 130, 64), (128, 127, 129, 300, 1)]
LEN = [(7, 5, 128, 131, 500), (128, 200, 256, 301, 129)]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("norm", ["none", "head", "row"])
@pytest.mark.parametrize("case", [0, 1])
def test_append_ragged(D, dtype, norm, case):
    """Packed rows of several sequences: none, one, whole pages, over a border."""
    from flashvsr_sm89_ops import append_kv
    Hq, H = (6, 2) if case else (3, 3)
    new, lengths = list(NEW[case]), list(LEN[case])
    T, g = sum(new), gen(D + case)
    table, N = tables(lengths, seed=3)
    pages = pool(N, H, D, seed=4)
    before = O.from_pages(*pages)
    qkv = torch.randn(T, Hq + 2 * H, D, generator=g).to(dtype)  # columns of one projection
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + H], qkv[:, Hq + H:]
    kw = qw = None
    if norm != "none":
        kw = (1 + 0.2 * torch.randn(D * (H if norm == "row" else 1), generator=g)).to(dtype)
        qw = (1 + 0.2 * torch.randn(D * (Hq if norm == "row" else 1), generator=g)).to(dtype)
    fr = freqs_of(600, D)
    pos = torch.cat([torch.arange(n - m, n) for m, n in zip(new, lengths)]).int()
    d = qkv.to(DEV)
    cu = starts(new)
    out = append_kv(pages, d[:, Hq:Hq + H], d[:, Hq + H:], table.to(DEV), i32(lengths).to(DEV),
                    cu.to(DEV), freqs_cis=fr.to(DEV), positions=pos.to(DEV),
                    k_weight=None if kw is None else kw.to(DEV), q=d[:, :Hq],
                    q_weight=None if qw is None else qw.to(DEV))
    assert out.shape == q.shape and out.dtype == dtype and out.is_contiguous()
    check_q(out, q, fr, pos, qw)
    check_append(pages, before, k, v, table, lengths, cu, fr, pos, kw)


@pytest.mark.parametrize("D,H", [(64, 5), (128, 2)])
@pytest.mark.parametrize("norm", ["none", "row"])
def test_append_tokens(D, H, norm):
    """One token for each sequence, again and again, of growing size: held codes are
    rounded again as the page's scale grows.  No rotation, so every code is exact (norm:
    by the bound)."""
    from flashvsr_sm89_ops import append_kv
    B, g = 5, gen(9)
    lengths = [1, 128, 129, 60, 255]
    table, N = tables([n + 8 for n in lengths], seed=1)
    pages = pool(N, H, D, seed=2)
    kw = None if norm == "none" else 1 + 0.2 * torch.randn(H * D, generator=g)
    for step in range(6):
        now = [n + step for n in lengths]
        before = O.from_pages(*pages)
        k = torch.randn(B, H, D, generator=g) * 3.0 ** step * 0.01
        v = torch.randn(B, H, D, generator=g) * 4.0 ** (step - 3)
        r = append_kv(pages, k.to(DEV), v.to(DEV), table.to(DEV), i32(now).to(DEV),
                      k_weight=None if kw is None else kw.to(DEV))
        assert r is None
        check_append(pages, before, k, v, table, now, None, None, None, kw)


@pytest.mark.parametrize("D,Hq,H", [(64, 3, 3), (128, 6, 2)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("norm", ["none", "head", "row"])
@pytest.mark.parametrize("packed", [False, True])
def test_append_token_with_q(D, Hq, H, dtype, norm, packed):
    """One token for each sequence with q, norms and a rotation, strided columns of one
    projection; the same as a packed call; a length of 0, a page outside the pool and one
    past the table."""
    from flashvsr_sm89_ops import append_kv
    lengths, g = [1, 128, 129, 77, 0, 200, 500], gen(D)
    B = len(lengths)
    table, N = tables(lengths, seed=1)
    table = table[:, :3].contiguous()
    table[5, 1] = N
    pages = pool(N, H, D, seed=2)
    before = O.from_pages(*pages)
    qkv = torch.randn(B, Hq + 2 * H, D, generator=g).to(dtype)
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + H], qkv[:, Hq + H:]
    kw = qw = None
    if norm != "none":
        kw = 1 + 0.2 * torch.randn(D * (H if norm == "row" else 1), generator=g)
        qw = 1 + 0.2 * torch.randn(D * (Hq if norm == "row" else 1), generator=g)
    fr, pos = freqs_of(300, D), i32([0, 127, 128, 76, 5, -3, 300])
    d = qkv.to(DEV)
    cu = torch.arange(B + 1).int() if packed else None
    out = append_kv(pages, d[:, Hq:Hq + H], d[:, Hq + H:], table.to(DEV), i32(lengths).to(DEV),
                    None if cu is None else cu.to(DEV), freqs_cis=fr.to(DEV),
                    positions=pos.to(DEV), k_weight=None if kw is None else kw.to(DEV),
                    q=d[:, :Hq], q_weight=None if qw is None else qw.to(DEV))
    check_q(out, q, fr, pos, qw)
    check_append(pages, before, k, v, table, lengths, cu, fr, pos, kw)


@pytest.mark.parametrize("D,Hq,H", [(64, 3, 3), (128, 6, 2)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("norm", ["none", "head", "row"])
@pytest.mark.parametrize("n", [2, 5, 8, 9])
def test_append_few_tokens(D, Hq, H, dtype, norm, n):
    """A few tokens for each sequence, within a page, over a border, from its start, behind
    position 0; held codes of small pages are rounded again."""
    from flashvsr_sm89_ops import append_kv
    lengths, g = [n, 128, 130, 77, 1, 256, 128 + n], gen(D)
    B = len(lengths)
    table, N = tables(lengths, seed=1)
    table[3, 0] = N
    pages = pool(N, H, D, seed=2)
    pages.k_scale.view(torch.uint8)[::2] -= 9
    pages.v_scale.view(torch.uint8)[::2] -= 9
    before = O.from_pages(*pages)
    q, k, v = (torch.randn(B * n, h, D, generator=g).to(dtype) for h in (Hq, H, H))
    kw = qw = None
    if norm != "none":
        kw = 1 + 0.2 * torch.randn(D * (H if norm == "row" else 1), generator=g)
        qw = 1 + 0.2 * torch.randn(D * (Hq if norm == "row" else 1), generator=g)
    fr = freqs_of(300, D)
    pos = torch.cat([torch.arange(L - n, L) for L in lengths]).clamp(min=0).int()
    out = append_kv(pages, k.to(DEV), v.to(DEV), table.to(DEV), i32(lengths).to(DEV),
                    freqs_cis=fr.to(DEV), positions=pos.to(DEV),
                    k_weight=None if kw is None else kw.to(DEV), q=q.to(DEV),
                    q_weight=None if qw is None else qw.to(DEV))
    check_q(out, q, fr, pos, qw)
    check_append(pages, before, k, v, table, lengths, None, fr, pos, kw)


@pytest.mark.parametrize("D", [64, 128])
def test_append_token_special_values(D):
    """As test_append_special_values, a token at a time."""
    from flashvsr_sm89_ops import append_kv
    H, B = 4, 6
    k, v = (torch.randn(B, H, D, generator=gen(i)) for i in range(2))
    k[0, 0, 5], k[1, 0, 6], k[2, 0, 7] = math.inf, -math.inf, math.nan
    k[:, 1] = 0.0
    k[:, 2] *= 1e-38
    k[:, 3] *= 1e37
    v[0] = math.nan
    v[1] = 0.0
    v[1, 0, 0], v[1, 1, 1], v[1, 2, 2] = 448.0, 448.0 * (1 + 2.0 ** -23), 3.5 * 2.0 ** -130
    lengths = [1, 129, 257, 2, 100, 128]
    table, N = tables(lengths)
    pages = pool(N, H, D)
    before = O.from_pages(*pages)
    append_kv(pages, k.to(DEV), v.to(DEV), table.to(DEV), i32(lengths).to(DEV))
    check_append(pages, before, k, v, table, lengths, None, None, None, None)


def test_native_and_general_path(monkeypatch):
    """The native host path serves the calls above and gives what the general one does."""
    from flashvsr_sm89_ops import _lib, append_kv, paged_attention
    H, D, B = 2, 128, 3
    table, N = tables([400] * B)
    q, k, v = (torch.randn(B * 7, h, D, generator=gen(h + i)).bfloat16().to(DEV)
               for i, h in enumerate((4, H, H)))
    w = torch.ones(H * D, device=DEV)
    fr, keep = freqs_of(30, D).to(DEV), torch.rand(B, 4, 1, 4, generator=gen(1)).lt(0.7).to(DEV)
    host, got = _lib.paged_host(), []
    assert host is not _lib._GeneralPath
    for general in (False, True):
        monkeypatch.setattr(_lib, "_paged_host", _lib._GeneralPath if general else host)
        pages = pool(N, H, D)
        t, n = table.to(DEV), i32([400, 300, 20]).to(DEV)
        r = [append_kv(pages, k, v, t, n, freqs_cis=fr, k_weight=w, q=q)]
        assert append_kv(pages, k, v, t, n) is None
        r += [paged_attention(q, pages, t, n), paged_attention(q, pages, t, n, keep=keep),
              paged_attention(q[:3], pages, t, n, causal=False, sm_scale=0.3)]
        got.append([x.view(torch.uint8) for x in (*r, *pages)])
    assert all(torch.equal(a, b) for a, b in zip(*got))
    monkeypatch.setattr(_lib, "_paged_host", host)
    c = (pages, k, v, t, n, None, fr, None, w, q, None, 1e-6)
    assert host.append_kv(*c).shape == q.shape and host.append_kv(*c[:9], None, None, 1e-6) is True
    assert host.paged_attention(q, pages, t, n, None, True, keep, None).shape == q.shape
    for i, bad in ((1, k.float()), (2, v[:5]), (3, t.long()), (4, n[:2]), (6, fr[:5]), (6, fr.T),
                   (7, n), (8, w[:5]), (9, q.half()), (0, pages[:3]), (1, k.cpu())):
        assert host.append_kv(*c[:i], bad, *c[i + 1:]) is None, i
    c = (q, pages, t, n, None, True, keep, None)
    for i, bad in ((0, q.float()), (0, q[:, :, :64]), (2, t[:2]), (4, n), (6, keep[:2]),
                   (6, keep.int()), (7, 0.0), (7, -1.0)):
        assert host.paged_attention(*c[:i], bad, *c[i + 1:]) is None, i


def test_append_long_row_norm():
    """Enough tokens that the rows' statistics have a launch of their own, without q; and
    no rotation of a table, row t of it by default."""
    from flashvsr_sm89_ops import append_kv
    T, H, D, g = 300, 12, 128, gen(4)
    lengths = [T + 77]
    table, N = tables(lengths)
    for fr in (None, freqs_of(T, D)):
        pages = pool(N, H, D)
        before = O.from_pages(*pages)
        k, v = (torch.randn(T, H, D, generator=g).bfloat16() for _ in range(2))
        kw = (1 + 0.1 * torch.randn(H * D, generator=g)).bfloat16()
        append_kv(pages, k.to(DEV), v.to(DEV), table.to(DEV), i32(lengths).to(DEV),
                  freqs_cis=None if fr is None else fr.to(DEV), k_weight=kw.to(DEV))
        check_append(pages, before, k, v, table, lengths, None, fr, torch.arange(T), kw)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,n,norm", [(128, 1100, "none"), (128, 1100, "row"), (64, 1100, "row"),
                                      (128, 1, "none"), (64, 5, "none")])
def test_append_codes_of_64_bits(D, dtype, norm, n):
    """Codes next to a border are those of the 64-bit value.  Four roundings of terms up to |a| +
    |b| and one of the value: where it is at least 0.7 of those, 2^-24 * (4 / 0.7 + 1) < 8 steps
    of it, which is the distance from a border within which it is computed in 64 bits.  (With
    sums in 64 bits from the start, as the rows of many tokens have them.)"""
    from flashvsr_sm89_ops import append_kv
    H, B = 4, 1 if n > 8 else 300
    lens, new = [n + 70] * B, [n] * B
    table, N = tables(lens, seed=3)
    pages, g = pool(N, H, D, seed=4), gen(D)
    k = torch.randn(B * n, H, D, generator=g).to(dtype)
    freqs = freqs_of(2000, D)
    pos = torch.randint(0, 2000, (B * n,), generator=g).int()
    kw = 1 + 0.1 * torch.randn(H * D, generator=g).to(dtype) if norm == "row" else None
    append_kv(pages, k.to(DEV), k.to(DEV), table.to(DEV), i32(lens).to(DEV),
              freqs_cis=freqs.to(DEV), positions=pos.to(DEV),
              k_weight=None if kw is None else kw.to(DEV))
    after = O.from_pages(*pages)
    x, size = O.turned(k, kw, freqs, pos, 1e-6), pair_size(k, kw, 1e-6)
    t = torch.arange(B * n)
    b, p = t // n, 70 + t % n
    page = table[b, p // 128].long()
    got = after["k"][page, :, p % 128]
    y = x / torch.exp2(after["ke"][page].double())[..., None]
    plain = (x.abs() >= 0.7 * size) & (y.abs() >= 2.0 ** -6)
    assert float(plain.double().mean()) > 0.2
    assert torch.equal(got[plain], O.e4m3(y)[plain])


@pytest.mark.parametrize("D", [64, 128])
def test_append_special_values(D):
    """Infinities and NaN are stored as NaN and leave the scale alone; zeros; values near
    fp32's ends; a value of 448 * 2^e and the next above it."""
    from flashvsr_sm89_ops import append_kv
    H, T = 4, 20
    k = torch.randn(T, H, D, generator=gen(1))
    k[3, 0, 5], k[4, 0, 6], k[5, 0, 7] = math.inf, -math.inf, math.nan
    k[:, 1] = 0.0
    k[:, 2] *= 1e-38
    k[:, 3] *= 1e37
    v = torch.zeros(T, H, D)
    v[0, 0, 0], v[1, 1, 1], v[2, 2, 2] = 448.0, 448.0 * (1 + 2.0 ** -23), 3.5 * 2.0 ** -130
    v[3, 3], v[4, 3, 0] = math.nan, 1.0
    table, N = tables([T])
    pages = pool(N, H, D)
    before = O.from_pages(*pages)
    append_kv(pages, k.to(DEV), v.to(DEV), table.to(DEV), i32([T]).to(DEV))
    check_append(pages, before, k, v, table, [T], None, None, None, None)
    p = int(table[0, 0])
    e = pages.v_scale.view(torch.uint8)[p].tolist()
    assert e == [127, 128, 1, 127 - 8]
    assert int(pages.k.view(torch.uint8)[p, 0, 3, 5]) & 0x7f == 0x7f


def test_append_outside():
    """Positions below 0, past the table, pages outside the pool and rows behind the last
    sequence are not stored; a position outside the rotations gives NaN."""
    from flashvsr_sm89_ops import append_kv
    H, D, new = 2, 64, [10, 200, 140]
    lengths, T = [4, 300, 140], sum(new) + 9
    table = i32([[5, 1], [0, 2], [7, 3]])  # 7, 5: no such pages; 300 tokens: three pages
    pages = pool(5, H, D)
    before = O.from_pages(*pages)
    k, v, q = (torch.randn(T, H, D, generator=gen(i)) for i in range(3))
    fr = freqs_of(250, D)
    pos = torch.arange(T).int()
    pos[3], pos[100] = -1, 250
    out = append_kv(pages, k.to(DEV), v.to(DEV), table.to(DEV), i32(lengths).to(DEV),
                    starts(new).to(DEV), freqs_cis=fr.to(DEV), positions=pos.to(DEV),
                    q=q.to(DEV))
    check_append(pages, before, k, v, table, lengths, starts(new), fr, pos, None)
    check_q(out, q, fr, pos, None)
    assert bool(torch.isnan(out[3]).all()) and bool(torch.isnan(out[100]).all())
    for a, b in zip(O.from_pages(*pages).values(), before.values()):
        assert torch.equal(a[4], b[4]) and torch.equal(a[1], b[1])


def test_append_odd_layouts():
    """Rows that are not 16-byte aligned or not contiguous in a head are copied first; rows
    of a table wider than its columns; fewer columns than the table's stride."""
    from flashvsr_sm89_ops import append_kv
    H, D, B = 3, 64, 2
    base = torch.randn(2, B * 7, H * D + 3, generator=gen(0)).bfloat16()
    k, v = (t[:, 1:1 + H * D].unflatten(1, (H, D)) for t in base)
    db = base.to(DEV)
    dk, dv = (t[:, 1:1 + H * D].unflatten(1, (H, D)) for t in db)
    table, N = tables([7, 7], width=5)
    pages = pool(N, H, D)
    before = O.from_pages(*pages)
    wide = table.to(DEV)
    append_kv(pages, dk, dv.transpose(1, 2).contiguous().transpose(1, 2), wide[:, :1],
              i32([7, 7]).to(DEV))
    check_append(pages, before, k, v, table[:, :1], [7, 7], None, None, None, None)


# --------------------------------------------------------------------------------------


def check_attention(out, q, pages, table, lengths, cu=None, causal=True, keep=None, sm_scale=None):
    cache = pages if isinstance(pages, dict) else O.from_pages(*pages)
    want, size, logit = O.attention(q, cache, table, lengths, cu, causal, keep, sm_scale)
    dt = q.dtype
    weight = 2.0 ** -8 if dt == torch.bfloat16 else 2.0 ** -12
    tol = torch.finfo(dt).eps / 2 * want.abs() + torch.finfo(dt).smallest_normal
    tol = tol + (weight + 2.0 ** -12 + 2 * 2.0 ** -12 * logit[..., None]) * size
    got = out.cpu().double()
    bad = ~(((got - want).abs() <= tol) | (torch.isnan(got) & torch.isnan(want)))
    assert not bool(bad.any()), (int(bad.sum()), float((got - want).abs().nan_to_num().max()))


LENGTHS = [(1, 2, 127, 128), (129, 0, 300, 1000), (640, 17, 257, 1)]


@pytest.mark.parametrize("D,dtype", [(64, torch.bfloat16), (128, torch.bfloat16),
                                     (64, torch.float16), (128, torch.float16)])
@pytest.mark.parametrize("Hq,H,n", [(3, 3, 1), (8, 2, 1), (16, 1, 1), (4, 2, 3), (2, 1, 8)])
@pytest.mark.parametrize("lens", LENGTHS)
def test_attention_few(D, dtype, Hq, H, n, lens):
    """Up to 16 rows of a key/value head; lengths below the rows' number leave the first
    ones without a key."""
    from flashvsr_sm89_ops import paged_attention
    B = len(lens)
    table, N = tables(lens, seed=5)
    pages = pool(N, H, D, seed=6)
    q = (2 * torch.randn(B * n, Hq, D, generator=gen(7))).to(dtype)
    for causal in (True, False):
        out = paged_attention(q.to(DEV), pages, table.to(DEV), i32(lens).to(DEV), causal=causal)
        check_attention(out, q, pages, table, lens, causal=causal)


@pytest.mark.parametrize("D,dtype", [(64, torch.bfloat16), (128, torch.bfloat16),
                                     (64, torch.float16), (128, torch.float16)])
@pytest.mark.parametrize("Hq,H", [(2, 2), (6, 2), (5, 1)])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_ragged(D, dtype, Hq, H, causal):
    """Packed rows: whole sequences, tails behind held tokens, one token, none; rows behind
    the last sequence are zeros in a new tensor and left alone in a given one."""
    from flashvsr_sm89_ops import paged_attention
    new, lens = [40, 1, 0, 130, 33], [40, 300, 20, 200, 10]
    T = sum(new) + 6
    table, N = tables(lens, seed=1)
    pages = pool(N, H, D, seed=2)
    q = (2 * torch.randn(T, Hq, D, generator=gen(3))).to(dtype)
    args = (q.to(DEV), pages, table.to(DEV), i32(lens).to(DEV), starts(new).to(DEV))
    out = paged_attention(*args, causal=causal)
    check_attention(out, q, pages, table, lens, starts(new), causal)
    assert int(torch.count_nonzero(out[sum(new):])) == 0
    given = torch.full((T, Hq, D + 4), 7.0, dtype=dtype, device=DEV)
    r = paged_attention(*args, causal=causal, out=given[..., :D])
    assert r.data_ptr() == given.data_ptr() and torch.equal(r[:sum(new)], out[:sum(new)])
    assert bool((given[sum(new):] == 7).all()) and bool((given[..., D:] == 7).all())


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [9, 32, 33, 128, 200])
def test_attention_equal_rows(D, n):
    """The same number of rows for every sequence, more than a few."""
    from flashvsr_sm89_ops import paged_attention
    lens, Hq, H = [n, n + 100, n - 3], 4, 2
    table, N = tables(lens, seed=1)
    pages = pool(N, H, D, seed=2)
    q = torch.randn(3 * n, Hq, D, generator=gen(n)).bfloat16()
    out = paged_attention(q.to(DEV), pages, table.to(DEV), i32(lens).to(DEV))
    check_attention(out, q, pages, table, lens)


@pytest.mark.parametrize("D,dtype", [(64, torch.bfloat16), (128, torch.bfloat16),
                                     (64, torch.float16), (128, torch.float16)])
@pytest.mark.parametrize("Hq,H,n", [(2, 2, 17), (8, 2, 5), (4, 1, 8), (20, 1, 1)])
@pytest.mark.parametrize("lens", [(1, 30, 127, 129), (700, 0, 64, 257), (2900, 128, 18, 1100)])
def test_attention_one_unit_of_32(D, dtype, Hq, H, n, lens):
    """17 to 32 rows of a key/value head, the same number for every sequence."""
    from flashvsr_sm89_ops import paged_attention
    table, N = tables(lens, seed=5)
    pages = pool(N, H, D, seed=6)
    q = (2 * torch.randn(len(lens) * n, Hq, D, generator=gen(7))).to(dtype)
    for causal in (True, False):
        out = paged_attention(q.to(DEV), pages, table.to(DEV), i32(lens).to(DEV), causal=causal)
        check_attention(out, q, pages, table, lens, causal=causal)


@pytest.mark.parametrize("D", [64, 128])
def test_attention_one_unit_of_32_odd_pages(D):
    """Missing pages between others, NaN behind the lengths, a last page far above all."""
    from flashvsr_sm89_ops import paged_attention
    H, n, lens = 2, 20, [1500, 400, 130]
    table, N = tables(lens)
    pages = pool(N, H, D, bad=True)
    good = pool(N, H, D)
    ku, vu = pages.k.view(torch.uint8), pages.v.view(torch.uint8)
    for b, L in enumerate(lens):
        for j in range(-(-L // 128)):
            p, m = int(table[b, j]), min(128, L - 128 * j)
            ku[p, :, :m] = good.k.view(torch.uint8)[p, :, :m]
            vu[p, :, :, :m] = good.v.view(torch.uint8)[p, :, :, :m]
    pages.k_scale.view(torch.uint8)[int(table[0, 11])] += 4
    q = torch.randn(3 * n, H, D, generator=gen(3)).bfloat16()
    args = (q.to(DEV), pages, table.to(DEV), i32(lens).to(DEV))
    out = paged_attention(*args)
    assert bool(torch.isfinite(out).all())
    check_attention(out, q, pages, table, lens)
    for at, page in (((1, 0), -1), ((1, 3), N), ((2, 1), 1 << 30)):
        t = table.clone()
        t[at] = page
        out = paged_attention(args[0], pages, t.to(DEV), args[3])
        check_attention(out, q, pages, t, lens)
        sees = torch.arange(lens[at[0]] - n, lens[at[0]]) >= at[1] * 128
        assert torch.equal(out[at[0] * n:(at[0] + 1) * n].isnan().all(-1).all(-1).cpu(), sees)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hq,H,causal,n", [(2, 2, False, 200), (4, 2, True, 140), (2, 1, False, 3)])
def test_attention_keep(dtype, Hq, H, causal, n):
    """A block mask for each head and sequence: random rows, an empty one, a full one, a mask
    smaller than the blocks."""
    from flashvsr_sm89_ops import paged_attention
    D, lens = 128, [n + 700, n]
    table, N = tables(lens, seed=1)
    pages = pool(N, H, D, seed=2)
    q = torch.randn(2 * n, Hq, D, generator=gen(3)).to(dtype)
    for nq, nk in ((-(-n // 128), 8), (1, 3)):
        keep = torch.rand(2, Hq, nq, nk, generator=gen(nk)) < 0.4
        keep[0, 0, 0] = False
        keep[0, 1, 0] = True
        out = paged_attention(q.to(DEV), pages, table.to(DEV), i32(lens).to(DEV), causal=causal,
                              keep=keep.to(DEV))
        check_attention(out, q, pages, table, lens, None, causal, keep)
    one = keep[0]
    out = paged_attention(q[:n].to(DEV), pages, table[:1].to(DEV), i32(lens[:1]).to(DEV),
                          causal=causal, keep=one.to(DEV))
    check_attention(out, q[:n], pages, table[:1], lens[:1], None, causal, one[None])
    none = paged_attention(q[:n].to(DEV), pages, table[:1].to(DEV), i32(lens[:1]).to(DEV),
                           keep=one[:, :0].to(DEV))
    assert int(torch.count_nonzero(none)) == 0


def test_attention_keep_many_pages():
    """More pages than a wave reads of the mask at once, kept ones far apart."""
    from flashvsr_sm89_ops import paged_attention
    n, H, D, lens = 130, 2, 64, [128 * 200 + 5]
    table, N = tables(lens)
    pages = pool(N, H, D)
    keep = torch.zeros(1, H, 2, 201, dtype=torch.bool)
    keep[0, 0, 0, [3, 63, 64, 190]] = True
    keep[0, 1, 1, [127, 200]] = True
    q = torch.randn(n, H, D, generator=gen(3)).bfloat16()
    out = paged_attention(q.to(DEV), pages, table.to(DEV), i32(lens).to(DEV), causal=False,
                          keep=keep.to(DEV))
    check_attention(out, q, pages, table, lens, None, False, keep)


@pytest.mark.parametrize("n,Hq", [(1, 4), (60, 2)])
@pytest.mark.parametrize("D", [64, 128])
def test_attention_hidden_nan(n, Hq, D):
    """NaN behind a length or under the causal mask does not count; one that a row sees
    makes it NaN (and v's only its dim)."""
    from flashvsr_sm89_ops import paged_attention
    H, lens = 2, [200, 90]
    table, N = tables(lens)
    pages = pool(N, H, D, bad=True)
    good = pool(N, H, D)
    ku, vu = pages.k.view(torch.uint8), pages.v.view(torch.uint8)
    for b, L in enumerate(lens):  # every token that is there is good
        for j in range(-(-L // 128)):
            p, m = int(table[b, j]), min(128, L - 128 * j)
            ku[p, :, :m] = good.k.view(torch.uint8)[p, :, :m]
            vu[p, :, :, :m] = good.v.view(torch.uint8)[p, :, :, :m]
    q = torch.randn(2 * n, Hq, D, generator=gen(3)).bfloat16()
    args = (q.to(DEV), pages, table.to(DEV), i32(lens).to(DEV))
    out = paged_attention(*args)
    assert bool(torch.isfinite(out).all())
    check_attention(out, q, pages, table, lens)
    # the last token's v, dim 7, and a k in the middle of the last few
    vu[int(table[0, 1]), 0, 7, 199 - 128] = 0x7f
    ku[int(table[1, 0]), 1, 80, 3] = 0xff
    for causal in (True, False):
        out = paged_attention(*args, causal=causal)
        check_attention(out, q, pages, table, lens, causal=causal)
        last = out[n - 1, 0].isnan()
        assert bool(last[7]) and int(last.sum()) == 1


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,L", [(8, 130), (30, 150), (100, 200), (100, 460)])
@pytest.mark.parametrize("which", ["k_scale", "v_scale"])
def test_attention_hidden_nan_scale(D, n, L, which):
    """A NaN scale makes the rows that see its page NaN and leaves the others' bits."""
    from flashvsr_sm89_ops import paged_attention
    H = 2
    table, N = tables([L])
    pages = pool(N, H, D)
    q = torch.randn(n, H, D, generator=gen(3)).bfloat16().to(DEV)
    args = (q, pages, table.to(DEV), i32([L]).to(DEV))
    good = paged_attention(*args)
    last = (L - 1) // 128
    getattr(pages, which).view(torch.uint8)[int(table[0, last]), 1] = 255
    out = paged_attention(*args)
    sees = torch.arange(L - n, L) >= last * 128
    assert bool(out[sees, 1].isnan().all()) and 0 < int(sees.sum()) < n
    assert torch.equal(out[~sees], good[~sees]) and torch.equal(out[:, 0], good[:, 0])


def test_attention_far_logits():
    """Large logits of either sign, one key far above all others in the last page, equal
    keys: the reference moves where it must."""
    from flashvsr_sm89_ops import paged_attention
    H, D, lens = 2, 128, [600]
    table, N = tables(lens)
    for n in (1, 40):
        pages = pool(N, H, D)
        pages.k_scale.view(torch.uint8)[int(table[0, 0])] += 4  # a first page of large logits
        pages.k_scale.view(torch.uint8)[int(table[0, 4])] += 6
        pages.k.view(torch.uint8)[int(table[0, 1])] = 0  # equal keys
        q = (3 * torch.randn(n, H, D, generator=gen(1))).bfloat16()
        for scale in (None, 1.0, 1e-3, 1e-30):
            out = paged_attention(q.to(DEV), pages, table.to(DEV), i32(lens).to(DEV),
                                  sm_scale=scale)
            assert bool(torch.isfinite(out).all())
            if scale != 1.0:  # (there a logit's own error, 2^-12 of hundreds, is all)
                check_attention(out, q, pages, table, lens, sm_scale=scale)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("pages", [3, 4, 9])
def test_attention_later_page_far_above(dtype, D, pages):
    """A later page's logits lie 2^100 above the first half page's for some rows and below
    for others: the tiles' pipeline keeps the first one's reference and is done again."""
    from flashvsr_sm89_ops import paged_attention
    H, n, lens = 2, 70, [128 * pages + 90]
    table, N = tables(lens)
    pool_ = pool(N, H, D)
    k = pool_.k.view(torch.uint8)
    code = int(torch.tensor(64.0).to(torch.float8_e4m3fn).view(torch.uint8))
    k[int(table[0, 0])] = 0
    k[int(table[0, pages - 1]), :, 5, 0] = code
    pool_.k_scale.view(torch.uint8).fill_(127)
    q = torch.randn(n, H, D, generator=gen(3)) * 0.01
    q[::2, :, 0], q[1::2, :, 0] = 1.5, -1.5
    q = q.to(dtype)
    for causal in (True, False):
        out = paged_attention(q.to(DEV), pool_, table.to(DEV), i32(lens).to(DEV), causal=causal,
                              sm_scale=1.0)
        check_attention(out, q, pool_, table, lens, causal=causal, sm_scale=1.0)


@pytest.mark.parametrize("D,Hq,H", [(128, 3, 3), (64, 4, 1), (128, 8, 2)])
def test_attention_many_tiles(D, Hq, H):
    """More units than the GPU has CUs, the last of them shared out over workgroups, packed and
    equal; every row against the definition on a sample of rows."""
    from flashvsr_sm89_ops import paged_attention
    new, lens = [5000, 900, 64], [6000, 4900, 3000]
    T = sum(new) * 3 if Hq == H else sum(new)
    new = [n * T // sum(new) for n in new]
    lens = [max(a, b) for a, b in zip(lens, new)]
    T = sum(new)
    table, N = tables(lens)
    pages = pool(N, H, D)
    q = torch.randn(T, Hq, D, generator=gen(2)).bfloat16()
    cu = starts(new)
    for causal in (True, False):
        out = paged_attention(q.to(DEV), pages, table.to(DEV), i32(lens).to(DEV), cu.to(DEV),
                              causal=causal).cpu()
        cache = O.from_pages(*pages)
        for b, (lo, n) in enumerate(O.rows_of(T, 3, cu)):
            some = sorted({0, 1, n // 3, n // 2, n - 2, n - 1})
            for i in some:
                # one row alone, at its position: a sequence that ends there (causal) or not
                L = lens[b] - n + i + 1 if causal else lens[b]
                one = q[lo + i:lo + i + 1]
                check_attention(out[lo + i:lo + i + 1], one, cache, table[b:b + 1], [L],
                                causal=False)


def test_attention_many_small_weights():
    """One key of weight 1 and thousands of 2^-15, all equal: small weights are not rounded
    away together."""
    from flashvsr_sm89_ops import paged_attention
    H, D, L = 1, 64, 128 * 64
    table, N = tables([L])
    pages = pool(N, H, D)
    pages.k.view(torch.uint8).zero_()
    pages.k_scale.view(torch.uint8).fill_(127)
    one = torch.tensor(1.0).to(torch.float8_e4m3fn).view(torch.uint8)
    pages.k.view(torch.uint8)[int(table[0, 0]), 0, 0, 0] = int(one)
    x = 15.3 * math.log(2)
    for n in (1, 40):
        q = torch.zeros(n, 1, D).half()
        q[..., 0] = x
        out = paged_attention(q.to(DEV), pages, table.to(DEV), i32([L]).to(DEV), causal=False,
                              sm_scale=1.0)
        check_attention(out, q, pages, table, [L], causal=False, sm_scale=1.0)


@pytest.mark.parametrize("D,Hq,H,n", [(128, 4, 2, 1), (64, 2, 2, 2), (128, 2, 1, 30)])
def test_attention_split(D, Hq, H, n):
    """One sequence whose pages are shared out over workgroups, and a table far wider than
    it; the same bits again."""
    from flashvsr_sm89_ops import paged_attention
    lens = [128 * 70 + 31]
    for width in (71, 700):
        table, N = tables(lens, width=width)
        pages = pool(N, H, D)
        q = torch.randn(n, Hq, D, generator=gen(3)).bfloat16()
        args = (q.to(DEV), pages, table.to(DEV), i32(lens).to(DEV))
        out = paged_attention(*args)
        check_attention(out, q, pages, table, lens)
        assert torch.equal(out, paged_attention(*args))


@pytest.mark.parametrize("new,Hq", [([2, 1, 0, 5], 4), ([20, 0, 33, 1], 2), ([90, 70, 1, 2], 4)])
def test_attention_packed_split(new, Hq):
    """Packed rows, few and many, whose pages are shared out over workgroups, with rows behind
    the last sequence."""
    from flashvsr_sm89_ops import paged_attention
    H, D, lens = 2, 128, [128 * 40 + 3, 900, 50, 128 * 30]
    T = sum(new) + 5
    table, N = tables(lens)
    pages = pool(N, H, D)
    q = torch.randn(T, Hq, D, generator=gen(3)).bfloat16()
    args = (q.to(DEV), pages, table.to(DEV), i32(lens).to(DEV), starts(new).to(DEV))
    for causal in (True, False):
        out = paged_attention(*args, causal=causal)
        check_attention(out, q, pages, table, lens, starts(new), causal)
        assert int(torch.count_nonzero(out[sum(new):])) == 0
        given = torch.full_like(out, 7.0)
        paged_attention(*args, causal=causal, out=given)
        assert torch.equal(given[:sum(new)], out[:sum(new)])
        assert bool((given[sum(new):] == 7).all())


def test_attention_bad_pages():
    """A page id outside the pool makes the rows that read it NaN, and no others."""
    from flashvsr_sm89_ops import paged_attention
    H, D, lens = 2, 128, [300, 300]
    table, N = tables(lens)
    table[1, 2] = N + 5
    pages = pool(N, H, D)
    for n in (2, 60):
        q = torch.randn(2 * n, H, D, generator=gen(3)).bfloat16()
        for t in (-7, 1 << 30):
            table[1, 2] = t
            out = paged_attention(q.to(DEV), pages, table.to(DEV), i32(lens).to(DEV))
            check_attention(out, q, pages, table, lens)
            assert bool(out[-1].isnan().all()) and not bool(out[:n].isnan().any())


def test_attention_non_finite_q():
    from flashvsr_sm89_ops import paged_attention
    H, D, lens = 2, 64, [140]
    table, N = tables(lens)
    pages = pool(N, H, D)
    for n in (3, 50):
        q = torch.randn(n, H, D, generator=gen(3)).half()
        q[0, 0, 5], q[1, 1, 6] = math.inf, math.nan
        out = paged_attention(q.to(DEV), pages, table.to(DEV), i32(lens).to(DEV))
        nan = out.isnan()
        assert bool(nan[0, 0].all()) and bool(nan[1, 1].all()) and int(nan.sum()) == 2 * D


def test_nothing():
    """No rows, no sequences, an empty pool, no columns."""
    from flashvsr_sm89_ops import append_kv, kv_pages, paged_attention
    pages = kv_pages(2, 2, 64, DEV)
    z = torch.zeros(0, 2, 64, dtype=torch.bfloat16, device=DEV)
    t, n = i32([[0]]).to(DEV), i32([0]).to(DEV)
    assert append_kv(pages, z, z, t, n, q=z).shape == z.shape
    assert paged_attention(z, pages, t, n).shape == z.shape
    assert paged_attention(z, pages, t[:0], n[:0]).shape == z.shape
    q = torch.ones(3, 2, 64, dtype=torch.bfloat16, device=DEV)
    assert int(torch.count_nonzero(paged_attention(q, pages, t[:0], n[:0], i32([0]).to(DEV)))) == 0
    assert int(torch.count_nonzero(paged_attention(q, pages, t[:, :0], n))) == 0
    append_kv(pages, q, q, t[:, :0], n + 3)
    none = kv_pages(0, 2, 64, DEV)
    append_kv(none, q, q, t, n + 3)
    assert bool(paged_attention(q, none, t, n + 3).isnan().all())
    assert all(int(torch.count_nonzero(p.view(torch.uint8))) == 0 for p in pages)


def test_far_pages():
    """Page offsets beyond 32 bits: a pool of 4.5 GB for k and for v."""
    from flashvsr_sm89_ops import KVPages, append_kv, paged_attention
    H, D = 8, 128
    N = (1 << 32) // (H * 128 * D) + 100
    e4, e8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
    pages = KVPages(torch.empty(N, H, 128, D, dtype=e4, device=DEV),
                    torch.empty(N, H, D, 128, dtype=e4, device=DEV),
                    torch.empty(N, H, dtype=torch.uint8, device=DEV).view(e8),
                    torch.empty(N, H, dtype=torch.uint8, device=DEV).view(e8))
    table, L = i32([[N - 1, 3, N - 50]]), 300
    k, v = (torch.randn(L, H, D, generator=gen(i)).bfloat16() for i in range(2))
    append_kv(pages, k.to(DEV), v.to(DEV), table.to(DEV), i32([L]).to(DEV))
    near = KVPages(*(p.view(torch.uint8)[table[0].long().to(DEV)].view(p.dtype) for p in pages))
    t3 = i32([[0, 1, 2]])
    empty = {"k": torch.zeros(3, H, 128, D).double(), "ke": torch.zeros(3, H).int()}
    O.store(empty["k"], empty["ke"], k.double(), t3, [L], None)
    got = O.from_pages(*near)
    assert torch.equal(got["k"][:2], empty["k"][:2]) and torch.equal(got["ke"], empty["ke"])
    for n in (1, 50):
        q = torch.randn(n, H, D, generator=gen(5)).bfloat16()
        out = paged_attention(q.to(DEV), pages, table.to(DEV), i32([L]).to(DEV))
        check_attention(out, q, near, t3, [L])


def test_together_as_used():
    """A prompt in two parts, then tokens one by one, shared heads: each step's attention
    against the cache as stored, and near the attention over the values before they were
    rounded to 8 bits."""
    from flashvsr_sm89_ops import append_kv, kv_pages, paged_attention
    B, Hq, H, D, g = 2, 8, 2, 128, gen(0)
    steps = [[100, 37], [60, 5]] + [[1, 1]] * 4
    pages = kv_pages(8, H, D, DEV)
    table = i32([[3, 1, 6], [2, 7, 4]])
    lens = [0, 0]
    fr = freqs_of(400, D)
    keys, values = [[], []], [[], []]
    for new in steps:
        lens = [a + b for a, b in zip(lens, new)]
        T, cu = sum(new), None if new[0] == new[1] else starts(new)
        q, k, v = (torch.randn(T, h, D, generator=g).bfloat16() for h in (Hq, H, H))
        pos = torch.cat([torch.arange(L - n, L) for n, L in zip(new, lens)]).int()
        d = dict(table=table.to(DEV), lens=i32(lens).to(DEV), cu=None if cu is None else cu.to(DEV))
        qr = append_kv(pages, k.to(DEV), v.to(DEV), d["table"], d["lens"], d["cu"],
                       freqs_cis=fr.to(DEV), positions=pos.to(DEV), q=q.to(DEV))
        check_q(qr, q, fr, pos, None)
        out = paged_attention(qr, pages, d["table"], d["lens"], d["cu"])
        check_attention(out, qr.cpu(), pages, table, lens, cu)
        kr = O.turned(k, None, fr, pos, 0.0)
        for b, (lo, n) in enumerate(O.rows_of(T, B, cu)):
            keys[b].append(kr[lo:lo + n])
            values[b].append(v[lo:lo + n].double())
            kk, vv = torch.cat(keys[b]), torch.cat(values[b])
            for c in range(Hq):
                x = qr[lo + n - 1, c].cpu().double() @ kk[:, c // 4].T / math.sqrt(D)
                o = torch.softmax(x, 0) @ vv[:, c // 4]
                err = (out[lo + n - 1, c].cpu().double() - o).norm() / o.norm()
                assert float(err) < 2.0 ** -3  # two roundings of 2^-4 at most, k's into the weights


def test_graph_and_stream():
    """A captured step, replayed as lengths and inputs change with eager work between, equals
    the eager step; a step on another stream."""
    from flashvsr_sm89_ops import append_kv, kv_pages, paged_attention
    B, Hq, H, D = 4, 8, 2, 128
    pages, other = kv_pages(80, H, D, DEV), kv_pages(80, H, D, DEV)
    table = torch.randperm(80, generator=gen(0)).int().view(4, 20).to(DEV)
    lengths = i32([900, 127, 1, 2400]).to(DEV)
    k0, v0 = (torch.randn(3428, H, D, generator=gen(i)).bfloat16().to(DEV) for i in (1, 2))
    for p in (pages, other):
        append_kv(p, k0, v0, table, lengths, starts([900, 127, 1, 2400]).to(DEV))
    q, k, v = (torch.randn(B, h, D, generator=gen(h)).bfloat16().to(DEV) for h in (Hq, H, H))
    w = torch.ones(H * D, device=DEV)
    lengths += 1

    def step(p):
        append_kv(p, k, v, table, lengths, k_weight=w)
        return paged_attention(q, p, table, lengths)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm = step(pages)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(warm, step(other))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(pages)
    for i in range(4):
        lengths += 1
        k.copy_(torch.randn(B, H, D, generator=gen(50 + i)).bfloat16())
        q.copy_(torch.randn(B, Hq, D, generator=gen(60 + i)).bfloat16())
        g.replay()
        want = step(other)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        for a, b in zip(pages, other):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("n", [5, 100])
def test_graph_of_many_rows(n):
    """A captured step of several rows per sequence (row norms: for many rows with their
    workspaces) equals the eager one, replay after replay."""
    from flashvsr_sm89_ops import append_kv, kv_pages, paged_attention
    B, Hq, H, D = 2, 8, 2, 128
    pages, other = kv_pages(60, H, D, DEV), kv_pages(60, H, D, DEV)
    table = torch.randperm(60, generator=gen(0)).int().view(2, 30).to(DEV)
    lengths = i32([n, 1500]).to(DEV)
    q, k, v = (torch.randn(B * n, h, D, generator=gen(h)).bfloat16().to(DEV) for h in (Hq, H, H))
    w, wq = torch.ones(H * D, device=DEV), torch.ones(Hq * D, device=DEV)
    freqs = freqs_of(B * n, D).to(DEV)

    def step(p):
        r = append_kv(p, k, v, table, lengths, freqs_cis=freqs, k_weight=w, q=q, q_weight=wq)
        return paged_attention(r, p, table, lengths)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm = step(pages)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(warm, step(other))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(pages)
    for i in range(4):
        lengths += n
        k.copy_(torch.randn(B * n, H, D, generator=gen(50 + i)).bfloat16())
        q.copy_(torch.randn(B * n, Hq, D, generator=gen(60 + i)).bfloat16())
        g.replay()
        want = step(other)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        for a, b in zip(pages, other):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_two_streams_of_one_pool():
    """Sequences of one pool stepping on two streams at once, their pages side by side."""
    from flashvsr_sm89_ops import append_kv, kv_pages, paged_attention
    Hq, H, D, steps = 8, 2, 128, 40
    table = torch.arange(40).int().view(20, 2).t().contiguous().to(DEV)  # even pages, odd pages
    q, k, v = (torch.randn(steps, 2, 60, h, D, generator=gen(h)).bfloat16().to(DEV)
               for h in (Hq, H, H))
    lens = [i32([60 * (i + 1)]).to(DEV) for i in range(steps)]

    def step(p, i, b):
        append_kv(p, k[i, b], v[i, b], table[b:b + 1], lens[i])
        return paged_attention(q[i, b], p, table[b:b + 1], lens[i])
    one, two = kv_pages(40, H, D, DEV), kv_pages(40, H, D, DEV)
    want = [[step(one, i, b) for b in (0, 1)] for i in range(steps)]
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for i in range(steps):
        row = []
        for b in (0, 1):
            with torch.cuda.stream(side[b]):
                row.append(step(two, i, b))
        got.append(row)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    for a, b in zip(one, two):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
