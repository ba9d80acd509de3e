"""pool_pages, select_pages and selected_attention against their 64-bit definitions.

Means and columns are exact: whole numbers and powers of two.  The attention's bounds are those of
paged_attention (test_gpu_paged_kv.py): a weight's terms leave 2^-8 of it (bf16), a sum of
products 2^-12 of its terms' magnitudes, the output one rounding.  In fp16 a weight is a half of
11 bits, w (1 + d) with |d| <= 2^-11, in the sum and in the products:
|sum w (1 + d) v / sum w (1 + d) - o| <= 2^-11 (sum w |v| / sum w + |o|) <= 2^-10 sum w |v| / sum w
but for terms of the second order, which the 2^-12 covers."""
import math

import pytest
import torch

from oracle import page_select as S
from oracle import paged_kv as O

DEV = "cuda"
pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16
E8 = torch.float8_e8m0fnu


def gen(seed):
    return torch.Generator().manual_seed(seed)


def i32(x):
    return torch.tensor(x, dtype=torch.int32)


def starts(counts):
    return i32([0] + list(counts)).cumsum(0).int()


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


def pool(N, H, D, seed=0):
    from flashvsr_sm89_ops import KVPages
    g = gen(seed)
    k, v = ((64 * torch.randn(s, generator=g)).clamp(-448, 448).to(torch.float8_e4m3fn)
            for s in ((N, H, 128, D), (N, H, D, 128)))
    s = torch.randint(119, 123, (2, N, H), generator=g, dtype=torch.uint8)
    return KVPages(k.to(DEV), v.to(DEV), s[0].to(DEV).view(E8), s[1].to(DEV).view(E8))


def random_means(N, H, D, seed=0, lo=115, hi=123, size=45.0):
    from flashvsr_sm89_ops import PageMeans
    g = gen(seed)
    mean = (size * torch.randn(N, H, D, generator=g)).round().clamp(-127, 127).to(torch.int8)
    scale = torch.randint(lo, hi, (N, H), generator=g, dtype=torch.int32).to(torch.uint8)
    return PageMeans(mean.to(DEV), scale.to(DEV).view(E8))


def bytes_of(scale):
    return scale.cpu().view(torch.uint8)


# --------------------------------------------------------------------------------------


def check_pool(pages, table, lengths, tokens, cu=None):
    from flashvsr_sm89_ops import pool_pages
    N, H, _, D = pages.k.shape
    means = random_means(N, H, D, seed=9)
    mean, scale = means.mean.cpu(), bytes_of(means.scale).clone()
    r = pool_pages(means, pages, table.to(DEV), i32(lengths).to(DEV),
                   None if cu is None else cu.to(DEV), tokens=tokens)
    assert r is means
    S.pooled(mean, scale, O.from_pages(*pages), bytes_of(pages.k_scale), table, lengths, tokens, cu)
    assert torch.equal(means.mean.cpu(), mean) and torch.equal(bytes_of(means.scale), scale)
    return means


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H", [1, 3])
@pytest.mark.parametrize("new,lengths", [
    ((0, 5, 1, 130, 64), (128, 127, 129, 300, 128)),
    ((128, 127, 129, 300, 1), (128, 256, 257, 301, 512)),
    ((1, 1, 1), (128, 256, 255)), ((500,), (500,)), ((200, 300), (100, 290))])
def test_pool(D, H, new, lengths):
    """Packed rows: whole pages, over a border, none; more rows than the length; the same counts
    without cu_tokens; and every full page."""
    table, N = tables(lengths, seed=1)
    pages = pool(N, H, D, seed=2)
    check_pool(pages, table, lengths, sum(new), starts(new))
    if len(set(new)) == 1:
        check_pool(pages, table, lengths, sum(new))
    check_pool(pages, table, lengths, None)
    check_pool(pages, table, lengths, None, starts(new))


@pytest.mark.parametrize("B", [1, 70, 200])
def test_pool_tokens(B):
    """A token for each of many sequences, some of which fill a page."""
    lengths = [(37 * b) % 300 + 1 for b in range(B)]
    lengths[-1] = 256
    table, N = tables(lengths, seed=1)
    pages = pool(N, 2, 64, seed=2)
    check_pool(pages, table, lengths, B)
    check_pool(pages, table, lengths, B, torch.arange(B + 1).int())


@pytest.mark.parametrize("D", [64, 128])
def test_pool_special_values(D):
    """Ties of the rounding, the largest sums, a zero page, NaN codes and scales, the
    least and the largest scales."""
    H, N = 10, 4
    pages = pool(N, H, D)
    k, s = pages.k.float().cpu(), bytes_of(pages.k_scale).clone()
    k[0, 0] = 0.0
    k[0, 1] = 448.0
    k[0, 2] = torch.where(torch.arange(D) % 2 == 0, 448.0, -448.0)
    k[0, 3] = 0.0                                       # 127 and sums that are x.5 of it
    k[0, 3, 0, 0], k[0, 3, 0, 1], k[0, 3, 0, 2], k[0, 3, 0, 3] = 127.0, 0.5, 1.5, -2.5
    k[0, 4] = 0.0
    k[0, 4, :, 0], k[0, 4, 5, 1] = 448.0, 2.0 ** -9     # 2^25 units beside one
    k[0, 5, 127, D - 1] = math.nan
    k[0, 6] = 0.0
    k[0, 6, 3, 7] = 2.0 ** -9
    k[0, 7] = 448.0
    k[0, 8] = 2.0 ** -9
    s[0] = torch.tensor([0, 120, 254, 120, 130, 120, 0, 254, 5, 255], dtype=torch.uint8)
    s[1] = torch.arange(10, dtype=torch.uint8) * 3
    s[2] = 254 - torch.arange(10, dtype=torch.uint8)
    pages.k.copy_(k.to(torch.float8_e4m3fn).to(DEV))
    pages.k_scale.view(torch.uint8).copy_(s.to(DEV))
    check_pool(pages, torch.arange(4)[None].int(), [512], None)


def test_pool_outside():
    """Page ids outside the pool, lengths past the table, negative ones and none at all."""
    from flashvsr_sm89_ops import pool_pages
    pages = pool(4, 2, 64)
    table = i32([[4, 0, -1], [1, 2, 1000000], [3, -5, 3]])
    for lengths in ([384, 384, 384], [2000, 385, -7], [0, 127, 2 ** 31 - 1]):
        check_pool(pages, table, lengths, None)
        check_pool(pages, table, lengths, 600)
        check_pool(pages, table, lengths, 600, starts([100, 0, 500]))
    means = random_means(4, 2, 64)
    for t, n, T in ((table[:0], i32([]), 0), (table[:0], i32([]), None), (table, i32([9] * 3), 0),
                    (table[:, :0].contiguous(), i32([128] * 3), None)):
        assert pool_pages(means, pages, t.to(DEV), n.to(DEV), tokens=T) is means
    assert torch.equal(means.mean, random_means(4, 2, 64).mean)


@pytest.mark.parametrize("B,H,P", [(64, 8, 32768), (300, 30, 8192), (2, 3, 32768), (1, 2, 40000)])
def test_pool_wide_tables(B, H, P):
    """Every full page of tables far wider than most lengths, with a sequence that fills its row, ids
    outside the pool among them: the same means as from a table of the pool's pages."""
    from flashvsr_sm89_ops import page_means, pool_pages
    N, D = 60, 64
    pages = pool(N, H, D, seed=2)
    g = gen(P)
    lengths = torch.randint(0, 700, (B,), generator=g).int()
    lengths[B // 2], lengths[B - 1] = P * 128, 2 ** 31 - 1
    table = torch.randint(-1, N - 1, (B, P), generator=g).int()
    table[table == N - 2] = N  # (the last two pages are in no table)
    table[B // 2] = torch.randint(5, 25, (P,), generator=g).int()
    table[B - 1, :P - 1] = torch.randint(20, 40, (P - 1,), generator=g).int()
    table[B - 1, P - 1] = 49
    want = pool_pages(page_means(pages), pages, torch.arange(N)[None].int().to(DEV),
                      i32([N * 128]).to(DEV))
    seen = torch.cat([t[:min(n // 128, P)] for t, n in zip(table, lengths.tolist())])
    listed = torch.zeros(N, dtype=torch.bool)
    listed[seen[(seen >= 0) & (seen < N)].long()] = True
    assert bool(listed[20:25].all()) and bool(listed[49]) and not bool(listed.all())
    means = random_means(N, H, D, seed=9)
    mean, scale = means.mean.clone(), means.scale.clone()
    pool_pages(means, pages, table.to(DEV), lengths.to(DEV))
    listed = listed.to(DEV)
    assert torch.equal(means.mean, torch.where(listed[:, None, None], want.mean, mean))
    got, old, new = (x.view(torch.uint8) for x in (means.scale, scale, want.scale))
    assert torch.equal(got, torch.where(listed[:, None], new, old))


# --------------------------------------------------------------------------------------


def check_select(q, means, table, lengths, top, first, recent, cu=None):
    from flashvsr_sm89_ops import select_pages
    got = select_pages(q.to(DEV), means, table.to(DEV), i32(lengths).to(DEV),
                       None if cu is None else cu.to(DEV), top=top, first=first, recent=recent)
    assert got.dtype == torch.int32 and got.is_contiguous()
    want = S.selected(q.double(), means.mean.cpu(), bytes_of(means.scale), table, lengths, top,
                      first, recent, cu)
    assert torch.equal(got.cpu(), want), (got.cpu() != want).nonzero()[:5]
    return got


GROUPS = [(3, 3), (4, 2), (3, 1), (8, 2), (5, 1), (8, 1), (12, 1), (32, 2), (20, 1), (70, 1)]


@pytest.mark.parametrize("Hq,H", GROUPS)
@pytest.mark.parametrize("D,dtype", [(64, BF), (128, FP), (128, BF), (64, FP)])
def test_select_tokens(Hq, H, D, dtype):
    """A token for each of sequences that see none, one, just `top` and more columns."""
    lengths = [0, 1, 128, 129, 5 * 128, 5 * 128 + 1, 40 * 128 - 1, 17 * 128]
    table, N = tables(lengths, seed=Hq)
    q = (2 * torch.randn(len(lengths), Hq, D, generator=gen(D))).to(dtype)
    check_select(q, random_means(N, H, D), table, lengths, 5, 1, 2)


@pytest.mark.parametrize("Hq,H", GROUPS)
@pytest.mark.parametrize("packed", [False, True])
def test_select_rows(Hq, H, packed):
    """More rows than a tile has, over pages' borders, odd numbers, rows before the sequence's
    start and behind the last sequence."""
    D, dtype = (128, BF) if Hq % 2 else (64, FP)
    new, lengths = ((19, 0, 3, 150), (140, 300, 2, 150 + 9 * 128)) if packed else \
        ((37,) * 3, (20, 400, 128 * 12 + 5))
    table, N = tables(lengths, seed=Hq)
    T = sum(new) + (4 if packed else 0)
    q = (2 * torch.randn(T, Hq, D, generator=gen(D))).to(dtype)
    check_select(q, random_means(N, H, D), table, lengths, 6, 1, 1, starts(new) if packed else None)


@pytest.mark.parametrize("B", [1, 9, 80])
def test_select_packed_tokens(B):
    """A token for each of many sequences, packed; some without one, and rows behind the last."""
    lengths = [(577 * b) % 4000 + 1 for b in range(B)]
    new = [int(b % 5 != 3) for b in range(B)]
    table, N = tables(lengths, seed=B)
    q = torch.randn(B, 4, 64, generator=gen(B)).bfloat16()
    check_select(q, random_means(N, 2, 64), table, lengths, 7, 1, 1, starts(new))


@pytest.mark.parametrize("top,first,recent", [(1, 0, 1), (4, 3, 1), (4, 0, 4), (9, 0, 1), (40, 8, 7),
                                              (200, 1, 1)])
@pytest.mark.parametrize("n", [1, 21])
def test_select_lists(top, first, recent, n):
    lengths = [30 * 128 + 5, 128 * 60, n, 9 * 128, 9 * 128 + 1]
    table, N = tables(lengths, seed=3)
    q = torch.randn(5 * n, 4, 128, generator=gen(top)).bfloat16()
    check_select(q, random_means(N, 2, 128), table, lengths, top, first, recent)


@pytest.mark.parametrize("n", [1, 20])
@pytest.mark.parametrize("size,lo,hi", [(0.0, 120, 121), (0.3, 120, 121), (0.5, 119, 122),
                                        (45.0, 0, 256), (45.0, 250, 256), (200.0, 0, 3)])
def test_select_ties(n, size, lo, hi):
    """Equal scores (products of small whole numbers), scales over the whole range, NaN among them."""
    lengths = [50 * 128, 128 * 33 - 1]
    table, N = tables(lengths, seed=5)
    table[0, 7] = N
    table[0, 9] = -1
    q = torch.randint(-2, 3, (2 * n, 4, 64), generator=gen(2)).to(BF)
    for top in (3, 12, 47):
        check_select(q, random_means(N, 2, 64, lo=lo, hi=hi, size=size), table, lengths, top, 1, 1)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_select_special_queries(dtype):
    """Zeros, infinities, NaN, subnormals, the borders of the rounding to integers."""
    n, D = 12, 64
    lengths = [30 * 128]
    table, N = tables(lengths)
    q = torch.randn(n, 4, D, generator=gen(1))
    q[0] = 0.0
    q[1, 0, 3], q[2, 1, 5], q[3, 2, 7] = math.inf, -math.inf, math.nan
    q[4] *= 2.0 ** -15                       # fp16's subnormals
    q[5] *= 2.0 ** -128                      # bf16's
    q[6, :, 0], q[6, :, 1:] = 127.0, torch.arange(D - 1) / 2.0
    q[7, :, 0], q[7, :, 1:] = 127.5, torch.arange(D - 1) / 2.0
    q[8, :2, 0], q[9, :2, 0] = 127 * 2.0 ** 8, 2.0 ** 15
    q[10] = torch.finfo(dtype).max
    q[11, 0, 0] = -torch.finfo(dtype).max
    check_select(q.to(dtype), random_means(N, 2, D), table, lengths, 5, 1, 1)


@pytest.mark.parametrize("pages,n,top", [(600, 1, 20), (1500, 3, 64), (3000, 1, 500),
                                         (9000, 2, 33), (32768, 1, 64), (600, 40, 20),
                                         (1100, 30, 64), (600, 33, 300), (140, 70, 40)])
def test_select_many_pages(pages, n, top):
    """Columns beyond what registers hold, in rows alone and in tiles, and the widest table."""
    lengths = [pages * 128 - 5]
    g = gen(pages)
    table, N = torch.randint(0, 700, (1, pages), generator=g).int(), 700  # pages shared: ties
    q = torch.randn(n, 2, 64, generator=g).bfloat16()
    check_select(q, random_means(N, 1, 64), table, lengths, top, 1, 3)


@pytest.mark.parametrize("Hq,H", [(3, 3), (4, 2), (8, 2), (8, 1), (16, 1), (20, 1)])
@pytest.mark.parametrize("D,dtype", [(128, BF), (128, FP), (64, BF)])
def test_select_groups(Hq, H, D, dtype):
    """Every width of a group: tokens over long tables, and rows enough for four operands."""
    lengths, new = [300 * 128, 5, 411 * 128 - 7], [1, 0, 1]
    table, N = tables(lengths, seed=1)
    q = (2 * torch.randn(3, Hq, D, generator=gen(Hq))).to(dtype)
    check_select(q[:2], random_means(N, H, D), table, lengths, 30, 1, 2, starts(new))
    check_select(q, random_means(N, H, D), table, lengths, 30, 1, 2)
    lengths = [20 * 128 + 40, 3000]
    table, N = tables(lengths, seed=1)
    q = (2 * torch.randn(70, Hq, D, generator=gen(Hq))).to(dtype)
    check_select(q, random_means(N, H, D), table, lengths, 6, 1, 1)


@pytest.mark.parametrize("top", [2, 20, 240, 256])
@pytest.mark.parametrize("pages", [257, 258, 300, 384, 386, 513, 770])
def test_select_waves_without_keys(pages, top):
    """A row that has its workgroup to itself, where the last waves' shares of the keys are short or
    empty."""
    table, N = tables([pages * 128], seed=1)
    q = torch.randn(1, 2, 64, generator=gen(pages)).bfloat16()
    check_select(q, random_means(N, 1, 64), table, [pages * 128], top, 1, 1)


def test_select_many_pages_of_many_heads():
    """A group past 16 queries over more pages than a wave's registers hold."""
    lengths, new = [600 * 128 - 9, 700 * 128], [2, 3]
    table, N = tables(lengths, seed=2)
    q = torch.randn(sum(new), 20, 64, generator=gen(1)).half()
    check_select(q, random_means(N, 1, 64), table, lengths, 50, 1, 3, starts(new))


def test_select_wide_table():
    """A table far wider than the lengths; rows of it strided."""
    lengths = [700, 1300]
    table, N = tables(lengths, width=30000)
    q = torch.randn(10, 4, 64, generator=gen(1)).bfloat16()
    check_select(q, random_means(N, 2, 64), table, lengths, 3, 0, 1)
    both = torch.cat([table, table], 1).to(DEV)
    from flashvsr_sm89_ops import select_pages
    args = (random_means(N, 2, 64),), dict(top=3)
    a = select_pages(q.to(DEV), *args[0], both[:, :30000], i32(lengths).to(DEV), top=3)
    b = select_pages(q.to(DEV), *args[0], table.to(DEV), i32(lengths).to(DEV), top=3)
    assert torch.equal(a, b)


def test_select_strided_and_nothing():
    from flashvsr_sm89_ops import select_pages
    lengths = [20 * 128, 11 * 128]
    table, N = tables(lengths)
    means = random_means(N, 2, 128)
    base = torch.randn(6, 1030, generator=gen(3)).bfloat16()
    for cols in (base[:, 6:518], base[:, 5:517]):  # 16-byte aligned or not
        q = cols.unflatten(1, (4, 128))
        d = base.to(DEV)[:, cols.storage_offset():][:, :512].unflatten(1, (4, 128))
        got = select_pages(d, means, table.to(DEV), i32(lengths).to(DEV), top=4)
        want = S.selected(q.double(), means.mean.cpu(), bytes_of(means.scale), table, lengths, 4, 1, 1)
        assert torch.equal(got.cpu(), want)
    none = select_pages(d[:0], means, table.to(DEV), i32(lengths).to(DEV), top=4)
    assert none.shape == (0, 2, 4)
    none = select_pages(d, means, table[:0].to(DEV), i32([]).to(DEV), starts([]).to(DEV), top=4)
    assert none.shape == (6, 2, 4) and bool((none == -1).all())
    none = select_pages(d, means, table[:, :0].contiguous().to(DEV), i32(lengths).to(DEV), top=4)
    assert bool((none == -1).all())
    empty = type(means)(means.mean[:0], means.scale[:0])  # a pool without pages: the lowest columns
    got = select_pages(d, empty, table.to(DEV), i32(lengths).to(DEV), top=4)
    assert got[0, 0].tolist() == [0, 1, 2, 19]


# --------------------------------------------------------------------------------------


def check_attention(out, q, pages, table, lengths, columns, cu=None, sm_scale=None, rows=None):
    """rows: those that are looked at (the definition is slow)."""
    cache = O.from_pages(*pages)
    if rows is not None:
        keep = torch.isin(torch.arange(len(columns)), rows)[:, None, None]
        columns, out = torch.where(keep, columns, -1), torch.where(keep, out.cpu(), 0)
    want, size, logit = S.attended(q, cache, table, lengths, columns, cu, sm_scale)
    dt = q.dtype
    weight = 2.0 ** -8 if dt == BF else 2.0 ** -10
    tol = torch.finfo(dt).eps / 2 * want.abs() + torch.finfo(dt).smallest_normal
    tol = tol + (weight + 2.0 ** -12 + 2 * 2.0 ** -12 * logit[..., None]) * size
    got = out.cpu().double()
    bad = ~(((got - want).abs() <= tol) | (torch.isnan(got) & torch.isnan(want)))
    assert not bool(bad.any()), (int(bad.sum()), float((got - want).abs().nan_to_num().max()))


def random_columns(T, H, n, lengths, counts, seed=0, wild=False):
    """Lists of distinct columns that a row sees, -1 behind them (wild: any numbers, in any
    order, some twice)."""
    g = gen(seed)
    out = torch.full((T, H, n), -1, dtype=torch.int32)
    t = 0
    for L, m in zip(lengths, counts):
        for i in range(m):
            p = L - m + i
            seen = p // 128 + 1 if p >= 0 else 0
            for h in range(H):
                if wild:
                    out[t, h] = torch.randint(-2, seen + 3, (n,), generator=g).int()
                else:
                    c = torch.randperm(seen, generator=g)[:n].sort().values.int()
                    out[t, h, :len(c)] = c
            t += 1
    return out


@pytest.mark.parametrize("D,dtype", [(64, BF), (128, BF), (64, FP), (128, FP)])
@pytest.mark.parametrize("Hq,H,n", [(3, 3, 1), (8, 2, 1), (16, 1, 2), (20, 1, 1), (4, 2, 5)])
@pytest.mark.parametrize("wild", [False, True])
def test_attention(D, dtype, Hq, H, n, wild):
    """A token or a few for each sequence; lists of every kind; lengths below the rows'."""
    from flashvsr_sm89_ops import selected_attention
    lengths = [1, 0, 127, 128, 129, 700, 1300]
    table, N = tables(lengths, seed=5, width=11)
    pages = pool(N, H, D, seed=6)
    T = len(lengths) * n
    q = (2 * torch.randn(T, Hq, D, generator=gen(7))).to(dtype)
    for m in (1, 3, 9):
        cols = random_columns(T, H, m, lengths, [n] * len(lengths), seed=m, wild=wild)
        out = selected_attention(q.to(DEV), pages, table.to(DEV), i32(lengths).to(DEV),
                                 cols.to(DEV))
        assert out.shape == q.shape and out.dtype == dtype and out.is_contiguous()
        check_attention(out, q, pages, table, lengths, cols)


@pytest.mark.parametrize("D,dtype", [(64, BF), (128, FP)])
@pytest.mark.parametrize("Hq,H", [(4, 4), (6, 2)])
def test_attention_packed(D, dtype, Hq, H):
    """Packed rows, a scale, rows behind the last sequence: zeros, or left alone in `out`."""
    from flashvsr_sm89_ops import selected_attention
    new, lengths = [0, 5, 30, 1], [128, 300, 30, 900]
    table, N = tables(lengths, seed=5)
    pages, T = pool(N, H, D, seed=6), sum(new) + 3
    q = (2 * torch.randn(T, Hq, D, generator=gen(7))).to(dtype)
    cols = random_columns(T, H, 4, lengths, new)
    args = (q.to(DEV), pages, table.to(DEV), i32(lengths).to(DEV), cols.to(DEV), starts(new).to(DEV))
    out = selected_attention(*args, sm_scale=0.3)
    check_attention(out, q, pages, table, lengths, cols, starts(new), sm_scale=0.3)
    wide = torch.full((T, Hq + 2, D + 4), 7.0, dtype=dtype, device=DEV)
    given = wide[:, 1:1 + Hq, 4:]
    assert selected_attention(*args, sm_scale=0.3, out=given) is given
    assert torch.equal(given[:-3], out[:-3]) and bool((given[-3:] == 7).all())
    wide[:, 1:1 + Hq, 4:] = 7.0
    assert bool((wide == 7).all())


@pytest.mark.parametrize("T,Hq,H,D,n,dtype", [
    (1, 2, 2, 128, 300, BF), (1, 4, 1, 64, 64, FP), (3, 8, 2, 128, 40, BF), (600, 8, 8, 64, 5, BF),
    (1100, 8, 4, 128, 4, FP), (4200, 40, 1, 64, 3, BF), (700, 16, 16, 128, 5, BF),
    (400, 32, 16, 64, 5, FP), (330, 48, 16, 128, 3, FP), (700, 16, 16, 64, 12, BF)])
def test_attention_counts(T, Hq, H, D, n, dtype):
    """Over a pool in which attention counts tokens: lists in pieces, a wave to a list; every
    entry of every list shows.  (300 pieces' sums: (4 + 300 / 64) * 2^-24 < 2^-17.)"""
    from flashvsr_sm89_ops import KVPages, selected_attention
    lengths = [max(n, 12) * 128 + 77] if T == 1 else [T + 1000]
    columns = -(-lengths[0] // 128)
    table = torch.arange(columns)[None].int()
    k, v, ks, vs = O.counting_pool(columns, H, D, table, most=3)
    e4 = torch.float8_e4m3fn
    pages = KVPages(k.to(DEV).view(e4), v.to(DEV).view(e4), ks.to(DEV).view(E8),
                    vs.to(DEV).view(E8))
    q = torch.zeros(T, Hq, D, dtype=dtype)
    q[..., 0] = 1
    cols = random_columns(T, H, n, lengths, [T], seed=n)
    out = selected_attention(q.to(DEV), pages, table.to(DEV), i32(lengths).to(DEV), cols.to(DEV),
                             sm_scale=math.log(2))
    want = S.counted(T, Hq, H, D, table, lengths, cols, most=3)
    assert O.counts_agree(out.cpu(), want)


def listed(T, H, n, columns, kind, seed):
    """[T, H, n] columns: those of neighbouring rows are disjoint as far as the columns go, rising or
    not, or any, some twice and some that no row sees."""
    if kind == "any":
        return torch.randint(-3, columns + 3, (T, H, n), generator=gen(seed)).int()
    t, h = torch.arange(T)[:, None, None], torch.arange(H)[None, :, None]
    c = ((t * n + 3 * h + torch.arange(n)) % columns).sort(-1).values
    return (c if kind == "rising" else c.flip(-1)).int().contiguous()


@pytest.mark.parametrize("kind", ["rising", "falling", "any"])
@pytest.mark.parametrize("T,Hq,H,D,n,dtype", [
    (7, 4, 4, 64, 255, BF), (7, 4, 4, 64, 256, FP), (7, 4, 2, 128, 257, BF), (7, 8, 2, 64, 512, BF),
    (7, 2, 2, 64, 1023, BF), (7, 4, 2, 64, 1024, FP), (7, 4, 2, 64, 1025, BF), (3, 20, 1, 64, 1025, BF),
    (9, 16, 16, 64, 255, BF), (9, 16, 16, 128, 256, BF), (9, 16, 16, 64, 256, FP), (9, 16, 16, 64, 257, FP),
    (40, 16, 16, 128, 64, BF), (40, 16, 16, 64, 64, FP), (100, 16, 16, 64, 24, BF), (70, 32, 16, 64, 32, BF),
    (90, 16, 16, 64, 43, BF), (45, 16, 16, 64, 128, BF), (45, 32, 16, 128, 129, FP)])
def test_attention_long_lists(T, Hq, H, D, n, dtype, kind):
    """Several rows whose lists, at the sizes where a unit gets a row fewer or the lists leave LDS, and
    disjoint lists that fill every entry it holds."""
    from flashvsr_sm89_ops import KVPages, selected_attention
    columns = max(n, 270 if n <= 128 else 0) + 2
    lengths = [columns * 128 - 5 - T // 2]
    table = torch.arange(columns)[None].int()
    k, v, ks, vs = O.counting_pool(columns, H, D, table, most=2)
    e4 = torch.float8_e4m3fn
    pages = KVPages(k.to(DEV).view(e4), v.to(DEV).view(e4), ks.to(DEV).view(E8), vs.to(DEV).view(E8))
    q = torch.zeros(T, Hq, D, dtype=dtype)
    q[..., 0] = 1
    cols = listed(T, H, n, columns, kind, seed=n)
    out = selected_attention(q.to(DEV), pages, table.to(DEV), i32(lengths).to(DEV), cols.to(DEV),
                             sm_scale=math.log(2))
    want = S.counted(T, Hq, H, D, table, lengths, cols, most=2)
    assert O.counts_agree(out.cpu(), want)


@pytest.mark.parametrize("T,Hq,H", [(1100, 16, 16), (530, 32, 8)])
def test_attention_units_of_a_wave(T, Hq, H):
    """bf16, heads of 128, more units than two waves of each have room for: a wave to a unit."""
    test_attention_counts(T, Hq, H, 128, 5, BF)
    test_attention_neighbours_of_non_finite_queries(T, Hq, H, 128, BF)
    test_attention_far_logits(T, Hq, H, 128, BF)
    if Hq == H:
        test_attention_bad_pages_and_hidden_nan(T, H, 128)


@pytest.mark.parametrize("where", ["", "k", "v", "k_scale", "v_scale"])
@pytest.mark.parametrize("wild", [False, True])
def test_attention_units_of_a_wave_with_nan(where, wild):
    test_attention_many_units(32, 32, 128, BF, wild, where)


@pytest.mark.parametrize("T,Hq,H,D,dtype", [(5, 4, 1, 64, BF), (30, 10, 2, 128, FP),
                                            (400, 8, 8, 64, FP), (800, 8, 4, 128, BF),
                                            (700, 16, 16, 128, BF), (400, 32, 16, 64, FP)])
def test_attention_neighbours_of_non_finite_queries(T, Hq, H, D, dtype):
    """A query with a NaN or an infinity is NaN; the rows and heads beside it are not."""
    from flashvsr_sm89_ops import selected_attention
    lengths = [T + 400]
    table, N = tables(lengths, seed=1)
    pages = pool(N, H, D, seed=2)
    cols = random_columns(T, H, 3, lengths, [T], seed=4)
    q = torch.randn(T, Hq, D, generator=gen(3)).to(dtype)
    q[1, 0, 3], q[4, Hq - 1, 9] = math.nan, math.inf
    out = selected_attention(q.to(DEV), pages, table.to(DEV), i32(lengths).to(DEV), cols.to(DEV))
    bad = torch.isnan(out.cpu()).any(-1)
    assert bool(bad[1, 0]) and bool(bad[4, Hq - 1]) and int(bad.sum()) == 2
    rows = torch.cat([torch.arange(5), torch.arange(5, T, 29)])  # (the definition is slow)
    want, size, logit = S.attended(q, O.from_pages(*pages), table, lengths, torch.where(
        torch.isin(torch.arange(T), rows)[:, None, None], cols, -1))
    tol = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -12 + 2.0 ** -11 * logit[..., None]) * size
    fine = ((out.cpu().double() - want).abs() <= tol + 1e-30) | torch.isnan(want)
    assert bool(fine[rows].all())


@pytest.mark.parametrize("T,Hq,H,D,dtype", [(1, 4, 2, 64, BF), (7, 4, 2, 128, FP), (650, 8, 8, 64, BF),
                                            (700, 16, 16, 128, FP), (700, 16, 16, 64, BF)])
def test_attention_far_logits(T, Hq, H, D, dtype):
    """Logits up to hundreds, growing from page to page, and rows whose first page comes late: the
    reference of a row moves while its neighbours' stay.  One channel alone is not zero, so that
    a logit is a single product and exact; its weight then has the weights' bound alone."""
    from flashvsr_sm89_ops import selected_attention
    P = 12
    lengths = [max(P * 128 - 5, T + 900)]
    P = -(-lengths[0] // 128)
    table, N = tables(lengths, seed=1)
    pages = pool(N, H, D, seed=2)
    k = torch.zeros(N, H, 128, D)
    for j in range(P):
        k[int(table[0, j]), :, :, 0] = float(2 ** (j % 9)) * (-1) ** (j // 9)
    pages.k.copy_(k.to(torch.float8_e4m3fn))
    pages.k_scale.view(torch.uint8).fill_(127)
    q = torch.zeros(T, Hq, D, dtype=dtype)
    q[..., 0] = torch.tensor([1.0, 2.5, -1.75, 0.25])[torch.arange(T * Hq) % 4].reshape(T, Hq).to(dtype)
    cols = random_columns(T, H, 4, lengths, [T], seed=4)
    out = selected_attention(q.to(DEV), pages, table.to(DEV), i32(lengths).to(DEV), cols.to(DEV),
                             sm_scale=1.0)
    rows = torch.arange(0, T, 1 if T < 20 else 31)
    keep = torch.isin(torch.arange(T), rows)[:, None, None]
    want, size, _ = S.attended(q, O.from_pages(*pages), table, lengths, torch.where(keep, cols, -1),
                               sm_scale=1.0)
    # exp2 of a logit in log2 units: its product's fp32 rounding, 2^-24 * 1000 of them, is 2^-14
    # of a weight, twice that of a quotient.
    tol = torch.finfo(dtype).eps / 2 * want.abs() + (2.0 ** -8 + 2.0 ** -12 + 2.0 ** -13) * size
    assert bool(((out.cpu().double() - want).abs() <= tol + 1e-30)[rows].all())


@pytest.mark.parametrize("Hq,H,D,dtype", [(8, 8, 64, BF), (8, 4, 128, FP), (16, 16, 128, BF),
                                          (32, 16, 64, FP)])
def test_attention_many_packed_rows(Hq, H, D, dtype):
    """Packed chunks and single tokens in one call, four waves or one to a unit; rows behind the last
    sequence are zeros, or left alone in `out`."""
    from flashvsr_sm89_ops import KVPages, selected_attention
    new, lengths = [300, 0, 1, 417, 2], [300, 128, 900, 1300, 2]
    T = sum(new) + 3
    columns = 11
    table = torch.arange(5 * columns).reshape(5, columns).int()
    k, v, ks, vs = O.counting_pool(5 * columns, H, D, table, most=3)
    e4 = torch.float8_e4m3fn
    pages = KVPages(k.to(DEV).view(e4), v.to(DEV).view(e4), ks.to(DEV).view(E8), vs.to(DEV).view(E8))
    q = torch.zeros(T, Hq, D, dtype=dtype)
    q[..., 0] = 1
    cols = random_columns(T, H, 4, lengths, new, seed=1)
    args = (q.to(DEV), pages, table.to(DEV), i32(lengths).to(DEV), cols.to(DEV), starts(new).to(DEV))
    out = selected_attention(*args, sm_scale=math.log(2))
    want = S.counted(T, Hq, H, D, table, lengths, cols, starts(new), most=3)
    assert O.counts_agree(out.cpu(), want)
    assert bool((out[-3:] == 0).all())
    given = torch.full_like(out, 7.0)
    selected_attention(*args, sm_scale=math.log(2), out=given)
    assert torch.equal(given[:-3], out[:-3]) and bool((given[-3:] == 7).all())


@pytest.mark.parametrize("T,H,D", [(1, 8, 64), (700, 8, 64), (700, 16, 64), (700, 16, 128)])
def test_attention_bad_pages_and_hidden_nan(T, H, D):
    """Page ids outside the pool make the rows that list them NaN; what lies behind a row's
    position, and pages that it does not list, may hold NaN."""
    from flashvsr_sm89_ops import selected_attention
    lengths = [T + 300]
    table, N = tables(lengths, seed=1)
    pages = pool(N, H, D, seed=2)
    P = table.shape[1]
    last = int(table[0, P - 1])
    pages.k[last, :, lengths[0] % 128:] = math.nan
    pages.v[last, :, :, lengths[0] % 128:] = math.nan
    pages.k[int(table[0, 1])] = math.nan
    table[0, 0] = N + 5
    cols = random_columns(T, H, 3, lengths, [T], seed=4)
    cols = torch.where(cols == 1, 2, cols)                     # column 1 is all NaN
    cols[:, 1:] = torch.where(cols[:, 1:] == 0, -1, cols[:, 1:])   # head 0 alone lists column 0
    q = torch.randn(T, H, D, generator=gen(3)).bfloat16()
    out = selected_attention(q.to(DEV), pages, table.to(DEV), i32(lengths).to(DEV), cols.to(DEV))
    reads = (cols[:, 0] == 0).any(-1)
    assert bool(torch.isnan(out.cpu()[:, 0][reads]).all()) and int(reads.sum()) > 0
    assert bool(torch.isfinite(out.cpu()[:, 1:]).all())
    check_attention(out, q, pages, table, lengths, cols)


@pytest.mark.parametrize("Hq,H,D,dtype", [(1, 1, 128, BF), (4, 1, 64, FP), (10, 2, 128, BF), (3, 1, 64, BF)])
@pytest.mark.parametrize("where", ["k", "v", "k_scale", "v_scale"])
def test_attention_neighbours_of_nan(Hq, H, D, dtype, where):
    """A NaN in a page is for the rows that list it and see it, and for none of the rows beside them."""
    from flashvsr_sm89_ops import selected_attention
    T, lengths = 50, [900]
    table, N = tables(lengths, seed=1)
    pages = pool(N, H, D, seed=2)
    for col in (1, 4, 7):
        page = int(table[0, col])
        if where == "k":
            pages.k[page, :, 5, 3] = math.nan
        elif where == "v":
            pages.v[page, :, 3, 3] = math.nan
        else:
            getattr(pages, where).view(torch.uint8)[page] = 255
    pages.v[int(table[0, 6]), :, 9, 100] = math.nan          # position 868: behind the first rows
    cols = random_columns(T, H, 3, lengths, [T], seed=4)
    q = torch.randn(T, Hq, D, generator=gen(3)).to(dtype)
    out = selected_attention(q.to(DEV), pages, table.to(DEV), i32(lengths).to(DEV), cols.to(DEV))
    clean = ~torch.isnan(out.cpu()).any(-1).all(-1)
    assert 0 < int(clean.sum()) < T
    check_attention(out, q, pages, table, lengths, cols)


@pytest.mark.parametrize("Hq,H,D,dtype", [(16, 16, 128, BF), (16, 16, 64, FP), (32, 16, 128, FP),
                                          (48, 16, 64, BF), (8, 8, 128, FP)])
@pytest.mark.parametrize("wild", [False, True])
@pytest.mark.parametrize("where", ["", "k", "v", "k_scale", "v_scale"])
def test_attention_many_units(Hq, H, D, dtype, wild, where):
    """Units of one, two or four waves, in lists of any kind, with NaN in some of the pages."""
    from flashvsr_sm89_ops import selected_attention
    T, lengths = 700, [1500]
    table, N = tables(lengths, seed=1)
    pages = pool(N, H, D, seed=2)
    for col in (1, 7):
        page = int(table[0, col])
        if where in ("k", "v"):
            getattr(pages, where)[page, :, 5, 3] = math.nan
        elif where:
            getattr(pages, where).view(torch.uint8)[page] = 255
    cols = random_columns(T, H, 4, lengths, [T], seed=4, wild=wild)
    q = torch.randn(T, Hq, D, generator=gen(3)).to(dtype)
    out = selected_attention(q.to(DEV), pages, table.to(DEV), i32(lengths).to(DEV), cols.to(DEV))
    rows = torch.cat([torch.arange(3, T, 37), torch.arange(T - 3, T)])
    if where:
        some = torch.isnan(out.cpu()[rows]).any(-1)
        assert bool(some.any()) and not bool(some.all())
    check_attention(out, q, pages, table, lengths, cols, rows=rows)


@pytest.mark.parametrize("T,Hq,H,D", [(1, 16, 2, 64), (1, 16, 2, 128), (5, 8, 2, 64), (5, 8, 2, 128),
                                      (700, 8, 8, 64), (700, 16, 16, 64), (700, 8, 8, 128),
                                      (700, 16, 16, 128), (1100, 16, 16, 128)])
def test_attention_bits_of_half_weights(T, Hq, H, D):
    """fp16: a weight is within 2^-12 of itself.  Two tokens count, one with the weight 1 (a power of two,
    so exact in any terms) and V of -1, one with e^x, x small, and V of 1: o = tanh(x / 2), off by 2^-12
    e^x / (1 + e^x) where the weight is off by 2^-12 of itself, and half a step of the output.  (x is one
    product of 11 bits with sm_scale 1; the hidden tokens' logits are -7168, weights of 0; exp2
    and the sums in fp32 are off by less than 2^-18.)"""
    from flashvsr_sm89_ops import selected_attention
    lengths = [T + 200]
    table, N = tables(lengths, seed=1)
    pages = pool(N, H, D, seed=2)
    k = torch.zeros(N, H, 128, D)
    k[:, :, 0, 0] = 1.0
    k[:, :, 2:, 1] = -448.0
    v = torch.ones(N, H, D, 128)
    v[..., 1] = -1.0
    pages.k.copy_(k.to(torch.float8_e4m3fn))
    pages.v.copy_(v.to(torch.float8_e4m3fn))
    for s in pages[2:]:
        s.view(torch.uint8).fill_(127)
    q = torch.zeros(T, Hq, D, dtype=FP)
    x = 0.001 + 0.01 * torch.rand(T, Hq, generator=gen(3))
    q[..., 0], q[..., 1] = x.half(), 16.0
    cols = torch.zeros(T, H, 1, dtype=torch.int32)
    out = selected_attention(q.to(DEV), pages, table.to(DEV), i32(lengths).to(DEV), cols.to(DEV),
                             sm_scale=1.0).cpu().double()
    want = torch.tanh(q[..., :1].double() / 2).expand(T, Hq, D)
    share = torch.sigmoid(q[..., :1].double())
    tol = 2.0 ** -12 * share + 2.0 ** -11 * want.abs() + 2.0 ** -18
    assert bool(((out - want).abs() <= tol).all()), float(((out - want).abs() / tol).max())


def test_attention_nothing():
    from flashvsr_sm89_ops import selected_attention
    lengths = [300, 128]
    table, N = tables(lengths)
    pages = pool(N, 2, 64)
    q = torch.randn(4, 4, 64, device=DEV).bfloat16()
    t, n, c = table.to(DEV), i32(lengths).to(DEV), torch.zeros(4, 2, 3, dtype=torch.int32, device=DEV)
    for cols in (c[..., :0], torch.full_like(c, -1), torch.full_like(c, 99)):
        assert bool((selected_attention(q, pages, t, n, cols.contiguous()) == 0).all())
    assert selected_attention(q[:0], pages, t, n, c[:0]).shape == (0, 4, 64)
    assert bool((selected_attention(q, pages, t[:0], n[:0], c, starts([]).to(DEV)) == 0).all())


def test_same_as_dense_where_all_is_listed():
    """With every column listed, the result is paged_attention's to the bounds of both."""
    from flashvsr_sm89_ops import paged_attention, selected_attention
    lengths = [500, 1000]
    table, N = tables(lengths)
    pages = pool(N, 2, 128)
    q = torch.randn(2, 8, 128, generator=gen(0)).half()
    cols = torch.arange(8, dtype=torch.int32).expand(2, 2, 8).contiguous()
    args = (q.to(DEV), pages, table.to(DEV), i32(lengths).to(DEV))
    out = selected_attention(*args, cols.to(DEV))
    check_attention(out, q, pages, table, lengths, cols)
    assert float((out - paged_attention(*args)).abs().max()) < 2.0 ** -9


def test_far_pages():
    """Offsets past 32 bits: pages at the end of a pool of 2.3 GB of keys."""
    from flashvsr_sm89_ops import (KVPages, PageMeans, pool_pages, select_pages, selected_attention)
    N, H, D = 140000, 1, 128
    e4 = torch.float8_e4m3fn
    k, v = (torch.zeros(s, dtype=torch.uint8, device=DEV) for s in ((N, H, 128, D), (N, H, D, 128)))
    s = torch.full((N, H), 120, dtype=torch.uint8, device=DEV)
    small = pool(12, H, D, seed=3)
    k[-12:], v[-12:] = small.k.view(torch.uint8), small.v.view(torch.uint8)
    pages = KVPages(k.view(e4), v.view(e4), s.view(E8), s.view(E8))
    near = KVPages(small.k, small.v, s[-12:].view(E8), s[-12:].view(E8))
    means = PageMeans(torch.zeros(N, H, D, dtype=torch.int8, device=DEV), torch.zeros_like(s).view(E8))
    few = PageMeans(means.mean[:12].clone(), means.scale[:12].clone())
    table = torch.arange(12).flip(0)[None].int().to(DEV)
    n = i32([12 * 128 - 3]).to(DEV)
    q = torch.randn(1, 4, D, generator=gen(1)).bfloat16().to(DEV)
    got = []
    for p, m, t in ((pages, means, table + N - 12), (near, few, table)):
        pool_pages(m, p, t, n)
        cols = select_pages(q, m, t, n, top=5)
        got.append((m.mean[-12:], cols, selected_attention(q, p, t, n, cols)))
    assert all(torch.equal(a, b) for a, b in zip(*got))


# --------------------------------------------------------------------------------------


def steps(B, H, Hq, D, prompt, n_steps, capture=False):
    """A prompt, then tokens one at a time; everything on the GPU.  Yields what a step read and gave."""
    from flashvsr_sm89_ops import (append_kv, kv_pages, page_means, pool_pages, rotary,
                                   rotary_frequencies, select_pages, selected_attention)
    g = gen(1)
    P = -(-(prompt + n_steps) // 128)
    pages = kv_pages(B * P + 1, H, D, device=DEV)
    means = page_means(pages)
    freqs = rotary_frequencies(D // 2, 500.0, scaling="parts", factor=4.0, context=200)
    table = torch.randperm(B * P + 1, generator=g)[:B * P].reshape(B, P).int().to(DEV)
    lengths = torch.zeros(B, dtype=torch.int32, device=DEV)
    for n in [prompt] + [1] * n_steps:
        x = torch.randn(B * n, Hq + 2 * H, D, generator=g).bfloat16().to(DEV)
        lengths += n
        pos = (lengths[:, None] - n + torch.arange(n, device=DEV, dtype=torch.int32)).reshape(-1).int()
        q, k = rotary(x[:, :Hq], x[:, Hq:Hq + H], freqs, pos, pairs="half")
        append_kv(pages, k, x[:, Hq + H:], table, lengths)
        pool_pages(means, pages, table, lengths, tokens=B * n)
        cols = select_pages(q, means, table, lengths, top=4, first=1, recent=1)
        out = selected_attention(q, pages, table, lengths, cols)
        yield x, freqs, pos, q, k, pages, means, table, lengths, cols, out


def test_together_as_used():
    """Rotation, append, means, choice and attention, from a prompt over page borders: each result
    against its definition on what the step before it gave."""
    B, H, Hq, D = 2, 2, 4, 64
    for x, freqs, pos, q, k, pages, means, table, lengths, cols, out in steps(B, H, Hq, D, 1020, 6):
        n, L = x.shape[0] // B, lengths.tolist()
        turns = freqs.turns.cpu()
        want = S.rotated(x[None, :, :Hq + H].cpu(), turns, freqs.gain, pos.cpu(), "half")[0]
        got = torch.cat([q, k], 1).cpu().double()
        assert bool(((got - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -20).all())
        t, cache = table.cpu(), O.from_pages(*pages)
        mean, scale = means.mean.cpu().zero_(), bytes_of(means.scale).zero_()
        S.pooled(mean, scale, cache, bytes_of(pages.k_scale), t, L, None)
        full = torch.cat([t[b, :L[b] // 128] for b in range(B)]).long()
        assert torch.equal(means.mean.cpu()[full], mean[full])
        assert torch.equal(bytes_of(means.scale)[full], scale[full])
        rows = torch.arange(0, x.shape[0], 37 if n > 1 else 1)
        want = S.selected(q.cpu().double(), means.mean.cpu(), bytes_of(means.scale), t, L, 4, 1, 1)
        assert torch.equal(cols.cpu(), want)
        want, size, logit = S.attended(q.cpu(), cache, t, L, cols.cpu())
        tol = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -12 + 2.0 ** -11 * logit[..., None]) * size
        assert bool(((out.cpu().double() - want).abs() <= tol + 1e-30)[rows].all())


def test_graph_and_stream():
    """A step captured on a stream of its own replays with lengths that grow over a page's end, between
    eager work of the same pool; each replay equals eager calls."""
    from flashvsr_sm89_ops import (append_kv, kv_pages, page_means, pool_pages, rotary,
                                   rotary_frequencies, select_pages, selected_attention)
    B, H, Hq, D, P = 3, 2, 8, 128, 12
    freqs = rotary_frequencies(D)
    table = torch.randperm(B * P, generator=gen(1)).reshape(B, P).int().to(DEV)
    x = torch.empty(B, Hq + 2 * H, D, dtype=BF, device=DEV)

    def state():
        pages = kv_pages(B * P, H, D, device=DEV)
        g = torch.Generator(device=DEV).manual_seed(2)
        for c in pages[:2]:
            c.copy_(torch.randn(c.shape, device=DEV, generator=g).to(c.dtype))
        for c in pages[2:]:
            c.view(torch.uint8).fill_(127)
        lengths = i32([1150, 1151, 700]).to(DEV)
        return pages, pool_pages(page_means(pages), pages, table, lengths), lengths

    def step(pages, means, lengths):
        lengths += 1
        q, k = rotary(x[:, :Hq], x[:, Hq:Hq + H], freqs, lengths)
        append_kv(pages, k, x[:, Hq + H:], table, lengths)
        pool_pages(means, pages, table, lengths, tokens=B)
        cols = select_pages(q, means, table, lengths, top=4)
        return cols, selected_attention(q, pages, table, lengths, cols)

    a, b = state(), state()
    x.normal_(generator=torch.Generator(device=DEV).manual_seed(0))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = step(*b)
    torch.cuda.current_stream().wait_stream(side)
    for i in range(5):
        x.normal_(generator=torch.Generator(device=DEV).manual_seed(i))
        want = step(*a)
        graph.replay()
        torch.cuda.synchronize()
        for u, v in zip((*want, *a[0], *a[1]), (*got, *b[0], *b[1])):
            assert torch.equal(u.view(torch.uint8), v.view(torch.uint8)), i


@pytest.mark.parametrize("H,D", [(8, 64), (16, 128)])
def test_graph_of_a_chunk(H, D):
    """A chunk's pooling, choice and attention captured, replayed as lengths and pages change."""
    from flashvsr_sm89_ops import page_means, pool_pages, select_pages, selected_attention
    Hq, T = H, 700
    table, N = tables([3000])
    pages = pool(N, H, D)
    means, t = page_means(pages), table.to(DEV)
    n = i32([2000]).to(DEV)
    q = torch.randn(T, Hq, D, device=DEV).half()

    def step():
        pool_pages(means, pages, t, n)
        cols = select_pages(q, means, t, n, top=5)
        return cols, selected_attention(q, pages, t, n, cols)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = step()
    torch.cuda.current_stream().wait_stream(side)
    for i, length in enumerate((2000, 2500, 701, 3000)):
        n.fill_(length)
        q.normal_()
        graph.replay()
        torch.cuda.synchronize()
        got_now = [x.clone() for x in got]
        assert all(torch.equal(a, b) for a, b in zip(step(), got_now)), i


def test_two_streams():
    """Calls on two streams at once, each with pieces of its own, give what they give alone."""
    from flashvsr_sm89_ops import select_pages, selected_attention
    H, Hq, D = 2, 8, 128
    table, N = tables([9000, 8000])
    pages, means = pool(N, H, D), random_means(N, H, D)
    t, n = table.to(DEV), i32([9000, 8000]).to(DEV)
    qs = [torch.randn(2, Hq, D, generator=gen(i)).bfloat16().to(DEV) for i in range(2)]

    def step(q):
        cols = select_pages(q, means, t, n, top=40)
        return selected_attention(q, pages, t, n, cols)
    want = [step(q) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    got = [[] for _ in qs]
    for _ in range(10):
        for s, q, g in zip(streams, qs, got):
            with torch.cuda.stream(s):
                g.append(step(q))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(w, x) for x in g)


def test_native_and_general_path(monkeypatch):
    """The native host path serves these calls and gives what the general one does."""
    from flashvsr_sm89_ops import (RotaryFrequencies, _lib, page_means, pool_pages, rotary,
                                   select_pages, selected_attention)
    H, D, B = 2, 128, 3
    lengths = [1400, 1300, 20]
    table, N = tables(lengths)
    q = torch.randn(B * 7, 4, D, generator=gen(1)).bfloat16().to(DEV)
    k = torch.randn(B * 7, 2, D, generator=gen(2)).bfloat16().to(DEV)
    f = RotaryFrequencies(torch.rand(32, generator=gen(3)).double().to(DEV), 1.5)
    pos = torch.randint(0, 99, (B, 7), generator=gen(4)).int().to(DEV)
    pages, t, n = pool(N, H, D), table.to(DEV), i32(lengths).to(DEV)
    cu = starts([7] * B).to(DEV)
    host, got = _lib.selected_host(), []
    assert host is not _lib._GeneralPath
    for general in (False, True):
        monkeypatch.setattr(_lib, "_selected_host", _lib._GeneralPath if general else host)
        means = pool_pages(page_means(pages), pages, t, n)
        pool_pages(means, pages, t, n, cu, tokens=B * 7)
        cols = select_pages(q, means, t, n, top=5, first=0, recent=2)
        r = [*means, cols, select_pages(q, means, t, n, cu, top=5)]
        r += [selected_attention(q, pages, t, n, cols),
              selected_attention(q, pages, t, n, cols, cu, sm_scale=0.3)]
        r += [*rotary(q, k, f), rotary(q, None, f, pairs="interleaved"),
              rotary(q.view(B, 7, 4, D), None, f, pos)]
        got.append([x.view(torch.uint8) for x in r])
    assert all(torch.equal(a, b) for a, b in zip(*got))
    c = (means, pages, t, n, None, 21)
    assert host.pool_pages(*c) is means and host.pool_pages(*c[:5], None) is means
    for i, bad in ((0, means[:1]), (0, (means.mean[:2], means.scale[:2])), (1, pages[:3]),
                   (2, t.long()), (3, n[:2]), (4, n), (5, 20), (5, -1), (5, 2.0), (5, 1 << 70)):
        assert host.pool_pages(*c[:i], bad, *c[i + 1:]) is None, i
    c = (q, means, t, n, None, 5, 1, 1)
    assert host.select_pages(*c).shape == (B * 7, H, 5)
    for i, bad in ((0, q.float()), (0, q[:, :3]), (0, q[..., :64]), (0, q.cpu()), (1, means[:1]),
                   (2, t[:2]), (5, 1), (5, 5.0), (5, 1 << 30), (6, -1), (7, 0)):
        assert host.select_pages(*c[:i], bad, *c[i + 1:]) is None, i
    c = (q, pages, t, n, cols, None, None)
    assert host.selected_attention(*c).shape == q.shape
    for i, bad in ((0, q.float()), (1, pages[:3]), (4, cols.long()), (4, cols[:, :1]),
                   (4, cols[..., ::2]), (5, n), (6, 0.0)):
        assert host.selected_attention(*c[:i], bad, *c[i + 1:]) is None, i
    c = (q, k, f, None, "half")
    assert len(host.rotary(*c)) == 2
    for i, bad in ((0, q.double()), (0, q[:5]), (0, q.transpose(1, 2)), (1, k.float()),
                   (1, k[..., :64]), (2, f[:1]), (2, (f.turns.float(), 1.0)), (3, pos),
                   (3, pos[0].long()), (4, "other"), (4, 3)):
        assert host.rotary(*c[:i], bad, *c[i + 1:]) is None, i


def test_dispatch_modes():
    """A call inside a dispatch mode goes by the general path and is seen by it."""
    from torch.utils._python_dispatch import TorchDispatchMode

    from flashvsr_sm89_ops import rotary, rotary_frequencies

    class Seen(TorchDispatchMode):
        names = []

        def __torch_dispatch__(self, f, types, args=(), kwargs=None):
            self.names.append(str(f))
            return f(*args, **(kwargs or {}))
    x = torch.randn(3, 2, 64, device=DEV)
    f = rotary_frequencies(64)
    want = rotary(x, None, f)
    with Seen():
        got = rotary(x, None, f)
    assert torch.equal(got, want) and any("empty" in n for n in Seen.names)
