"""paged_attention counting tokens (oracle.counting_pool): every page, piece and token of every
kernel form counts once, with its weight, over tables of up to 1100 pages and up to 150 packed sequences;
and append_kv of as many."""
import math

import pytest
import torch

from oracle import paged_kv as O
from test_gpu_paged_kv import DEV, check_append, gen, i32, pool, starts, tables

pytestmark = pytest.mark.gpu
TYPES = [(64, torch.bfloat16), (128, torch.bfloat16), (64, torch.float16), (128, torch.float16)]


def check_counts(D, dtype, Hq, H, lens, new, packed, causal=True, keep=None, width=None, tail=0,
                 most=0):
    from flashvsr_sm89_ops import KVPages, paged_attention
    table, N = tables(lens, seed=5, width=width)
    k, v, ks, vs = (t.to(DEV) for t in O.counting_pool(N, H, D, table, most=most))
    e4, e8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
    pages = KVPages(k.view(e4), v.view(e4), ks.view(e8), vs.view(e8))
    T, cu = sum(new) + tail, starts(new) if packed else None
    q = 2 * torch.randn(T, Hq, D, generator=gen(7))
    q[..., 0] = 1.0
    out = paged_attention(q.to(dtype).to(DEV), pages, table.to(DEV), i32(lens).to(DEV),
                          None if cu is None else cu.to(DEV), causal=causal,
                          keep=None if keep is None else keep.to(DEV),
                          sm_scale=math.log(2) if most else None).cpu()
    want = O.counted(T, Hq, H, D, table.shape[1], lens, cu, causal, keep, most)
    assert O.counts_agree(out, want)


@pytest.mark.parametrize("D,dtype", TYPES)
@pytest.mark.parametrize("Hq,H,n", [(3, 3, 1), (8, 2, 1), (2, 1, 8), (2, 2, 17), (8, 2, 5),
                                    (20, 1, 1), (2, 2, 40), (4, 1, 60), (2, 1, 200)])
def test_equal_rows(D, dtype, Hq, H, n):
    """Units of 16 and 32 rows and tiles; a table as wide as the lengths and one far wider."""
    for lens in ([128 * 70 + 31, 300, 0, 128 * 9], [128 * 20 + 1]):
        for width in (None, 700):
            for causal in (True, False):
                check_counts(D, dtype, Hq, H, lens, [n] * len(lens), False, causal, width=width)


@pytest.mark.parametrize("D,dtype", TYPES)
@pytest.mark.parametrize("Hq,H,n", [(4, 2, 1), (5, 1, 4), (1, 1, 150)])
def test_long_axis(D, dtype, Hq, H, n):
    """1100 pages: the most pieces, and more pages than a tile lists at once."""
    check_counts(D, dtype, Hq, H, [128 * 1099 + 31], [n], False)
    check_counts(D, dtype, Hq, H, [128 * 1099 + 31], [n], True, causal=False)


@pytest.mark.parametrize("D,dtype", TYPES)
@pytest.mark.parametrize("most,Hq,H", [(3, 4, 2), (12, 4, 1), (90, 4, 1), (60, 2, 2)])
def test_many_packed_sequences(D, dtype, most, Hq, H):
    """150 sequences, some of no rows, with rows behind the last one."""
    g = gen(most)
    new = torch.randint(0, most + 1, (150,), generator=g).tolist()
    lens = [n + int(x) for n, x in zip(new, torch.randint(0, 2500, (150,), generator=g))]
    lens[3] = 128 * 60 + 77
    for causal in (True, False):
        check_counts(D, dtype, Hq, H, lens, new, True, causal, tail=9)


@pytest.mark.parametrize("D,dtype", TYPES)
@pytest.mark.parametrize("new,Hq", [([2, 1, 0, 5], 4), ([20, 0, 33, 1], 2), ([90, 70, 1, 2], 4),
                                    ([1, 1, 1, 700], 4)])
def test_packed_split(D, dtype, new, Hq):
    """Packed rows, few and many and both, over long and short lengths."""
    lens = [128 * 300 + 3, 900, 50, 128 * 30]
    check_counts(D, dtype, Hq, 2, lens, new, True, tail=5)


@pytest.mark.parametrize("D,dtype", TYPES)
@pytest.mark.parametrize("n", [1, 300])
@pytest.mark.parametrize("share", [0.02, 0.4])
def test_kept_pages(D, dtype, n, share):
    """A block mask over 700 pages."""
    lens = [128 * 699 + 5, 128 * 3]
    keep = torch.rand(2, 4, -(-n // 128), 700, generator=gen(n)) < share
    keep[0, 1, 0] = False
    for causal in (True, False):
        check_counts(D, dtype, 4, 2, lens, [n, n], False, causal, keep)


@pytest.mark.parametrize("D,dtype", TYPES)
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("Hq,H,n", [(2, 2, 1), (4, 1, 5), (2, 2, 40), (4, 1, 150)])
def test_weights_of_pages(D, dtype, packed, Hq, H, n):
    """Pages whose tokens weigh 2^x, x from page to page and head to head: waves, pieces and
    list after list are added at their references.  (fp16: shares within its range.)"""
    most = 20 if dtype == torch.bfloat16 else 3
    check_counts(D, dtype, Hq, H, [128 * 59 + 31, 700], [n, n], packed, most=most)
    check_counts(D, dtype, Hq, H, [128 * 59 + 31, 700], [n, n], packed, False, width=700, most=most)
    check_counts(D, dtype, Hq, H, [128 * 1099 + 31], [n], packed, most=most)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("norm", ["none", "row"])
@pytest.mark.parametrize("most", [1, 40])
def test_append_many_packed_sequences(D, norm, most):
    from flashvsr_sm89_ops import append_kv
    H, g = 2, gen(most)
    new = torch.randint(0, most + 1, (150,), generator=g).tolist()
    lens = [n + int(x) for n, x in zip(new, torch.randint(0, 300, (150,), generator=g))]
    table, N = tables(lens, seed=3)
    pages = pool(N, H, D, seed=4)
    before = O.from_pages(*pages)
    T = sum(new) + 9
    k, v = (torch.randn(T, H, D, generator=g).bfloat16() for _ in range(2))
    kw = 1 + 0.2 * torch.randn(H * D, generator=g) if norm == "row" else None
    append_kv(pages, k.to(DEV), v.to(DEV), table.to(DEV), i32(lens).to(DEV), starts(new).to(DEV),
              k_weight=None if kw is None else kw.to(DEV))
    check_append(pages, before, k, v, table, lens, starts(new), None, None, kw)
