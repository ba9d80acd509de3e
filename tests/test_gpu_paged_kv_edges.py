"""append_kv and paged_attention at the edges of what their documentation allows."""
import math

import pytest
import torch

from oracle import paged_kv as O
from test_gpu_paged_kv import DEV, check_append, check_q, freqs_of, gen, i32, pool, tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("norm", ["none", "head", "row"])
@pytest.mark.parametrize("T", [3, 200])
def test_append_q_without_sequences(D, norm, T):
    """Rows that belong to nobody: q is turned all the same and no page is touched."""
    from flashvsr_sm89_ops import append_kv
    Hq, H, g = 6, 2, gen(D + T)
    pages = pool(3, H, D)
    before = [p.view(torch.uint8).clone() for p in pages]
    q, k = (torch.randn(T, h, D, generator=g).bfloat16() for h in (Hq, H))
    kw = qw = None
    if norm != "none":
        kw = 1 + 0.2 * torch.randn(D * (H if norm == "row" else 1), generator=g)
        qw = 1 + 0.2 * torch.randn(D * (Hq if norm == "row" else 1), generator=g)
    fr, pos = freqs_of(T + 50, D), torch.arange(T).int() + 50
    none = torch.zeros(0, 4, dtype=torch.int32, device=DEV)
    dq, dk = q.to(DEV), k.to(DEV)
    stale = torch.full_like(dq, math.nan)  # what an unwritten result would be made of
    del stale
    out = append_kv(pages, dk, dk, none, none[:, 0], i32([0]).to(DEV), freqs_cis=fr.to(DEV),
                    positions=pos.to(DEV), k_weight=None if kw is None else kw.to(DEV), q=dq,
                    q_weight=None if qw is None else qw.to(DEV))
    check_q(out, q, fr, pos, qw)
    assert append_kv(pages, dk, dk, none, none[:, 0], i32([0]).to(DEV)) is None
    assert all(torch.equal(a, b.view(torch.uint8)) for a, b in zip(before, pages))


SIGNALLING = {torch.bfloat16: (torch.int16, 0x7f81), torch.float16: (torch.int16, 0x7c01),
              torch.float32: (torch.int32, 0x7f800001)}


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", list(SIGNALLING))
@pytest.mark.parametrize("T", [1, 5, 40, 300])
@pytest.mark.parametrize("where", ["some", "last"])
def test_append_signalling_nan(D, dtype, T, where):
    """A NaN that signals is stored as NaN and leaves the scale alone, as any other."""
    from flashvsr_sm89_ops import append_kv
    H, g = 3, gen(T)
    table, N = tables([T])
    pages = pool(N, H, D)
    before = O.from_pages(*pages)
    k, v = (torch.randn(T, H, D, generator=g).to(dtype) for _ in range(2))
    if where == "some":
        at = torch.rand(T, H, D, generator=g) < 0.2
    else:  # the last of every eight, behind all others of a thread
        at = torch.zeros(T, H, D, dtype=torch.bool)
        at[..., 7::8] = True
    integer, bits = SIGNALLING[dtype]
    for x in (k, v):
        x.view(integer)[at] = bits
    append_kv(pages, k.to(DEV), v.to(DEV), table.to(DEV), i32([T]).to(DEV))
    check_append(pages, before, k, v, table, [T], None, None, None, None)
