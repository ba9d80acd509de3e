"""append_kv and paged_attention at the edges of what their documentation allows."""
import math

import pytest
import torch

from test_gpu_paged_kv import DEV, check_q, freqs_of, gen, i32, pool

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
