"""The check by counted tokens: it takes the definition's own outputs and sees every page, piece and
token left out or taken twice, at the lengths at which the kernels are checked."""
import math

import pytest
import torch

from oracle import paged_kv as O


def cache_of(N, H, D, table, most=0):
    k, v, ks, vs = O.counting_pool(N, H, D, table, most=most)
    e4, e8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
    return O.from_pages(k.view(e4), v.view(e4), ks.view(e8), vs.view(e8))


@pytest.mark.parametrize("D,H,Hq,dtype", [(64, 2, 4, torch.bfloat16), (128, 1, 2, torch.float16)])
@pytest.mark.parametrize("causal", [True, False])
def test_definition_is_taken(D, H, Hq, dtype, causal):
    lens, new = [300, 0, 128, 129], [140, 3, 0, 129]
    table = torch.randperm(12, generator=torch.Generator().manual_seed(1)).int().view(4, 3)
    T, cu = sum(new), torch.tensor([0] + new).cumsum(0)
    keep = torch.rand(4, Hq, 2, 3, generator=torch.Generator().manual_seed(2)) < 0.6
    q = torch.randn(T, Hq, D, generator=torch.Generator().manual_seed(3)).to(dtype)
    for k in (None, keep):
        out = O.attention(q, cache_of(12, H, D, table), table, lens, cu, causal, k)[0]
        want = O.counted(T, Hq, H, D, 3, lens, cu, causal, k)
        assert float((out - want).abs().max()) < 1e-12
        assert O.counts_agree(out.to(dtype), want)
    q[..., 0] = 1.0
    for most in (3, 20):
        cache = cache_of(12, H, D, table, most)
        out = O.attention(q, cache, table, lens, cu, causal, keep, math.log(2))[0]
        want = O.counted(T, Hq, H, D, 3, lens, cu, causal, keep, most)
        assert float((out - want).abs().max()) < 1e-12 and O.counts_agree(out.to(dtype), want)


def test_pool_holds_its_numbers():
    """Every lift and value is a code times its scale, whatever the scale."""
    table = torch.arange(600).int().view(1, 600)
    c = cache_of(600, 3, 64, table, 20)
    for h in range(3):
        k, v = (c[a][:, h] * torch.exp2(c[e][:, h].double())[:, None, None]
                for a, e in (("k", "ke"), ("v", "ve")))
        assert torch.equal(k[..., 0], torch.tensor([[float(O.lift(j, h, 20))] * 128
                                                    for j in range(600)]).double())
        assert int((k[..., 1:] != 0).sum()) == 0 and set(v.unique().tolist()) == {0.0, 1.0}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("pages,splits", [(71, 8), (1100, 64)])
def test_what_is_left_out_is_seen(dtype, D, pages, splits):
    L = 128 * (pages - 1) + 31
    want = O.counted(1, 1, 1, D, pages, [L])
    assert O.counts_agree(want.to(dtype), want)
    tokens = torch.full((pages,), 128.0).double()
    tokens[-1] = 31

    def of(t):
        dims = torch.zeros(pages, D).double()
        dims[torch.arange(pages), torch.arange(pages) % D] = 1
        return (t @ dims / t.sum()).view(1, 1, D).to(dtype)
    assert O.counts_agree(of(tokens), want)
    for j in range(pages):
        for times in (0, 2):
            t = tokens.clone()
            t[j] *= times
            assert not O.counts_agree(of(t), want), (j, times)
    for s in range(splits):  # a piece that is not added
        t = tokens.clone()
        t[pages * s // splits:pages * (s + 1) // splits] = 0
        assert not O.counts_agree(of(t), want), s
    if pages < D:  # (a dim of its own for every page)
        for j in range(pages):
            t = tokens.clone()
            t[j] -= 1
            assert not O.counts_agree(of(t), want), j
