"""append_kv and paged_attention at the edges of what their documentation allows."""
import math

import pytest
import torch

from oracle import paged_kv as O
from test_gpu_paged_kv import (DEV, check_append, check_attention, check_q, freqs_of, gen, i32,
                               pool, starts, tables)

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


def above_border(x, rms, low):
    """Weights with which each x * w / rms (x nonzero) lies less than two fp32 steps above
    the border `low` between two codes, in 64 bits."""
    w = torch.where(x == 0, 1.0, low * rms / x.abs().double().clamp(min=1e-30)).float()
    under = (x.abs().double() * w.double() / rms <= low) & (x != 0)
    return torch.where(under, torch.nextafter(w, torch.full_like(w, math.inf)), w)


@pytest.mark.parametrize("D,H", [(64, 256), (128, 128)])
@pytest.mark.parametrize("n", [1, 5, 20])
def test_append_row_norm_codes_next_to_a_border(D, H, n):
    """A row whose squares add up badly in fp32: a lane's sum starts at 1, and each of the
    31 squares behind it, a little over half a step, counts as a whole one.  That is 31 * 2^-24 of
    the sum and half of it, 15 steps, in each value; their codes are those of the 64-bit value."""
    from flashvsr_sm89_ops import append_kv
    x = torch.zeros(H * D // 512, 64, 8)  # [turn of a wave, lane, element]
    x[0, :, 0] = 1.0
    x[1:, :, 0] = 2.0 ** -12 * (1 + 2.0 ** -10)
    x = x.reshape(H * D)
    rms = math.sqrt(float((x.double() ** 2).mean()) + 1e-6)
    w = above_border(x, rms, 1.9375)
    T = 2 * n
    k = torch.where(torch.rand(T, H * D, generator=gen(n)) < 0.5, x, -x).view(T, H, D)
    table, N = tables([n, n])
    pages = pool(N, H, D)
    append_kv(pages, k.to(DEV), k.to(DEV), table.to(DEV), i32([n, n]).to(DEV), k_weight=w.to(DEV))
    got = O.from_pages(*pages)
    for b in range(2):
        page = int(table[b, 0])
        s = torch.exp2(got["ke"][page].double())[:, None, None]
        y = O.turned(k[b * n:(b + 1) * n], w, None, None, 1e-6).transpose(0, 1)
        assert torch.equal(got["k"][page, :, :n], O.e4m3(y / s))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,norm", [(1100, "head"), (1, "head"), (5, "head"), (1, "row"),
                                    (5, "row"), (30, "row")])
def test_append_codes_of_64_bits_with_norms(D, dtype, norm, n):
    """Codes are those of the 64-bit value where the rotation leaves 0.7 of its terms, for the
    norms and counts of tokens whose sums are taken beside the values."""
    from flashvsr_sm89_ops import append_kv
    H, B = 4, 1 if n > 8 else 300
    lens = [n + 70] * B
    table, N = tables(lens, seed=3)
    pages, g = pool(N, H, D, seed=4), gen(D + n)
    k = torch.randn(B * n, H, D, generator=g).to(dtype)
    freqs = freqs_of(2000, D)
    pos = torch.randint(0, 2000, (B * n,), generator=g).int()
    kw = 1 + 0.1 * torch.randn(D * (H if norm == "row" else 1), generator=g)
    append_kv(pages, k.to(DEV), k.to(DEV), table.to(DEV), i32(lens).to(DEV),
              freqs_cis=freqs.to(DEV), positions=pos.to(DEV), k_weight=kw.to(DEV))
    after = O.from_pages(*pages)
    x = O.turned(k, kw, freqs, pos, 1e-6)
    a = O.turned(k, kw, None, None, 1e-6).abs()
    size = (a[..., 0::2] + a[..., 1::2]).repeat_interleave(2, -1)
    t = torch.arange(B * n)
    b, p = t // n, 70 + t % n
    page = table[b, p // 128].long()
    y = x / torch.exp2(after["ke"][page].double())[..., None]
    plain = (x.abs() >= 0.7 * size) & (y.abs() >= 2.0 ** -6)
    assert float(plain.double().mean()) > 0.2
    assert torch.equal(after["k"][page, :, p % 128][plain], O.e4m3(y)[plain])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("norm", ["head", "row"])
@pytest.mark.parametrize("n", [1, 5, 30, 100])
@pytest.mark.parametrize("size", [1e-30, 1e25, 1e38])
def test_append_norm_of_far_values(D, norm, n, size):
    """Keys whose squares fp32 does not hold are normed as any others."""
    from flashvsr_sm89_ops import append_kv
    H, g = 4, gen(n)
    table, N = tables([n])
    pages = pool(N, H, D)
    before = O.from_pages(*pages)
    k = (torch.randn(n, H, D, generator=g) * size).clamp(-3e38, 3e38).bfloat16()
    v = torch.randn(n, H, D, generator=g).bfloat16()
    kw = 1 + 0.2 * torch.randn(D * (H if norm == "row" else 1), generator=g)
    eps = 1e-70 if size < 1 else 1e-6  # (fp32: 0)
    append_kv(pages, k.to(DEV), v.to(DEV), table.to(DEV), i32([n]).to(DEV), k_weight=kw.to(DEV),
              eps=eps)
    check_append(pages, before, k, v, table, [n], None, None, None, kw, 0.0 if size < 1 else eps)


def test_append_double_rotations_are_not_kept():
    """A complex128 table is read as it is at the call: changed behind autograd's back, first
    used by a captured call, made in inference mode."""
    from flashvsr_sm89_ops import append_kv
    H, D, T, g = 2, 64, 20, gen(1)
    table, N = tables([T])
    pages = pool(N, H, D)
    q, k = (torch.randn(T, H, D, generator=g).bfloat16() for _ in range(2))
    dq, dk, t, n = q.to(DEV), k.to(DEV), table.to(DEV), i32([T]).to(DEV)
    host = freqs_of(2 * T, D).to(torch.complex128)
    fr = host[:T].to(DEV)

    def step():
        return append_kv(pages, dk, dk, t, n, freqs_cis=fr, q=dq)
    pos = torch.arange(T)
    check_q(step(), q, host[:T], pos, None)
    fr.data.copy_(host[T:])
    check_q(step(), q, host[T:], pos, None)
    # A call that is captured first, and an eager one before any replay.
    fr = host[:T].to(DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    check_q(step(), q, host[:T], pos, None)
    for rows in (host[T:], host[:T], host[T:]):
        fr.copy_(rows)
        graph.replay()
        check_q(out, q, rows, pos, None)
        check_q(step(), q, rows, pos, None)
    with torch.inference_mode():
        fr = host[:T].to(DEV) * 1
        check_q(step(), q, host[:T], pos, None)
    for dtype in (torch.complex64, torch.complex128):
        fr = host[:T].to(dtype).to(DEV).conj()
        check_q(step(), q, host[:T].conj(), pos, None)


@pytest.mark.parametrize("n", [1, 5, 9])
def test_append_lengths_near_two_billion(n):
    """Positions up to 2^31 - 1 lie past every table: nothing is stored, and q comes back."""
    from flashvsr_sm89_ops import append_kv
    H, D = 2, 64
    pages = pool(4, H, D)
    before = [p.view(torch.uint8).clone() for p in pages]
    q = torch.randn(3 * n, H, D, generator=gen(n)).bfloat16()
    d = q.to(DEV)
    table = i32([[0, 1], [2, 3], [0, 1]]).to(DEV)
    lengths = i32([2 ** 31 - 1, 2 ** 31 - 3, 2 ** 31 - 128]).to(DEV)
    for cu in (None, starts([n, n, n]).to(DEV)):
        assert torch.equal(append_kv(pages, d, d, table, lengths, cu, q=d), d)
    assert all(torch.equal(a, b.view(torch.uint8)) for a, b in zip(before, pages))


@pytest.mark.parametrize("n,Hq", [(1, 1), (2, 2), (20, 1)])
def test_attention_of_many_sequences(n, Hq):
    """More sequences of few rows than a grid's third dimension holds."""
    from flashvsr_sm89_ops import paged_attention
    B, D, some = 66000, 64, 6
    lens = [200, n, 0, 129, 128, 1]
    table, N = tables(lens)
    pages = pool(N, 1, D)
    q = torch.randn(some * n, Hq, D, generator=gen(n)).bfloat16()
    t, L = table.repeat(B // some, 1).to(DEV), i32(lens).repeat(B // some).to(DEV)
    out = paged_attention(q.to(DEV).repeat(B // some, 1, 1), pages, t, L)
    check_attention(out[:some * n], q, pages, table, lens)
    assert torch.equal(out.view(B // some, some * n, Hq, D),
                       out[:some * n].expand(B // some, -1, -1, -1))
