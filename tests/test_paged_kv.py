"""append_kv and paged_attention on the CPU: what they refuse, in Python and at the C
ABI; nothing here launches a kernel."""
import ctypes
import math

import pytest
import torch

BF, E4, E8, I32 = torch.bfloat16, torch.float8_e4m3fn, torch.float8_e8m0fnu, torch.int32


def cpu_pages(N=4, H=2, D=64):
    from flashvsr_sm89_ops import kv_pages
    return kv_pages(N, H, D, device="cpu")


def append_args(**kw):
    a = dict(pages=cpu_pages(), k=torch.zeros(6, 2, 64, dtype=BF), v=torch.zeros(6, 2, 64, dtype=BF),
             page_table=torch.zeros(2, 3, dtype=I32), lengths=torch.zeros(2, dtype=I32))
    a.update(kw)
    return a


def attend_args(**kw):
    a = dict(q=torch.zeros(6, 4, 64, dtype=BF), pages=cpu_pages(),
             page_table=torch.zeros(2, 3, dtype=I32), lengths=torch.zeros(2, dtype=I32))
    a.update(kw)
    return a


def test_pool():
    p = cpu_pages(3, 2, 128)
    assert p.k.shape == (3, 2, 128, 128) and p.v.shape == (3, 2, 128, 128)
    assert p.k.dtype == E4 and p.k_scale.dtype == E8 and p.v_scale.shape == (3, 2)
    assert cpu_pages(3, 2, 64).v.shape == (3, 2, 64, 128)
    for bad in ((-1, 2, 64), (1, 0, 64), (1, 2, 96)):
        with pytest.raises(ValueError):
            cpu_pages(*bad)


def test_calls_need_a_gpu():
    from flashvsr_sm89_ops import append_kv, paged_attention
    with pytest.raises(RuntimeError, match="GPU only"):
        append_kv(**append_args())
    with pytest.raises(RuntimeError, match="GPU only"):
        paged_attention(**attend_args())


z = torch.zeros
SHARED = [
    (dict(page_table=z(2, 3, dtype=torch.int64)), TypeError),
    (dict(lengths=z(2, dtype=torch.int64)), TypeError),
    (dict(lengths=z(3, dtype=I32)), ValueError),
    (dict(page_table=z(3, 2, dtype=I32).t()), ValueError),
    (dict(page_table=z(3, dtype=I32)), ValueError),
    (dict(page_table=z(1, 3, dtype=I32).expand(2, 3)), ValueError),
    (dict(page_table=z(4, 3, dtype=I32), lengths=z(4, dtype=I32)), ValueError),  # 6 rows over 4
    (dict(cu_tokens=z(2, dtype=I32)), ValueError),
    (dict(cu_tokens=z(3)), TypeError),
]


@pytest.mark.parametrize("change,error", SHARED)
def test_both_refuse(change, error):
    from flashvsr_sm89_ops import append_kv, paged_attention
    with pytest.raises(error):
        append_kv(**append_args(**change))
    with pytest.raises(error):
        paged_attention(**attend_args(**change))


def test_pages_refused():
    from flashvsr_sm89_ops import KVPages, append_kv, paged_attention
    k, v, ks, vs = cpu_pages()
    for p, error in ((KVPages(k, v.transpose(2, 3), ks, vs), ValueError),
                     (KVPages(k, v, ks[:3], vs), ValueError),
                     (KVPages(k[:, :, :64], v, ks, vs), ValueError),
                     (KVPages(k.float(), v, ks, vs), TypeError),
                     (KVPages(k, v, ks.view(torch.uint8), vs), TypeError),
                     (KVPages(k.transpose(0, 1).contiguous().transpose(0, 1), v, ks, vs),
                      ValueError)):
        with pytest.raises(error):
            append_kv(**append_args(pages=p))
        with pytest.raises(error):
            paged_attention(**attend_args(pages=p))


@pytest.mark.parametrize("change,error", [
    (dict(k=z(6, 3, 64, dtype=BF)), ValueError),
    (dict(k=z(6, 2, 32, dtype=BF)), ValueError),
    (dict(v=z(5, 2, 64, dtype=BF)), ValueError),
    (dict(v=z(6, 2, 64)), TypeError),
    (dict(k=z(6, 2, 64, dtype=torch.float64)), TypeError),
    (dict(q=z(6, 4, 64)), TypeError),
    (dict(q=z(4, 4, 64, dtype=BF)), ValueError),
    (dict(q_weight=z(64)), ValueError),
    (dict(k_weight=z(65)), ValueError),
    (dict(k_weight=z(64, dtype=torch.float64)), TypeError),
    (dict(k_weight=z(64), q=z(6, 4, 64, dtype=BF), q_weight=z(64, dtype=BF)), TypeError),
    (dict(positions=z(6, dtype=I32)), ValueError),
    (dict(freqs_cis=z(9, 64)), ValueError),
    (dict(freqs_cis=z(9, 16, dtype=torch.complex64)), ValueError),
    (dict(freqs_cis=z(5, 32, dtype=torch.complex64)), ValueError),
    (dict(freqs_cis=z(0, 32, dtype=torch.complex64), positions=z(6, dtype=I32)), ValueError),
    (dict(freqs_cis=z(9, 32, dtype=torch.complex64), positions=z(6, dtype=torch.int64)), TypeError),
    (dict(freqs_cis=z(9, 32, dtype=torch.complex64), positions=z(5, dtype=I32)), ValueError),
])
def test_append_refuses(change, error):
    from flashvsr_sm89_ops import append_kv
    with pytest.raises(error):
        append_kv(**append_args(**change))


@pytest.mark.parametrize("change,error", [
    (dict(q=z(6, 3, 64, dtype=BF)), ValueError),
    (dict(q=z(6, 4, 32, dtype=BF)), ValueError),
    (dict(q=z(6, 256, dtype=BF)), ValueError),
    (dict(q=z(6, 4, 64)), TypeError),
    (dict(sm_scale=0.0), ValueError),
    (dict(sm_scale=-1.0), ValueError),
    (dict(sm_scale=math.nan), ValueError),
    (dict(sm_scale=math.inf), ValueError),
    (dict(keep=z(2, 4, 1, 3)), TypeError),
    (dict(keep=z(4, 1, 3, dtype=torch.bool)), ValueError),   # two sequences
    (dict(keep=z(2, 2, 1, 3, dtype=torch.bool)), ValueError),
    (dict(out=z(6, 4, 64)), TypeError),
    (dict(out=z(6, 4, 32, dtype=BF)), ValueError),
    (dict(out=z(6, 4, 66, dtype=BF)[..., :64]), ValueError),
])
def test_attention_refuses(change, error):
    from flashvsr_sm89_ops import paged_attention
    with pytest.raises(error):
        paged_attention(**attend_args(**change))


def test_c_entries_check_arguments():
    """Statuses before any launch: device pointers are never followed."""
    from flashvsr_sm89_ops import _lib
    from flashvsr_sm89_ops.paged_kv import _Cache
    L = _lib.lib()
    fake = 1 << 20

    def cache(**kw):
        f = dict(k=fake, v=fake, k_scale=fake, v_scale=fake, pages=4, heads=2, head_dim=128,
                 table=fake, table_stride=3, table_pages=3, lengths=fake, cu=None, sequences=2)
        f.update(kw)
        return ctypes.byref(_Cache(**f))

    def append(c=None, k=fake, ts=256, hs=128, q=None, qh=0, out=None, dt=0, T=4, kw=None, kn=0,
               cs=None, rows=0, ws=None, nws=0):
        return L.fvsr_kv_append(c or cache(), k, ts, hs, fake, ts, hs, q, 512, 128, qh, out, dt, T,
                                kw, kn, None, 0, 0, 1e-6, cs, rows, None, ws, nws, None)

    def attend(c=None, q=fake, ts=512, hs=128, qh=4, o=fake, ots=512, dt=0, T=4, keep=None, nq=0,
               scale=1.0, ws=None, nws=0):
        return L.fvsr_paged_attn(c or cache(), q, ts, hs, qh, o, ots, 128, dt, T, 1, keep, nq, 3,
                                 scale, 1, ws, nws, None)
    for f in (append, attend):
        assert f(T=0) == _lib.FVSR_OK and f(cache(sequences=0)) == _lib.FVSR_OK
        assert f(T=3) == _lib.FVSR_EINVAL  # two sequences
        for bad in (dict(pages=-1), dict(heads=0), dict(table_stride=2), dict(k=None),
                    dict(lengths=None), dict(table=None), dict(sequences=-1)):
            assert f(cache(**bad)) == _lib.FVSR_EINVAL, bad
        for bad in (dict(head_dim=96), dict(k=fake + 8), dict(pages=1 << 40)):
            assert f(cache(**bad)) == _lib.FVSR_EUNSUPPORTED, bad
        assert f(ts=250) == _lib.FVSR_EUNSUPPORTED
        assert f(dt=7) == _lib.FVSR_EINVAL
    assert append(k=None) == _lib.FVSR_EINVAL
    assert append(kn=1) == _lib.FVSR_EINVAL and append(kn=5) == _lib.FVSR_EINVAL
    assert append(q=fake, qh=4) == _lib.FVSR_EINVAL
    assert append(cs=fake, rows=3) == _lib.FVSR_EINVAL
    assert append(T=4000, kw=fake, kn=2) == _lib.FVSR_EWORKSPACE
    assert L.fvsr_kv_append_workspace_floats(4000, 2) == 8000
    assert L.fvsr_kv_append_workspace_floats(4000, 1) == 0
    assert attend(dt=2) == _lib.FVSR_EINVAL and attend(qh=3) == _lib.FVSR_EINVAL
    assert attend(scale=0.0) == _lib.FVSR_EINVAL and attend(scale=math.nan) == _lib.FVSR_EINVAL
    assert attend(q=None) == _lib.FVSR_EINVAL and attend(o=None) == _lib.FVSR_EINVAL
    assert attend(o=fake + 4) == _lib.FVSR_EUNSUPPORTED
    assert attend(keep=fake, nq=-1) == _lib.FVSR_EINVAL
    wide = cache(table_stride=4000, table_pages=4000)
    assert attend(wide) == _lib.FVSR_EWORKSPACE
    assert L.fvsr_paged_attn_workspace_floats(wide, 4, 4, 0) > 0
    assert L.fvsr_paged_attn_workspace_floats(cache(head_dim=96), 4, 4, 0) == 0


def test_launches_too_large_are_refused():
    """A launch holds 2^32 threads; what needs more is refused before it."""
    from flashvsr_sm89_ops import _lib
    from flashvsr_sm89_ops.paged_kv import _Cache
    L = _lib.lib()
    fake = 1 << 20

    def append(heads, T, B, packed=False, qh=0):
        c = _Cache(fake, fake, fake, fake, 4, heads, 128, fake, 3, 3, fake,
                   fake if packed else None, B)
        return L.fvsr_kv_append(ctypes.byref(c), fake, 128 * heads, 128, fake, 128 * heads, 128,
                                fake if qh else None, 128 * qh, 128, qh, fake if qh else None, 0,
                                T, None, 0, None, 0, 0, 1e-6, None, 0, None, None, 0, None)
    # 2^22 packed tokens x 2 heads: 2^24 workgroups of 512 threads
    assert append(2, 0x3ffff0, 0x3ffff0, packed=True) == _lib.FVSR_EUNSUPPORTED
    assert append(1, 1 << 21, 1 << 21, qh=128) == _lib.FVSR_EUNSUPPORTED  # 2^26 waves of q
    assert append(1, 1 << 28, 1, qh=1) == _lib.FVSR_EUNSUPPORTED


def test_definition_of_e4m3():
    """The oracle's rounding is torch's for every value between codes, and its exponent the
    least that holds a value."""
    from oracle import paged_kv as O
    x = torch.cat([torch.linspace(-448, 448, 100001), torch.randn(10000) * 2.0 ** -6,
                   torch.tensor([0.0, 448.0, 2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10])]).double()
    assert torch.equal(O.e4m3(x), x.float().to(E4).float().double().where(
        x.float().double() == x, O.e4m3(x)))
    xf = x.float().double()
    assert torch.equal(O.e4m3(xf), xf.float().to(E4).float().double())
    for top in (1e-45, 0.3, 1.0, 448.0, 448.0001, 1e30, 3.4e38):
        e = O.exponent(top)
        assert top <= 448 * 2.0 ** e and (e == -126 or top > 448 * 2.0 ** (e - 1))
