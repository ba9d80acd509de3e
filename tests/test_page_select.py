"""pool_pages, select_pages and selected_attention on the CPU: what they refuse, in Python and at
the C ABI, and that their definitions see what is wrong; nothing here launches a kernel."""
import ctypes
import math
from fractions import Fraction

import pytest
import torch

BF, E4, E8, I32 = torch.bfloat16, torch.float8_e4m3fn, torch.float8_e8m0fnu, torch.int32
z = torch.zeros
FAKE = 1 << 20


def cpu_pages(N=4, H=2, D=64):
    from flashvsr_sm89_ops import kv_pages
    return kv_pages(N, H, D, device="cpu")


def steps(**kw):
    return dict(page_table=z(2, 3, dtype=I32), lengths=z(2, dtype=I32), **kw)


def pool_args(**kw):
    from flashvsr_sm89_ops import page_means
    return {**steps(means=page_means(cpu_pages()), pages=cpu_pages(), tokens=6), **kw}


def select_args(**kw):
    from flashvsr_sm89_ops import page_means
    return {**steps(q=z(6, 4, 64, dtype=BF), means=page_means(cpu_pages()), top=3), **kw}


def attend_args(**kw):
    return {**steps(q=z(6, 4, 64, dtype=BF), pages=cpu_pages(), columns=z(6, 2, 5, dtype=I32)), **kw}


def test_means():
    from flashvsr_sm89_ops import page_means
    m = page_means(cpu_pages(3, 2, 128))
    assert m.mean.shape == (3, 2, 128) and m.mean.dtype == torch.int8
    assert m.scale.shape == (3, 2) and m.scale.dtype == E8


def test_calls_need_a_gpu():
    from flashvsr_sm89_ops import pool_pages, select_pages, selected_attention
    for f, a in ((pool_pages, pool_args), (select_pages, select_args),
                 (selected_attention, attend_args)):
        with pytest.raises(RuntimeError, match="GPU only"):
            f(**a())


SHARED = [
    (dict(page_table=z(2, 3, dtype=torch.int64)), TypeError),
    (dict(lengths=z(2, dtype=torch.int64)), TypeError),
    (dict(lengths=z(3, dtype=I32)), ValueError),
    (dict(lengths=z(4, dtype=I32)[::2]), ValueError),
    (dict(page_table=z(3, 2, dtype=I32).t()), ValueError),
    (dict(page_table=z(3, dtype=I32)), ValueError),
    (dict(page_table=z(1, 3, dtype=I32).expand(2, 3)), ValueError),
    (dict(page_table=z(4, 3, dtype=I32), lengths=z(4, dtype=I32)), ValueError),  # 6 rows over 4
    (dict(page_table=z(0, 3, dtype=I32), lengths=z(0, dtype=I32)), ValueError),  # 6 rows over none
    (dict(cu_tokens=z(2, dtype=I32)), ValueError),
    (dict(cu_tokens=z(3)), TypeError),
]


@pytest.mark.parametrize("change,error", SHARED)
def test_all_refuse(change, error):
    from flashvsr_sm89_ops import pool_pages, select_pages, selected_attention
    for f, a in ((pool_pages, pool_args), (select_pages, select_args),
                 (selected_attention, attend_args)):
        with pytest.raises(error):
            f(**a(**change))


def means_of(mean=None, scale=None):
    from flashvsr_sm89_ops import PageMeans
    return PageMeans(z(4, 2, 64, dtype=torch.int8) if mean is None else mean,
                     z(4, 2, dtype=torch.uint8).view(E8) if scale is None else scale)


@pytest.mark.parametrize("means,error", [
    (dict(mean=z(4, 2, 64)), TypeError),
    (dict(mean=z(4, 2, 64, dtype=torch.uint8)), TypeError),
    (dict(scale=z(4, 2)), TypeError),
    (dict(scale=z(4, 1, dtype=torch.uint8).view(E8)), ValueError),
    (dict(mean=z(4, 2, 96, dtype=torch.int8)), ValueError),
    (dict(mean=z(4, 128, dtype=torch.int8)), ValueError),
    (dict(mean=z(2, 4, 64, dtype=torch.int8).transpose(0, 1)), ValueError),
    (dict(mean=z(521, dtype=torch.int8)[9:].view(4, 2, 64)), ValueError),  # not aligned
])
def test_means_refused(means, error):
    from flashvsr_sm89_ops import pool_pages, select_pages
    for f, a in ((pool_pages, pool_args), (select_pages, select_args)):
        with pytest.raises(error):
            f(**a(means=means_of(**means)))


@pytest.mark.parametrize("change,error", [
    (dict(tokens=-1), ValueError),
    (dict(tokens=5), ValueError),
    (dict(pages="other"), ValueError),
    (dict(means="other"), ValueError),
])
def test_pool_refuses(change, error):
    from flashvsr_sm89_ops import page_means, pool_pages
    if "pages" in change:
        change = dict(pages=cpu_pages(4, 2, 128))
    if "means" in change:
        change = dict(means=page_means(cpu_pages(5, 2, 64)))
    with pytest.raises(error):
        pool_pages(**pool_args(**change))


@pytest.mark.parametrize("change,error", [
    (dict(q=z(6, 3, 64, dtype=BF)), ValueError),
    (dict(q=z(6, 4, 128, dtype=BF)), ValueError),
    (dict(q=z(6, 256, dtype=BF)), ValueError),
    (dict(q=z(6, 4, 64)), TypeError),
    (dict(q=z(6, 4, 64, dtype=torch.float64)), TypeError),
    (dict(q=z(6, 0, 64, dtype=BF)), ValueError),
    (dict(top=1), ValueError),            # first and recent are 1 each
    (dict(top=0, first=0, recent=0), ValueError),
    (dict(recent=0), ValueError),
    (dict(first=-1), ValueError),
    (dict(first=3), ValueError),
    (dict(top=1 << 24), ValueError),      # refused before the list is allocated
    (dict(page_table=z(2, 32769, dtype=I32)), ValueError),
])
def test_select_refuses(change, error):
    from flashvsr_sm89_ops import select_pages
    with pytest.raises(error):
        select_pages(**select_args(**change))


@pytest.mark.parametrize("change,error", [
    (dict(q=z(6, 3, 64, dtype=BF)), ValueError),
    (dict(q=z(6, 4, 32, dtype=BF)), ValueError),
    (dict(q=z(6, 4, 64)), TypeError),
    (dict(columns=z(6, 2, 5)), TypeError),
    (dict(columns=z(6, 2, 5, dtype=torch.int64)), TypeError),
    (dict(columns=z(6, 4, 5, dtype=I32)), ValueError),
    (dict(columns=z(5, 2, 5, dtype=I32)), ValueError),
    (dict(columns=z(6, 2, dtype=I32)), ValueError),
    (dict(columns=z(6, 2, 10, dtype=I32)[..., ::2]), ValueError),
    (dict(sm_scale=0.0), ValueError),
    (dict(sm_scale=math.nan), ValueError),
    (dict(sm_scale=math.inf), ValueError),
    (dict(out=z(6, 4, 64)), TypeError),
    (dict(out=z(6, 4, 32, dtype=BF)), ValueError),
    (dict(out=z(6, 4, 66, dtype=BF)[..., :64]), ValueError),
    (dict(out=z(1, 4, 64, dtype=BF).expand(6, 4, 64)), ValueError),
    (dict(pages="k"), TypeError),
])
def test_attention_refuses(change, error):
    from flashvsr_sm89_ops import KVPages, selected_attention
    if "pages" in change:
        k, v, ks, vs = cpu_pages()
        change = dict(pages=KVPages(k.float(), v, ks, vs))
    with pytest.raises(error):
        selected_attention(**attend_args(**change))


def cache(**kw):
    from flashvsr_sm89_ops.paged_kv import _Cache
    f = dict(k=FAKE, v=FAKE, k_scale=FAKE, v_scale=FAKE, pages=4, heads=2, head_dim=128, table=FAKE,
             table_stride=3, table_pages=3, lengths=FAKE, cu=None, sequences=2)
    f.update(kw)
    return ctypes.byref(_Cache(**f))


def c_pool(c=None, mean=FAKE, scale=FAKE, T=4):
    from flashvsr_sm89_ops import _lib
    return _lib.lib().fvsr_pool_pages(c or cache(), mean, scale, T, None)


def c_select(c=None, mean=FAKE, scale=FAKE, q=FAKE, ts=512, hs=128, qh=4, dt=0, T=4, top=3, first=1,
             recent=1, out=FAKE):
    from flashvsr_sm89_ops import _lib
    return _lib.lib().fvsr_select_pages(c or cache(), mean, scale, q, ts, hs, qh, dt, T, top, first,
                                        recent, out, None)


def c_attend(c=None, q=FAKE, ts=512, hs=128, qh=4, o=FAKE, ots=512, dt=0, T=4, cols=FAKE, top=3,
             scale=1.0, ws=None, nws=0):
    from flashvsr_sm89_ops import _lib
    return _lib.lib().fvsr_selected_attn(c or cache(), q, ts, hs, qh, o, ots, 128, dt, T, cols, top,
                                         scale, 1, ws, nws, None)


def test_c_entries_check_arguments():
    """Statuses before any launch: device pointers are never followed."""
    from flashvsr_sm89_ops import _lib
    L = _lib.lib()
    for f in (c_pool, c_select, c_attend):
        assert f(T=0) == _lib.FVSR_OK and f(cache(sequences=0)) == _lib.FVSR_OK
        assert f(T=3) == _lib.FVSR_EINVAL  # two sequences
        for bad in (dict(pages=-1), dict(heads=0), dict(table_stride=2), dict(lengths=None),
                    dict(table=None), dict(sequences=-1)):
            assert f(cache(**bad)) == _lib.FVSR_EINVAL, bad
        for bad in (dict(head_dim=96), dict(pages=1 << 40)):
            assert f(cache(**bad)) == _lib.FVSR_EUNSUPPORTED, bad
    for f in (c_pool, c_attend):
        assert f(cache(k=None)) == _lib.FVSR_EINVAL
        assert f(cache(k=FAKE + 8)) == _lib.FVSR_EUNSUPPORTED
    for f in (c_pool, c_select):
        assert f(mean=None) == _lib.FVSR_EINVAL and f(scale=None) == _lib.FVSR_EINVAL
        assert f(mean=FAKE + 8) == _lib.FVSR_EUNSUPPORTED
    for f in (c_select, c_attend):
        assert f(ts=250) == _lib.FVSR_EUNSUPPORTED and f(q=FAKE + 8) == _lib.FVSR_EUNSUPPORTED
        assert f(dt=2) == _lib.FVSR_EINVAL and f(qh=3) == _lib.FVSR_EINVAL
        assert f(q=None) == _lib.FVSR_EINVAL
    assert c_pool(T=-2) == _lib.FVSR_EINVAL
    assert c_pool(cache(lengths=None), T=-1) == _lib.FVSR_EINVAL
    assert c_select(out=None) == _lib.FVSR_EINVAL
    for bad in (dict(top=1), dict(recent=0), dict(first=-1)):
        assert c_select(**bad) == _lib.FVSR_EINVAL, bad
    assert c_select(cache(table_stride=40000, table_pages=40000)) == _lib.FVSR_EUNSUPPORTED
    assert c_select(top=1 << 30) == _lib.FVSR_EUNSUPPORTED
    assert c_attend(o=None) == _lib.FVSR_EINVAL and c_attend(cols=None) == _lib.FVSR_EINVAL
    assert c_attend(top=-1) == _lib.FVSR_EINVAL and c_attend(scale=0.0) == _lib.FVSR_EINVAL
    assert c_attend(scale=math.nan) == _lib.FVSR_EINVAL
    assert c_attend(o=FAKE + 4) == _lib.FVSR_EUNSUPPORTED
    assert c_attend(top=400) == _lib.FVSR_EWORKSPACE
    assert L.fvsr_selected_attn_workspace_floats(cache(), 4, 4, 400) > 0
    assert L.fvsr_selected_attn_workspace_floats(cache(head_dim=96), 4, 4, 400) == 0


@pytest.mark.parametrize("T", [1, 1 << 24, (1 << 30) - 1])
@pytest.mark.parametrize("heads", [1 << 40, 1 << 62, (1 << 63) - 1])
def test_heads_past_any_launch_are_refused(heads, T):
    from flashvsr_sm89_ops import _lib
    one = dict(sequences=1)
    for c, qh in ((cache(**one, heads=1), heads), (cache(**one, heads=heads), heads)):
        assert c_select(c, qh=qh, T=T) == _lib.FVSR_EUNSUPPORTED
        assert c_attend(c, qh=qh, T=T) == _lib.FVSR_EUNSUPPORTED
        assert _lib.lib().fvsr_selected_attn_workspace_floats(c, T, qh, 400) == 0
    assert c_pool(cache(**one, heads=heads), T=T) == _lib.FVSR_EUNSUPPORTED


def test_launches_too_large_are_refused():
    from flashvsr_sm89_ops import _lib
    many = 1 << 22
    for c, T in ((cache(sequences=many - 1, table_pages=1 << 23, table_stride=1 << 23), -1),
                 (cache(sequences=many - 1, heads=1 << 10), (many - 1) * 8)):
        assert c_pool(c, T=T) == _lib.FVSR_EUNSUPPORTED
    assert c_select(cache(sequences=1, heads=64), qh=64, T=(1 << 24) - 1) == _lib.FVSR_EUNSUPPORTED
    assert c_attend(cache(sequences=1, heads=1), qh=128, T=(1 << 24) - 1) == _lib.FVSR_EUNSUPPORTED


def test_definition_of_means():
    """Against fractions made another way: the exponent is the least, codes are nearest."""
    from oracle import page_select as S
    g = torch.Generator().manual_seed(0)
    for seed in range(20):
        codes = (64 * torch.randn(128, 4, generator=g) * 2.0 ** (seed - 12)).clamp(-448, 448).to(E4)
        m, byte = S.mean_of(codes.double(), 100 + seed)
        mean = [sum(Fraction(float(x)) for x in col) / 128 * Fraction(2) ** (seed - 27)
                for col in codes.double().T]
        unit = Fraction(2) ** (byte - 127)
        assert all(abs(Fraction(a) - x / unit) <= Fraction(1, 2) for a, x in zip(m, mean))
        top = max(map(abs, mean))
        assert top <= 127 * unit and (top == 0 or top > 127 * unit / 2)
    assert S.mean_of(z(128, 3).double(), 120) == ([0, 0, 0], 0)
    assert S.mean_of(torch.full((128, 3), math.nan).double(), 120) == ([0, 0, 0], 255)


def test_definition_of_the_choice():
    """A score that is highest by one step is found, ties go to the lower column."""
    from oracle import page_select as S
    P = 12
    table, mean = torch.arange(P)[None].int(), z(P, 1, 64, dtype=torch.int8)
    scale = torch.full((P, 1), 120, dtype=torch.uint8)
    q = z(1, 2, 64).double()
    q[0, 0, 0], q[0, 1, 1] = 1.0, 1.0
    assert S.selected(q, mean, scale, table, [P * 128], 4, 1, 1)[0, 0].tolist() == [0, 1, 2, 11]
    mean[7, 0, 1] = 1
    assert S.selected(q, mean, scale, table, [P * 128], 4, 1, 1)[0, 0].tolist() == [0, 1, 7, 11]
    mean[9, 0, 0] = 3
    scale[9] = 119
    assert S.selected(q, mean, scale, table, [P * 128], 3, 1, 1)[0, 0].tolist() == [0, 9, 11]
    assert S.selected(q, mean, scale, table, [P * 128 - 128], 3, 1, 1)[0, 0].tolist() == [0, 9, 10]
    scale[9] = 255
    assert S.selected(q, mean, scale, table, [P * 128], 3, 1, 1)[0, 0].tolist() == [0, 7, 11]
    assert S.selected(q, mean, scale, table, [0], 3, 1, 1)[0, 0].tolist() == [-1, -1, -1]
    assert S.selected(q, mean, scale, table, [129], 3, 1, 1)[0, 0].tolist() == [0, 1, -1]


def test_pool_does_not_ask_for_v():
    """v and its scales are not read, so they may be missing: with or without a number of rows the
    first refusal is that of the launch's size."""
    from flashvsr_sm89_ops import _lib
    many = (1 << 22) - 1
    for bad in (dict(v=None, v_scale=None), dict(v=FAKE + 8)):
        c = cache(sequences=many, heads=8, **bad)
        assert c_pool(c, T=many) == _lib.FVSR_EUNSUPPORTED
        assert c_pool(c, T=-1) == _lib.FVSR_EUNSUPPORTED
        c = cache(sequences=many, heads=8, k=None, **bad)
        assert c_pool(c, T=many) == _lib.FVSR_EINVAL and c_pool(c, T=-1) == _lib.FVSR_EINVAL
        c = cache(sequences=many, heads=8, k_scale=None, **bad)
        assert c_pool(c, T=many) == _lib.FVSR_EINVAL and c_pool(c, T=-1) == _lib.FVSR_EINVAL
