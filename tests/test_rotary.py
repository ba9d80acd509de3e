"""rotary and rotary_frequencies on the CPU: the frequencies' formulas, what both refuse, in Python
and at the C ABI; nothing here launches a kernel."""
import ctypes
import math

import pytest
import torch

BF, I32 = torch.bfloat16, torch.int32
z = torch.zeros
FAKE = 1 << 20


def inverse(f):
    return f.turns * (2 * math.pi)


def test_frequencies():
    from flashvsr_sm89_ops import rotary_frequencies

    def freqs(*a, **k):
        return rotary_frequencies(*a, device="cpu", **k)
    f = freqs(8, 100.0)
    assert f.turns.dtype == torch.float64 and f.gain == 1.0
    plain = torch.tensor([1.0, 100.0 ** -0.25, 0.1, 100.0 ** -0.75]).double()
    assert torch.allclose(inverse(f), plain, rtol=1e-6)
    # (rtol of float32 literals; the ratios below are of doubles)
    g = freqs(8, 100.0, scaling="linear", factor=4.0)
    assert torch.equal(g.turns, f.turns / 4) and g.gain == 1.0
    g = freqs(8, 100.0, scaling="base", factor=4.0)
    assert torch.allclose(g.turns[0], f.turns[0], rtol=1e-15)
    assert torch.allclose(g.turns[3], f.turns[3] / 4, rtol=1e-14)
    # 1000 tokens: 159, 50, 16 and 5 turns; whole down to 100, divided from 10 on
    g = freqs(8, 100.0, scaling="parts", factor=4.0, context=1000, fast=100.0, slow=10.0)
    ratio = g.turns / f.turns
    r = 1000 * f.turns
    keep = float((r[1] - 10) / 90)
    assert float(ratio[0]) == 1.0 and abs(float(ratio[3]) - 0.25) < 1e-15
    assert abs(float(ratio[1]) - (keep + (1 - keep) / 4)) < 1e-14
    assert 0.25 < float(ratio[2]) < float(ratio[1]) < 1.0
    assert g.gain == 0.1 * math.log(4.0) + 1.0
    assert freqs(8, scaling="parts", factor=4.0, context=1000, gain=1.0).gain == 1.0
    assert torch.equal(freqs(8, scaling="linear").turns, freqs(8).turns)
    assert freqs(2).turns.tolist() == [1 / (2 * math.pi)]


@pytest.mark.parametrize("a,k", [
    ((7,), {}), ((0,), {}), ((-2,), {}), ((8, 0.0), {}), ((8, -1.0), {}), ((8, math.inf), {}),
    ((8, math.nan), {}), ((8,), dict(factor=2.0)), ((8,), dict(scaling="ntk")),
    ((8,), dict(scaling="linear", factor=0.5)), ((8,), dict(scaling="linear", factor=math.nan)),
    ((2,), dict(scaling="base", factor=2.0)), ((8,), dict(scaling="parts", factor=2.0)),
    ((8,), dict(scaling="parts", factor=2.0, context=0)),
    ((8,), dict(scaling="parts", factor=2.0, context=100, fast=1.0, slow=1.0)),
    ((8,), dict(scaling="parts", factor=2.0, context=100, slow=-1.0)),
    ((8,), dict(gain=math.nan)), ((8,), dict(gain=math.inf)),
])
def test_frequencies_refuse(a, k):
    from flashvsr_sm89_ops import rotary_frequencies
    with pytest.raises(ValueError):
        rotary_frequencies(*a, device="cpu", **k)


def args(**kw):
    from flashvsr_sm89_ops import rotary_frequencies
    return {**dict(q=z(6, 4, 64, dtype=BF), k=z(6, 2, 64, dtype=BF),
                   freqs=rotary_frequencies(64, device="cpu")), **kw}


def test_needs_a_gpu():
    from flashvsr_sm89_ops import rotary
    with pytest.raises(RuntimeError, match="GPU only"):
        rotary(**args())
    with pytest.raises(RuntimeError, match="GPU only"):
        rotary(**args(k=None, positions=z(6, dtype=I32)))


@pytest.mark.parametrize("change,error", [
    (dict(q=z(6, 64, dtype=BF)), ValueError),
    (dict(q=z(1, 1, 6, 4, 64, dtype=BF)), ValueError),
    (dict(k=z(5, 2, 64, dtype=BF)), ValueError),
    (dict(k=z(6, 2, 32, dtype=BF)), ValueError),
    (dict(k=z(1, 6, 2, 64, dtype=BF)), ValueError),
    (dict(k=z(6, 2, 64)), TypeError),
    (dict(q=z(6, 4, 64, dtype=torch.float64), k=None), TypeError),
    (dict(q=z(6, 4, 64, dtype=torch.int32), k=None), TypeError),
    (dict(q=z(6, 4, 32, dtype=BF), k=None), ValueError),          # 64 channels of 32
    (dict(pairs="other"), ValueError),
    (dict(positions=z(6)), TypeError),
    (dict(positions=z(6, dtype=torch.int64)), TypeError),
    (dict(positions=z(5, dtype=I32)), ValueError),
    (dict(positions=z(6, 1, dtype=I32)), ValueError),
    (dict(positions=z(12, dtype=I32)[::2]), ValueError),
    (dict(freqs="fp32"), TypeError),
    (dict(freqs="two"), ValueError),
    (dict(freqs="strided"), ValueError),
    (dict(freqs="grad"), ValueError),
])
def test_refuses(change, error):
    from flashvsr_sm89_ops import RotaryFrequencies, rotary
    turns = {"fp32": z(32), "two": z(2, 16).double(), "strided": z(64).double()[::2],
             "grad": z(32).double().requires_grad_()}
    if "freqs" in change:
        change = dict(freqs=RotaryFrequencies(turns[change["freqs"]]))
    with pytest.raises(error):
        rotary(**args(**change))


def test_positions_for_batches():
    from flashvsr_sm89_ops import rotary
    x = z(2, 6, 4, 64, dtype=BF)
    for p in (z(6, dtype=I32), z(2, 6, dtype=I32), z(1, 6, dtype=I32).expand(2, 6)):
        with pytest.raises(RuntimeError, match="GPU only"):
            rotary(**args(q=x, k=None, positions=p))
    for p in (z(2, dtype=I32), z(6, 2, dtype=I32), z(1, 6, dtype=I32), z(6, 2, dtype=I32).t()):
        with pytest.raises(ValueError):
            rotary(**args(q=x, k=None, positions=p))


def test_c_entry_checks_arguments():
    from flashvsr_sm89_ops import _lib
    from flashvsr_sm89_ops.rotary import _Rows
    L = _lib.lib()

    def rows(x=FAKE, y=FAKE, heads=2, b=1024, t=128, h=64):
        return ctypes.byref(_Rows(x, y, heads, b, t, h))

    def call(q=None, k=None, dt=0, B=1, S=8, D=64, R=64, turns=FAKE, pos=None, pairs=0):
        return L.fvsr_rotary(q or rows(), k, dt, B, S, D, R, turns, pos, 0, 1.0, pairs, 0, None)
    assert call(B=0) == _lib.FVSR_OK and call(S=0) == _lib.FVSR_OK
    assert call(rows(heads=0)) == _lib.FVSR_OK
    for bad in (dict(B=-1), dict(S=-1), dict(D=0), dict(R=66), dict(R=-2), dict(R=3), dict(dt=3),
                dict(pairs=2), dict(turns=None), dict(q=rows(x=None)), dict(k=rows(y=None)),
                dict(q=rows(heads=-1)), dict(turns=FAKE + 4)):
        assert call(**bad) == _lib.FVSR_EINVAL, bad
    for bad in (dict(q=rows(x=FAKE + 1)), dict(D=1 << 21), dict(S=1 << 40), dict(B=1 << 40),
                dict(B=1 << 30, S=1 << 30), dict(S=(1 << 31) - 1, q=rows(heads=1 << 20))):
        assert call(**bad) == _lib.FVSR_EUNSUPPORTED, bad
    assert L.fvsr_rotary(None, None, 0, 1, 8, 64, 64, FAKE, None, 0, 1.0, 0, 0, None) == _lib.FVSR_EINVAL


def test_definition():
    """The definition against complex numbers, both layouts, and back."""
    from oracle import page_select as S
    g = torch.Generator().manual_seed(0)
    x = torch.randn(2, 5, 3, 10, generator=g).double()
    turns, pos = torch.rand(4, generator=g).double(), torch.tensor([3, 0, -7, 100, 5])
    ang = 2 * math.pi * (pos[:, None].double() * turns)
    w = torch.polar(torch.full_like(ang, 1.5), ang)[:, None]
    y = torch.view_as_real(torch.view_as_complex(x[..., :8].reshape(2, 5, 3, 4, 2)) * w).flatten(-2)
    got = S.rotated(x, turns, 1.5, pos, "interleaved")
    assert torch.allclose(got[..., :8], y, atol=1e-10) and torch.equal(got[..., 8:], x[..., 8:])
    mix = torch.cat([x[..., 0:8:2], x[..., 1:8:2], x[..., 8:]], -1)
    half = S.rotated(mix, turns, 1.5, pos, "half")
    assert torch.allclose(half[..., :4], y[..., 0::2], atol=1e-10)
    assert torch.allclose(half[..., 4:8], y[..., 1::2], atol=1e-10)
    there = S.rotated(got, turns, 1 / 1.5 ** 2 * 1.5, pos, "interleaved", back=True)
    assert torch.allclose(there, x, atol=1e-10)
