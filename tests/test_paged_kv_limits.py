"""The paged cache's C entries at sizes beyond any memory; nothing here launches a kernel."""
import ctypes

import pytest

FAKE = 1 << 20


def cache(heads=1, sequences=1, columns=3):
    from flashvsr_sm89_ops.paged_kv import _Cache
    return ctypes.byref(_Cache(FAKE, FAKE, FAKE, FAKE, 4, heads, 128, FAKE, columns, columns, FAKE,
                               None, sequences))


def append(c, T, q_heads=0):
    from flashvsr_sm89_ops import _lib
    q = FAKE if q_heads else None
    return _lib.lib().fvsr_kv_append(c, FAKE, 128, 128, FAKE, 128, 128, q, 128, 128, q_heads, q, 0,
                                     T, None, 0, None, 0, 0, 1e-6, None, 0, None, None, 0, None)


def attend(c, T, q_heads):
    from flashvsr_sm89_ops import _lib
    return _lib.lib().fvsr_paged_attn(c, FAKE, 128, 128, q_heads, FAKE, 128, 128, 0, T, 1, None, 0,
                                      0, 1.0, 1, None, 0, None)


def floats(c, T, q_heads):
    from flashvsr_sm89_ops import _lib
    return _lib.lib().fvsr_paged_attn_workspace_floats(c, T, q_heads, 0)


@pytest.mark.parametrize("T", [1, 1 << 24, (1 << 30) - 1])
@pytest.mark.parametrize("heads", [1 << 40, 1 << 62, (1 << 63) - 1])
def test_heads_past_any_launch_are_refused(heads, T):
    """Their products with T pass 64 bits: a status, not a plan from what is left of them (which
    divided by zero)."""
    from flashvsr_sm89_ops import _lib
    for c, q_heads in ((cache(), heads), (cache(heads=heads), heads)):
        assert append(c, T, q_heads) == _lib.FVSR_EUNSUPPORTED
        assert attend(c, T, q_heads) == _lib.FVSR_EUNSUPPORTED
        assert floats(c, T, q_heads) == 0


def test_units_past_a_joining_launch_are_not_cut():
    """Pieces of a unit are added by a workgroup for each of its rows, up to 128: what a launch
    does not hold goes uncut, without a workspace, and fewer units are still cut."""
    for B in (200000, 1 << 21):
        assert floats(cache(sequences=B, columns=100000), B * 40, 1) == 0
    assert floats(cache(sequences=20, columns=100000), 20 * 40, 1) > 0


def test_workspace_of_rows_past_any_call():
    from flashvsr_sm89_ops import _lib
    f = _lib.lib().fvsr_kv_append_workspace_floats
    assert f((1 << 30) - 1, _lib.NORM_ROW) == (1 << 31) - 2
    for T in (1 << 30, 1 << 62, (1 << 63) - 1, -1):
        assert f(T, _lib.NORM_ROW) == 0
