"""CPU tests of refusals of the encoder operators' C entry points."""
import ctypes

import pytest

from mamtorch_amd import capi


def _attention(**changes):
    a = capi.DiffAttention(q=256, k=256, v=256, lam=256, B=1, Lq=2, Lk=2, H=2, Hkv=1, D=8, Dv=8, scale=1.0)
    for n, v in changes.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("scale", [1e-46, 1e-300])
def test_a_scale_that_float32_holds_as_zero_is_refused(scale):
    # masked scores of -inf times a scale of 0 would be NaN
    l, one = capi.lib(), ctypes.c_void_p(256)
    a, strides = _attention(scale=scale), (ctypes.c_int64 * 3)(16, 8, 8)
    assert l.mam_diff_attention(a, None, None, None, None, 0, None) == -1
    assert b"scale" in l.mam_last_error()
    assert l.mam_diff_attention_backward(a, one, strides, one, one, one, one, one, one, one, None, 0, None) == -1
    assert b"scale" in l.mam_last_error()
