"""Rests of some tensors' 8-bit moments only are refused (before the device is touched)."""
import ctypes

import pytest

from mymedialite_amd import _native as N


def test_some_rests_are_refused():
    one = dict(param=256, grad=256, m=256, v=256, m_scale=256, v_scale=256, n=5)
    t = (N.AdamwTensor * 3)(N.AdamwTensor(**one), N.AdamwTensor(n=0), N.AdamwTensor(rest=256, **one))
    p = N.AdamwParams(learn_rate=1e-3, beta1=0.9, beta2=0.999, epsilon=1e-8, weight_decay=0.0,
                      state_bits=8)
    with pytest.raises(N.MMLError, match="rests of some") as e:
        N.check(N.lib().mml_adamw_step_device(t, 3, ctypes.byref(p), 256, 0, None))
    assert e.value.status == -1
