"""The refusal of 8-bit moments without their rests (before the device is touched)."""
import ctypes

import pytest

from mymedialite_amd import _native as N


def test_missing_rests_are_refused():
    t = (N.AdamwTensor * 1)(N.AdamwTensor(param=256, grad=256, m=256, v=256, m_scale=256, v_scale=256,
                                          n=5))
    p = N.AdamwParams(learn_rate=1e-3, beta1=0.9, beta2=0.999, epsilon=1e-8, weight_decay=0.0,
                      state_bits=8)
    with pytest.raises(N.MMLError, match="rests") as e:
        N.check(N.lib().mml_adamw_step_device(t, 1, ctypes.byref(p), 256, 0, None))
    assert e.value.status == -1
