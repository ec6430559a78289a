"""AdamW's argument checks that need no GPU (every one comes before the device is touched)."""
import ctypes

import pytest
import torch

from mymedialite_amd import AdamW
from mymedialite_amd import _native as N


def call(tensors=None, n=0, params=None, state=256):
    t = (N.AdamwTensor * max(n, 1))(*(tensors or []))
    p = dict(learn_rate=1e-3, beta1=0.9, beta2=0.999, epsilon=1e-8, weight_decay=0.0, state_bits=32)
    p.update(params or {})
    N.check(N.lib().mml_adamw_step_device(t if tensors is not None else None, n,
                                          ctypes.byref(N.AdamwParams(**p)), state, 0, None))


def tensor(**kw):
    a = dict(param=256, grad=256, m=256, v=256, n=5)
    a.update(kw)
    return N.AdamwTensor(**a)


@pytest.mark.parametrize("kw,text", [
    (dict(state=None), "step_state"), (dict(n=-1), "tensors"), (dict(n=1), "tensors"),
    (dict(params=dict(state_bits=16)), "state_bits"), (dict(params=dict(beta1=1.0)), "beta"),
    (dict(params=dict(beta2=-0.5)), "beta"), (dict(params=dict(learn_rate=-1.0)), "learn_rate"),
    (dict(params=dict(learn_rate=float("nan"))), "learn_rate"),
    (dict(params=dict(epsilon=float("inf"))), "epsilon"),
    (dict(params=dict(weight_decay=-1.0)), "weight_decay"),
    (dict(n=1, tensors=[tensor(n=-1)]), "size"), (dict(n=1, tensors=[tensor(param=None)]), "null"),
    (dict(n=1, tensors=[tensor(grad=None)]), "null"), (dict(n=1, tensors=[tensor(v=None)]), "null"),
    (dict(n=1, tensors=[tensor(param_dtype=3)]), "dtype"),
    (dict(n=1, tensors=[tensor(grad_dtype=-1)]), "dtype"),
    (dict(n=1, tensors=[tensor()], params=dict(state_bits=8)), "scales")])
def test_refusals(kw, text):
    with pytest.raises(N.MMLError, match=text) as e:
        call(**kw)
    assert e.value.status == -1


def test_cpu_parameters_are_refused():
    with pytest.raises(ValueError, match="on the GPU"):
        AdamW([torch.zeros(3)])
    with pytest.raises(ValueError, match="StateBits"):
        AdamW([], StateBits=4)
