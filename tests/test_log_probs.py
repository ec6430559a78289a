"""BPRMF.log_probs, WRMF.log_probs and BPRMF.apply_softmax: the refusals that need no GPU."""
import numpy as np
import pytest

import mymedialite_amd as mml
from mymedialite_amd import _native as N


@pytest.mark.parametrize("cls", [mml.BPRMF, mml.WRMF])
def test_no_model(cls):
    with pytest.raises(RuntimeError, match="not initialised"):
        cls().log_probs([0])


def test_apply_softmax_no_model():
    with pytest.raises(RuntimeError, match="not initialised"):
        mml.BPRMF().apply_softmax([0], [0])


@pytest.mark.parametrize("symbol", ["mml_bpr_log_probs", "mml_wrmf_log_probs"])
def test_null_handle(symbol):
    u = np.zeros(1, np.int32)
    with pytest.raises(N.MMLError, match="null handle") as e:
        N.check(getattr(N.lib(), symbol)(None, N.ptr(u, N._i32p), None, 1, 0, 0, None, None, None,
                                         None, None))
    assert e.value.status == -1


def test_result_type_is_one():
    from mymedialite_amd.item_softmax import ItemLogProbs
    assert mml.ItemLogProbs is ItemLogProbs is N.ItemLogProbs
