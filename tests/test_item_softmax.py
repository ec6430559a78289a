"""The catalogue softmax's argument checks that need no GPU."""
import ctypes

import pytest
import torch

from mymedialite_amd import _native as N
from mymedialite_amd import item_log_probs


def args(**kw):
    a = dict(dtype=N.DTYPE_F32, num_factors=8, n_rows=4, n_users=4, n_items=50, ld_users=8,
             ld_items=8)
    a.update(kw)
    return N.ItemSoftmaxArgs(**a)


def workspace(a, grad=0):
    n = ctypes.c_int64(0)
    N.check(N.lib().mml_item_log_probs_workspace(ctypes.byref(a) if a else None, grad,
                                                 ctypes.byref(n)))
    return n.value


@pytest.mark.parametrize("bad,text", [
    (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"), (dict(num_factors=0), "num_factors"),
    (dict(num_factors=257, ld_users=257, ld_items=257), "num_factors"), (dict(n_rows=-1), "n_rows"),
    (dict(n_rows=5), "more rows"), (dict(n_items=0), "n_items"), (dict(n_users=0, users=256), "n_users"), (dict(ld_users=7), "stride"),
    (dict(ld_items=7), "stride"), (dict(n_top=129), "n_top"), (dict(n_top=-1), "n_top"),
    (dict(n_exclude=-1), "n_exclude")])
def test_bad_sizes(bad, text):
    for grad in (0, 1):
        with pytest.raises(N.MMLError, match=text) as e:
            workspace(args(**bad), grad)
        assert e.value.status == -1


def test_workspace_sizes():
    with pytest.raises(N.MMLError, match="args is null"):
        workspace(None)
    for grad in (0, 1):
        assert workspace(args(n_rows=0), grad) > 0  # no rows are a call too
        for rows in (1, 31, 32, 33, 5000):
            for items in (1, 255, 257, 70_000):
                for k in (1, 16, 17, 64, 256):
                    assert workspace(args(n_rows=rows, n_users=rows, n_items=items, num_factors=k,
                                          ld_users=k, ld_items=k, n_top=5 * (1 - grad)), grad) > 0
    small, large = workspace(args()), workspace(args(n_rows=4, n_items=500))
    assert 0 < small < large
    assert workspace(args(n_top=5)) > small
    assert workspace(args(), 1) > small
    # sizes beyond 32 bits
    big = workspace(args(n_rows=1 << 20, n_users=1 << 20, n_items=1 << 22, n_top=10), 0)
    assert big > 1 << 36


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError, match="on the GPU"):
        item_log_probs(torch.zeros(2, 4), torch.zeros(3, 4))
