"""The models' set and get calls return every factor bit for bit: widths with and without padding on the
device, more rows than go through the packed buffer at a time (16 M floats)."""
import ctypes

import numpy as np
import pytest

from mymedialite_amd import _native as N

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("model", ["bmf", "bpr"])
@pytest.mark.parametrize("k,n_users,n_items", [(1, 7, 5), (3, 70, 50), (10, 943, 1682), (64, 300, 200),
                                               (100, 170_001, 9), (128, 1000, 2), (130, 33, 129_100),
                                               (256, 31, 32)])
def test_model_round_trip(model, k, n_users, n_items):
    rs = np.random.default_rng(k)
    U, V = (rs.normal(0, 1, (n, k)).astype(np.float32) for n in (n_users, n_items))
    bu, bi = (rs.normal(0, 1, n).astype(np.float32) for n in (n_users, n_items))
    L, h, f = N.lib(), N._vp(), lambda x: N.ptr(x, N._f32p)
    ctx = N.Context(0)
    try:
        got = [np.full_like(x, 7.0) for x in (U, V, bu, bi)]
        if model == "bmf":
            p = N.BmfParams(k, N.LOSS_RMSE, 0, N.SCHEDULE_HOGWILD, 1.0, 0.01, 0.015, 0.015)
            N.check(L.mml_bmf_create(ctx.handle, ctypes.byref(p), n_users, n_items, ctypes.byref(h)))
            N.check(L.mml_bmf_set_model(h, f(U), f(V), f(bu), f(bi), 0.1, 1.0, 5.0))
            N.check(L.mml_bmf_get_model(h, *map(f, got)))
            want = (U, V, bu, bi)
        else:
            p = N.BprParams(k, N.BPR_SAMPLER_UNIFORM_USER, 1, 0.05, 0.0025, 0.0025, 0.00025, 0.0, 0,
                            N.BPR_SCHEDULE_HOGWILD)
            N.check(L.mml_bpr_create(ctx.handle, ctypes.byref(p), n_users, n_items, ctypes.byref(h)))
            N.check(L.mml_bpr_set_model(h, f(U), f(V), f(bi)))
            N.check(L.mml_bpr_get_model(h, f(got[0]), f(got[1]), f(got[3])))
            want, got = (U, V, bi), (got[0], got[1], got[3])
        for x, y in zip(want, got):
            np.testing.assert_array_equal(x, y)
    finally:
        getattr(L, f"mml_{model}_destroy")(h)
        ctx.close()
