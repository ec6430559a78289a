"""The oracle's loops that take neighbouring ratings, triples or rows together give what they give one by
one, bit for bit (sizes small enough that rows collide in a group, and large enough that they do not)."""
import ctypes

import numpy as np
import pytest

import oracle as O


@pytest.mark.parametrize("k", [1, 7, 64])
@pytest.mark.parametrize("n_users,n_items", [(3, 4), (30, 20), (5000, 4000)])
def test_bmf_iterate(k, n_users, n_items):
    rs = np.random.default_rng(k + n_users)
    n = 1003
    u, i = rs.integers(0, n_users, n).astype(np.int32), rs.integers(0, n_items, n).astype(np.int32)
    v = rs.integers(1, 6, n).astype(np.float32)
    start = (rs.normal(0, 0.3, (n_users, k)).astype(np.float32),
             rs.normal(0, 0.3, (n_items, k)).astype(np.float32),
             rs.normal(0, 0.3, n_users).astype(np.float32), rs.normal(0, 0.3, n_items).astype(np.float32))
    kw = dict(gb=np.float32(0.2), min_rating=np.float32(1), range_=np.float32(4), lr=0.05)
    order = rs.permutation(n).astype(np.int32)
    a, b, c = ([x.copy() for x in start] for _ in range(3))
    O.bmf_iterate(u, i, v, order, *a, **kw)
    for x in order:
        O.bmf_iterate(u, i, v, np.array([x], np.int32), *b, **kw)
    O.bmf_iterate_lockstep(u, i, v, order, *c, streams=1, step=1, threads=2, **kw)
    for x, y, z in zip(a, b, c):
        np.testing.assert_array_equal(x, y)
        np.testing.assert_array_equal(x, z)
    many, one = ([x.copy() for x in start] for _ in range(2))
    O.bmf_iterate_lockstep(u, i, v, order, *many, streams=37, step=3, threads=5, **kw)
    O.bmf_iterate_lockstep(u, i, v, order, *one, streams=37, step=3, threads=1, **kw)
    for x, y in zip(many, one):
        np.testing.assert_array_equal(x, y)


@pytest.mark.parametrize("k", [1, 33, 128])
@pytest.mark.parametrize("n_users,n_items", [(3, 4), (40, 60), (5000, 9000)])
def test_bpr_triples_and_epochs(k, n_users, n_items):
    rs = np.random.default_rng(k + n_users)
    n = 1003
    tu = rs.integers(0, n_users, n).astype(np.int32)
    ti, tj = (rs.integers(0, n_items, n).astype(np.int32) for _ in range(2))
    start = (rs.normal(0, 0.3, (n_users, k)).astype(np.float32),
             rs.normal(0, 0.3, (n_items, k)).astype(np.float32), rs.normal(0, 0.3, n_items).astype(np.float32))
    kw = dict(learn_rate=0.05, reg_u=0.0025, reg_i=0.003, reg_j=0.0004, bias_reg=0.01)
    a, b = ([x.copy() for x in start] for _ in range(2))
    O.bpr_apply_triples(tu, ti, tj, *a, **kw)
    for x in range(n):
        O.bpr_apply_triples(tu[x:x + 1], ti[x:x + 1], tj[x:x + 1], *b, **kw)
    for x, y in zip(a, b):
        np.testing.assert_array_equal(x, y)
    if n_items < 10:
        return
    key = np.unique(rs.integers(0, n_users, 3000).astype(np.int64) * n_items
                    + rs.integers(0, n_items, 3000))
    off, rows, srt = O.bpr_csr_distinct((key // n_items).astype(np.int32),
                                        (key % n_items).astype(np.int32), n_users)
    a, b, r = [x.copy() for x in start], [x.copy() for x in start], [O.Rng(5), O.Rng(5)]
    trace = np.empty((len(key), 3), np.int32)
    for _ in range(2):  # the generator goes on where the epoch left it
        O.bpr_epoch_from(r[0], off, rows, srt, len(key), *a, trace=trace, **kw)
        p = O._BprParams(k, 1, 1, 1, 0.05, 0.0025, 0.003, 0.0004, 0.01, n_users - 1, n_items - 1)
        plain = np.empty_like(trace)
        O.lib().ora_bpr_epoch(r[1]._buf, ctypes.byref(p), O._p(off, O._i64p), O._p(rows, O._i32p),
                              O._p(srt, O._i32p), len(key), *(O._p(x, O._f32p) for x in b),
                              O._p(plain, O._i32p))
        np.testing.assert_array_equal(trace, plain)
        for x, y in zip(a, b):
            np.testing.assert_array_equal(x, y)


def test_wrmf_threads():
    rs = np.random.default_rng(1)
    off = np.concatenate([[0], np.cumsum(rs.integers(0, 9, 40))]).astype(np.int64)
    cols = rs.integers(0, 50, off[-1]).astype(np.int32)
    H = rs.normal(0, 0.3, (50, 24)).astype(np.float32)
    many = np.zeros((40, 24), np.float32)
    O.wrmf_optimize(off, cols, many, H, 1.5, 0.02)
    one, HH = np.zeros_like(many), O.wrmf_square(H)
    O.lib().ora_wrmf_optimize_rows(O._p(off, O._i64p), O._p(cols, O._i32p), 0, 40, 40,
                                   O._p(one, O._f32p), O._p(H, O._f32p), O._p(HH, O._f64p), 24, 1.5, 0.02)
    np.testing.assert_array_equal(many, one)
