"""Where the softmax over the catalogue loses bits if G or the scores are held carelessly."""
import numpy as np
import pytest
import torch

from mymedialite_amd import item_log_probs, item_log_probs_grad

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
EPS = 2.0 ** -24


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("k", [3, 64, 256])
def test_confident_rows(k, dtype):
    """Rows that give their item a probability of 1 - 1e-3 to 1 - 1e-6: dL/dU is made of G_t = w (1 - p_t),
    and what is lost is a share of that, not of w p_t.

    The users' factors are 0, so that scores are the biases, exactly: item 0 has 0 and the others less,
    row r excludes the others up to r.  Tolerance: with log_norm near 0, p_t = 2^x for a tiny x is off by
    two roundings next to 1, w p_t and the sum w - w p_t by one each, 4 EPS w in all; another p_j has an
    argument of 30 at most in base 2, known to 3 roundings of it and one of its own, 128 EPS of p_j;
    G's planes lose 2^-16 of an element (f32, f16: 2^-21, and 2^-37 of the row's largest); sums of 41
    elements in f32 round 2 x 3 products x 4 steps of 16 times; half a step of the result's type."""
    n, rows, w = 41, 39, -0.5
    rs = np.random.default_rng(k)
    V = torch.tensor(rs.normal(0, 1, (n, k)), dtype=F32).to(dtype)
    U = torch.zeros(rows, k, dtype=dtype)
    b = np.concatenate([[0.0], -10.5 - 0.08 * np.arange(n - 1)]).astype(np.float32)
    lists = [np.arange(1, r + 1) for r in range(rows)]
    off = np.concatenate([[0], np.cumsum([len(x) for x in lists])])
    c = dict(user_factors=U.cuda(), item_factors=V.cuda(), item_bias=torch.tensor(b).cuda(),
             items=torch.zeros(rows, dtype=torch.int32, device="cuda"),
             exclude=(torch.tensor(off).cuda(),
                      torch.tensor(np.concatenate(lists), dtype=torch.int32).cuda()))
    r = item_log_probs(**c)
    gu, gv, gb = item_log_probs_grad(**c, log_norm=r.log_norm,
                                     grad_log_probs=torch.full((rows,), w, device="cuda"))
    s = np.repeat(b[None].astype(np.float64), rows, 0)
    for x in range(rows):
        s[x, 1:x + 1] = -np.inf
    p = np.exp(s - r.log_norm.cpu().double().numpy()[:, None])  # of the norm that was handed over
    G = -w * p
    # the norm is f32's nearest, so 1 - p_t is the exact sum of the others up to 2^-24 of itself
    assert np.abs(p.sum(1) - 1).max() < 1e-6 and 5e-7 < (1 - p[:, 0]).min() < 1e-5
    G[:, 0] = w * -np.expm1(-r.log_norm.cpu().double().numpy())
    Vd = V.double().numpy()
    half = 0.0 if dtype == F32 else torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == F16 else 0.0
    split = 2.0 ** -16 if dtype == BF16 else 2.0 ** -21
    off_g = (128 + 48) * EPS * np.abs(G) + split * np.abs(G)
    off_g[:, 0] += 4 * EPS * abs(w)
    if dtype != BF16:
        off_g += 2.0 ** -37 * np.abs(G).max(1)[:, None]
    want = G @ Vd
    tol = off_g @ np.abs(Vd) + half * np.abs(want) + tiny
    err = np.abs(gu.double().cpu().numpy() - want)
    assert (err <= tol).all(), (err / tol).max()
    assert (gv == 0).all()
    tol_b = off_g.sum(0) + 39 * EPS * np.abs(G).sum(0)
    assert (np.abs(gb.double().cpu().numpy() - G.sum(0)) <= tol_b).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("level", [-3e3, -1e9, -1e13, -1e23, -9.9e27, -2e29])
@pytest.mark.parametrize("rows,n", [(5, 333), (300, 30_001)], ids=["few", "many"])
def test_scores_of_any_size_count(rows, n, level, dtype):
    """Items of a bias far below the others' but above -1e28 count where nothing else is left, in the
    rows that exclude the ten others.  From -1e9 on the products (at most 32, half a unit of f32 there)
    vanish beside the bias, and those rows are uniform, exactly so.  Below -1e28 (the last level) they
    are empty.  The same from one user tile and from many, for small and large factors (f32 factors are
    scaled by their largest).

    Tolerance: at -3e3 a score is off by (12 + 12 KT + 8) EPS of the largest |b| + sum |u v|, KT = 2, a
    log probability by twice that, an entropy by 2 d (H + 1) for both the scores and the norm; beyond,
    the scores are exact.  The norm is rounded to f32 and has lost log n from -1e9 on; the log
    probability, of the given item's score in 64 bits, is off by units of 2^-52 of the level.  Sums round twice an item that a lane sees,
    EPS n in all, the logarithm and the exponents 64 EPS."""
    rs = np.random.default_rng(3)
    k, left = 17, n - 10
    b = torch.full((n,), level)
    b[:10] = 0
    even = torch.arange(0, rows, 2)
    off = torch.tensor(np.concatenate([[0], np.cumsum([10 if r % 2 == 0 else 0 for r in range(rows)])]))
    ids = torch.arange(10, dtype=torch.int32).repeat(len(even))
    items = torch.tensor(rs.integers(10, n, rows), dtype=torch.int32)
    items[1::2] = 3
    for size in (1e-3, 1.0):
        U, V = (torch.tensor(rs.normal(0, size, x), dtype=F32).to(dtype) for x in ((rows, k), (n, k)))
        c = dict(user_factors=U.cuda(), item_factors=V.cuda(), item_bias=b.cuda(), items=items.cuda(),
                 exclude=(off.cuda(), ids.cuda()))
        r = item_log_probs(**c, n_top=4)
        norm, lp, H = (x.cpu().double().numpy() for x in (r.log_norm, r.log_probs, r.entropy))
        if level < -1e28:
            assert (norm[even] == -np.inf).all() and (lp[even] == -np.inf).all()
            assert (H[even] == 0).all() and (r.top_items.cpu()[even] == -1).all()
        else:
            S = (U.double() @ V[10:].double().T).numpy()[even]
            assert np.abs(S).max() < 32
            exact = S.copy()
            tol = 0.0
            if level > -1e8:
                A = (np.abs(U.double().numpy()) @ np.abs(V.double().numpy()).T).max() - level
                tol = (12 + 12 * 2 + 8) * EPS * A
            else:
                S[:] = 0.0
            want = np.log(np.exp(S - S.max(1)[:, None]).sum(1)) + S.max(1)  # without the level
            P = S - want[:, None]
            ent = -(np.exp(P) * P).sum(1)
            sums = EPS * (n + 64) * (1 + np.log(left))
            assert (np.abs(norm[even] - (level + want)) <= tol + sums - EPS * level).all()
            # the given item's own score is made in 64 bits
            given = ((exact + level) - level)[np.arange(len(even)), items.numpy()[even] - 10] - want
            assert (np.abs(lp[even] - given) <= 2 * tol + sums - 2.0 ** -51 * level).all()
            assert (np.abs(H[even] - ent) <= 4 * tol * (ent + 1) + sums).all()
            best = np.argsort(-S, axis=1, kind="stable")[:, :4]
            top = r.top_items.cpu().numpy()[even] - 10
            if level < -1e20:  # 64 bits lose the products too: the lowest ids
                np.testing.assert_array_equal(top, best)
            elif tol > 0:  # groups of items that come closer than the scores' error: any of them
                assert (np.take_along_axis(S, top, 1) >= np.take_along_axis(S, best, 1) - 2 * tol).all()
        odd = np.arange(1, rows, 2)
        S = (U.double() @ V[:10].double().T).numpy()[odd]
        want = np.log(np.exp(S).sum(1))
        np.testing.assert_allclose(norm[odd], want, rtol=0, atol=1e-5 * (1 + np.abs(S).max()))
        np.testing.assert_allclose(lp[odd], S[:, 3] - want, rtol=0, atol=1e-5 * (1 + np.abs(S).max()))
        g = torch.zeros(rows, device="cuda")
        g[1::2] = -1.0
        gu, gv, gb = item_log_probs_grad(**c, log_norm=r.log_norm, grad_log_probs=g)
        for x in (gu, gv, gb):
            assert torch.isfinite(x).all()
        assert (gu[0::2] == 0).all() and (gb[10:] == 0).all() and (gu[1::2] != 0).any()
        if level < -1e6:  # no gradient of such a norm (an empty row has none at all)
            g[0] = -1.0
            gu, gv, gb = item_log_probs_grad(**c, log_norm=r.log_norm, grad_log_probs=g)
            assert torch.isnan(gu[0]).all() if level >= -1e28 else (gu[0] == 0).all()
            assert torch.isfinite(gu[1:]).all()
