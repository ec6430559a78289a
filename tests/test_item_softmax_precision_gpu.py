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
