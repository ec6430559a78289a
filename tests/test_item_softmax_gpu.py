"""The softmax over the catalogue (item_log_probs, item_log_probs_grad) against its definition in 64
bits.

Tolerances.  With A_r = max_j (sum_f |u_f v_jf| + |b_j|) a score is off by at most
(12 + 12 KT + 8) 2^-24 A_r: f32 factors are split into two f16 planes, hi off by 2^-11, lo (below
2^-11 of the value) by 2^-11 of itself, so a factor is off by 2^-22 = 4 units of 2^-24, two factors by
8, the dropped lo lo is 4 more; two roundings for each of at most 6 KT accumulations (KT = steps of 16
factors); 8 for the bias and the product with log2 e.  The planes are scaled to a largest magnitude
of 2^12 at least and end at 2^-25 (half the smallest f16): 2^-37 of the matrix' largest value, for each
of the k products and both factors, is lost below.  The log normaliser adds the roundings of the exponents (|y| <= 64 where e
counts) and of the sum (one per tile and 16 within).  Half-precision factors are exact operands, so
the bound holds for them too.  An entropy moves by 2 d (H + 1) for a change d of every log p, and
its sum rounds as the normaliser's: 4 d (H + 1).
Gradients: G is off by 4 d |G|-like terms (G's parts taken with their magnitudes), each product's
split by 12 x 2^-24 as above (f32) or 2^-16 (G in two planes), every accumulated step rounds twice, and
G's planes lose 2^-37 of the largest |G| of the kept row, for each element of the sum.  What
is returned in half precision is off by half a step, finfo.eps / 2, more.
"""
import numpy as np
import pytest
import torch

from mymedialite_amd import _native as N
from mymedialite_amd import item_log_probs, item_log_probs_grad

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
EPS = 2.0 ** -24


def steps(k):
    kt = 1
    while 16 * kt < k:
        kt *= 2
    return kt


def make(R, n_items, k, dtype, seed=0, n_users=None, seen=0, std=None):
    rs = np.random.default_rng(seed)
    n_users = n_users or R
    std = std or np.sqrt(2.0 / np.sqrt(k))
    U = torch.tensor(rs.normal(0, std, (n_users, k)), dtype=F32).to(dtype)
    V = torch.tensor(rs.normal(0, std, (n_items, k)), dtype=F32).to(dtype)
    b = torch.tensor(-0.8 * np.log(1.0 + rs.permutation(n_items)), dtype=F32)
    users = torch.tensor(rs.integers(0, n_users, R), dtype=torch.int32) if n_users != R else None
    items = torch.tensor(rs.integers(0, n_items, R), dtype=torch.int32)
    ex = None
    if seen:
        lists = [rs.integers(0, n_items, rs.integers(0, 2 * seen + 1)) for _ in range(n_users)]
        off = np.concatenate([[0], np.cumsum([len(x) for x in lists])])
        ex = (torch.tensor(off, dtype=torch.int64),
              torch.tensor(np.concatenate(lists), dtype=torch.int32))
    return dict(U=U, V=V, b=b, users=users, items=items, ex=ex)


def reference(d, n_top=0, g_lp=None, g_ent=None):
    """The definition in 64 bits on the CPU, with the magnitudes that the tolerances need."""
    U, V = d["U"].double().numpy(), d["V"].double().numpy()
    n = V.shape[0]
    b = np.zeros(n) if d["b"] is None else d["b"].double().numpy()
    users = np.arange(U.shape[0]) if d["users"] is None else d["users"].numpy()
    R = len(users)
    u = np.zeros((R, U.shape[1]))
    known = (users >= 0) & (users < U.shape[0])
    u[known] = U[users[known]]
    gone = np.zeros((R, n), bool)
    gone[:, b <= -1e30] = True
    if d["ex"] is not None:
        off, ids = d["ex"][0].numpy(), d["ex"][1].numpy()
        for r in np.flatnonzero(known):
            x = ids[off[users[r]]:off[users[r] + 1]]
            gone[r, x[(x >= 0) & (x < n)]] = True
    Vz = np.where(np.isfinite(V), V, 0.0)
    bz = np.where(b <= -1e30, 0.0, b)
    s = u @ Vz.T + bz
    A = np.where(gone, 0.0, np.abs(u) @ np.abs(Vz).T + np.abs(bz)).max(1)
    s[gone] = -np.inf
    m = s.max(1)
    m0 = np.where(np.isfinite(m), m, 0.0)
    with np.errstate(divide="ignore", invalid="ignore"):
        lse = m0 + np.log(np.exp(s - m0[:, None]).sum(1))
        logp = s - lse[:, None]
    logp[~np.isfinite(m)] = -np.inf
    p = np.exp(logp)
    lz = np.where(p > 0, logp, 0.0)
    H = -(p * lz).sum(1)
    out = dict(lse=lse, H=H, A=A, gone=gone)
    t = np.full(R, -1) if d["items"] is None else d["items"].numpy()
    has = (t >= 0) & (t < n)
    tt = np.where(has, t, 0)
    out["lp"] = np.where(has, logp[np.arange(R), tt], 0.0)
    if n_top:
        ids = np.full((R, n_top), -1, np.int64)
        lp = np.full((R, n_top), -np.inf)
        for r in range(R):
            o = np.lexsort((np.arange(n), -s[r]))[:n_top]
            o = o[~gone[r, o]]
            ids[r, :len(o)], lp[r, :len(o)] = o, logp[r, o]
        out["top"], out["top_lp"] = ids, lp
    if g_lp is not None or g_ent is not None:
        w = np.zeros(R) if g_lp is None else g_lp.double().numpy().copy()
        h = np.zeros(R) if g_ent is None else g_ent.double().numpy()
        w[~has | (p[np.arange(R), tt] == 0) | ~known] = 0.0
        w[~np.isfinite(lse)] = 0.0
        h = np.where(np.isfinite(lse) & known, h, 0.0)
        delta = np.zeros_like(p)
        delta[np.arange(R), tt] = w
        G = delta - w[:, None] * p - h[:, None] * p * (lz + H[:, None])
        mag = np.abs(delta) + np.abs(w)[:, None] * p + np.abs(h)[:, None] * p * (
            np.abs(lz) + H[:, None] + 1)
        out.update(gu=G @ Vz, gv=G.T @ u, gb=G.sum(0), mag=mag, magu=mag @ np.abs(Vz),
                   magv=mag.T @ np.abs(u), magb=mag.sum(0),
                   sumv=np.abs(Vz).sum(0), sumu=np.abs(np.where(np.isfinite(u), u, 0)).sum(0))
    return out


def tol_score(d, ref):
    k, n = d["V"].shape[1], d["V"].shape[0]
    tiles = -(-n // 32)
    top = lambda x: float(x[torch.isfinite(x).all(1)].abs().max().double())
    return EPS * ((12 + 12 * steps(k) + 8) * ref["A"] + 64 + tiles + 16
                  + 2 * 2.0 ** -13 * k * top(d["U"]) * top(d["V"]) + 4 * np.abs(np.where(np.isfinite(ref["lse"]), ref["lse"], 0)))


def to_gpu(d):
    g = lambda x: None if x is None else x.cuda()
    return dict(U=g(d["U"]), V=g(d["V"]), b=g(d["b"]), users=g(d["users"]), items=g(d["items"]),
                ex=None if d["ex"] is None else tuple(x.cuda() for x in d["ex"]))


def forward(c, n_top=0):
    return item_log_probs(c["U"], c["V"], c["b"], items=c["items"], users=c["users"],
                          exclude=c["ex"], n_top=n_top)


def backward(c, r, g_lp, g_ent):
    return item_log_probs_grad(c["U"], c["V"], c["b"], items=c["items"], users=c["users"],
                               exclude=c["ex"], log_norm=r.log_norm, entropy=r.entropy,
                               grad_log_probs=None if g_lp is None else g_lp.cuda(),
                               grad_entropy=None if g_ent is None else g_ent.cuda())


def near(got, want, tol):
    got = got.double().cpu().numpy()
    fine = np.isfinite(want)
    np.testing.assert_array_equal(np.where(fine, 0, got), np.where(fine, 0, want))
    off = np.abs(np.where(fine, got - np.where(fine, want, 0), 0))
    assert (off <= np.broadcast_to(tol, off.shape)).all(), (off / np.broadcast_to(tol, off.shape)).max()


def check_forward(d, r, n_top=0, ref=None):
    ref = ref or reference(d, n_top)
    tol = tol_score(d, ref)
    near(r.log_norm, ref["lse"], tol)
    near(r.log_probs, ref["lp"], 2 * tol + EPS * np.abs(np.where(np.isfinite(ref["lp"]), ref["lp"], 0)))
    near(r.entropy, ref["H"], 4 * tol * (ref["H"] + 1))
    if n_top:
        np.testing.assert_array_equal(r.top_items.cpu().numpy(), ref["top"])
        near(r.top_log_probs, ref["top_lp"], 2 * tol[:, None] + 64 * EPS)


def check_backward(d, got, ref):
    k, n, R = d["V"].shape[1], d["V"].shape[0], len(ref["lse"])
    tol = tol_score(d, ref)
    split = 12 * EPS if d["U"].dtype == F32 else 2.0 ** -16
    half = 0.0 if d["U"].dtype == F32 else torch.finfo(d["U"].dtype).eps / 2
    tiny = 0.0 if d["U"].dtype != F16 else 2.0 ** -25  # half the smallest f16
    gu, gv, gb = got
    assert gu.dtype == gv.dtype == d["U"].dtype and gb.dtype == F32
    # f32 holds nothing below 2^-126: a p, a G or a lower plane of G under it is lost, which is at
    # most 2^-126 (|w| + |h| (|log p| + H)) < 2^-126 * 2^8 per element (|log p| <= 88 where p is
    # held, w and h <= 1 here), times the other factor, for each of the contracted rows
    lost = 2.0 ** -118
    lost_u = lost * n * float(d["V"][torch.isfinite(d["V"]).all(1)].abs().max().double())
    lost_v = lost * R * float(d["U"].abs().max().double())
    fine = 2.0 ** -37 * ref["mag"]
    below_u = fine.max(1)[:, None] * ref["sumv"]
    below_v = fine.max(0)[:, None] * ref["sumu"]
    acc = lambda m: 24 * -(-m // 32) * EPS  # 2 steps x 6 products x 2 roundings per tile
    near(gu, ref["gu"], ref["magu"] * (4 * tol[:, None] + split + acc(n) + 64 * EPS)
         + half * np.abs(ref["gu"]) + tiny + lost_u + below_u)
    near(gv, ref["gv"], ref["magv"] * (4 * tol.max() + split + acc(R) + 64 * EPS)
         + half * np.abs(ref["gv"]) + tiny + lost_v + below_v)
    near(gb, ref["gb"], ref["magb"] * (4 * tol.max() + (R + 64) * EPS) + lost * R)


SHAPES = [  # rows, items, k, n_users
    (1, 1, 1, 1), (1, 33, 3, 4), (2, 31, 16, 2), (7, 100, 10, 20), (32, 64, 17, 32),
    (33, 1682, 10, 50), (64, 500, 64, 64), (65, 333, 100, 65), (130, 257, 128, 131),
    (31, 4099, 33, 31), (40, 129, 256, 40), (3, 700, 200, 5),
]


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_forward(shape, dtype):
    R, n, k, nu = shape
    for seen, n_top in ((0, 0), (9, 5)):
        d = make(R, n, k, dtype, seed=R + n, n_users=nu, seen=seen)
        if seen == 0:
            d["b"] = None
        check_forward(d, forward(to_gpu(d), n_top), n_top)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_gradient(shape, dtype):
    R, n, k, nu = shape
    rs = np.random.default_rng(5)
    for seen, ent in ((0, False), (9, True)):
        d = make(R, n, k, dtype, seed=R + 2 * n, n_users=nu, seen=seen)
        g_lp = torch.tensor(rs.normal(0, 1.0 / R, R), dtype=F32)
        g_ent = torch.tensor(rs.normal(0, 0.3 / R, R), dtype=F32) if ent else None
        c = to_gpu(d)
        ref = reference(d, 0, g_lp, g_ent)
        check_backward(d, backward(c, forward(c), g_lp, g_ent), ref)


@pytest.mark.parametrize("rows,n_items,k", [(300, 20_001, 64), (40, 70_003, 32), (1, 100_000, 64),
                                            (500, 3001, 48)])
def test_long_catalogue(rows, n_items, k):
    """Many tiles and splits, top 100, a user listed several times."""
    d = make(rows, n_items, k, F32, seed=3, n_users=max(1, rows // 2), seen=60)
    c = to_gpu(d)
    r = forward(c, 100)
    g_lp = torch.full((rows,), -1.0 / rows)
    ref = reference(d, 100, g_lp)
    check_forward(d, r, 100, ref)
    check_backward(d, backward(c, r, g_lp, None), ref)


def test_gradient_against_differences():
    """The gradient against central differences of the forward definition in 64 bits."""
    d = make(5, 40, 6, F32, seed=1, seen=4)
    rs = np.random.default_rng(2)
    g_lp, g_ent = (torch.tensor(rs.normal(0, 1, 5), dtype=F32) for _ in range(2))

    def loss(e):
        r = reference(e)
        lp = np.where(np.isfinite(r["lp"]), r["lp"], 0.0)
        return float((lp * g_lp.double().numpy()).sum() + (r["H"] * g_ent.double().numpy()).sum())

    c = to_gpu(d)
    got = backward(c, forward(c), g_lp, g_ent)
    step = 1e-5
    for name, g in (("U", got[0]), ("V", got[1]), ("b", got[2])):
        x = d[name].double()
        want = torch.zeros_like(x)
        for i in range(x.numel()):
            e = [dict(d), dict(d)]
            for s, y in ((step, e[0]), (-step, e[1])):
                z = x.clone()
                z.view(-1)[i] += s
                y[name] = z
            want.view(-1)[i] = (loss(e[0]) - loss(e[1])) / (2 * step)
        # differences: step^2 / 6 x third derivatives (< 100 here) + rounding 1e-15 / step
        np.testing.assert_allclose(g.double().cpu().numpy(), want.numpy(), atol=2e-5, rtol=2e-5)


def test_masks_and_empty_rows():
    """-inf, the type's lowest value and -1e30 in the bias exclude an item for everyone, whatever
    its factors hold; a row whose list holds the rest is empty."""
    d = make(40, 70, 20, F32, seed=4, n_users=40)
    d["b"][3] = -np.inf
    d["b"][50] = torch.finfo(F32).min
    d["b"][69] = -1e30
    d["V"][3] = float("nan")
    d["V"][50, 2] = float("inf")
    off = np.zeros(41, np.int64)
    off[6:] = 140  # user 5: every item, twice, unsorted, and ids outside the catalogue
    off[8:] = 144  # user 7: two items and two ids outside
    ids = np.concatenate([np.arange(70)[::-1], np.arange(70), [4, -1, 70, 9]])
    d["ex"] = (torch.tensor(off), torch.tensor(ids, dtype=torch.int32))
    d["items"][0] = 3     # excluded for everyone
    d["items"][7] = 9     # excluded for user 7
    d["items"][1] = -1
    d["items"][2] = 70
    c = to_gpu(d)
    r = forward(c, 4)
    g_lp, g_ent = torch.full((40,), 0.25), torch.full((40,), -0.5)
    ref = reference(d, 4, g_lp, g_ent)
    check_forward(d, r, 4, ref)
    assert r.log_norm[5] == -np.inf and r.entropy[5] == 0 and (r.top_items[5] == -1).all()
    assert r.log_probs[5] == -np.inf and r.log_probs[0] == -np.inf and r.log_probs[7] == -np.inf
    assert r.log_probs[1] == 0 and r.log_probs[2] == 0
    got = backward(c, r, g_lp, g_ent)
    check_backward(d, got, ref)
    assert (got[0][5] == 0).all()
    for i in (3, 50, 69):
        assert (got[1][i] == 0).all() and got[2][i] == 0


def test_everything_excluded():
    d = make(3, 40, 8, F32)
    d["b"][:] = -np.inf
    c = to_gpu(d)
    r = forward(c, 2)
    assert (r.log_norm == -np.inf).all() and (r.entropy == 0).all() and (r.top_items == -1).all()
    for g in backward(c, r, torch.ones(3), torch.ones(3)):
        assert (g == 0).all()


def test_not_finite_values_stay_in_their_rows():
    """A NaN user row makes its own outputs NaN and no other's; without a gradient of its own it
    adds nothing to the items'.  An unknown user is NaN; a NaN item makes every row NaN unless the
    row excludes it."""
    d = make(34, 90, 12, F32, seed=6, n_users=34)
    d["users"] = torch.arange(34, dtype=torch.int32)
    clean = reference(d)
    d["U"][10, 3] = float("nan")
    d["U"][33, 0] = float("inf")
    d["users"][4] = 34
    d["users"][5] = -7
    c = to_gpu(d)
    r = forward(c, 3)
    bad = np.zeros(34, bool)
    bad[[10, 33, 4, 5]] = True
    for x in (r.log_norm, r.entropy, r.log_probs):
        np.testing.assert_array_equal(np.isnan(x.cpu().numpy()), bad)
    assert (r.top_items.cpu().numpy()[bad] == -1).all()
    tol = tol_score(d, clean)
    np.testing.assert_array_less(np.abs(r.log_norm.cpu().numpy() - clean["lse"])[~bad], tol[~bad])
    g_lp = torch.full((34,), 1.0)
    g_lp[[10, 33]] = 0.0
    gu, gv, gb = backward(c, r, g_lp, None)
    assert torch.isfinite(gu).all() and torch.isfinite(gv).all() and torch.isfinite(gb).all()
    assert (gu[[4, 5, 10, 33]] == 0).all()
    g_lp[10] = 1.0
    gu, gv, gb = backward(c, r, g_lp, None)
    assert torch.isnan(gu[10]).all() and torch.isfinite(gu[[0, 9, 11]]).all()

    d = make(3, 90, 12, F32, seed=6)
    d["V"][77, 1] = float("nan")
    d["ex"] = (torch.tensor([0, 0, 1, 1]), torch.tensor([77], dtype=torch.int32))
    c = to_gpu(d)
    r = forward(c, 3)
    np.testing.assert_array_equal(np.isnan(r.log_norm.cpu().numpy()), [True, False, True])
    check = reference(d, 3)
    assert abs(float(r.log_norm[1]) - check["lse"][1]) <= tol_score(d, check)[1]
    np.testing.assert_array_equal(r.top_items[1].cpu().numpy(), check["top"][1])
    gu, _, _ = backward(c, r, torch.tensor([0.0, 1.0, 0.0]), None)
    assert torch.isfinite(gu[1]).all()


def test_ties_go_to_the_lowest_id():
    """Rows of zeros (untrained users and items) tie exactly; n_top over the catalogue pads."""
    d = make(5, 300, 16, F32, seed=8)
    d["b"] = None
    d["U"][1] = 0
    d["V"][100:260] = d["V"][7]
    c = to_gpu(d)
    check_forward(d, forward(c, 120), 120)
    assert (forward(c, 128).top_items[1].cpu() == torch.arange(128)).all()
    d = make(2, 5, 4, F32, seed=9)
    r = forward(to_gpu(d), 8)
    check_forward(d, r, 8)
    assert (r.top_items[:, 5:] == -1).all()


def test_large_scores():
    """Scores of several hundred: the softmax is nearly one-hot and nothing overflows."""
    d = make(33, 400, 64, F32, seed=10, std=4.0)
    g_lp, g_ent = torch.ones(33), torch.full((33,), 0.1)
    c = to_gpu(d)
    r = forward(c, 3)
    ref = reference(d, 3, g_lp, g_ent)
    check_forward(d, r, 3, ref)
    check_backward(d, backward(c, r, g_lp, g_ent), ref)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
def test_strides_and_offsets(dtype):
    """Padded rows, columns of a wider matrix, an unaligned base, a transposed matrix, every other
    entry of a vector: the same numbers as contiguous tensors bit for bit."""
    d = make(40, 200, 24, dtype, seed=11, seen=5)
    c = to_gpu(d)
    want = forward(c, 4)
    g = torch.full((40,), 0.5)
    gw = backward(c, want, g, None)

    def wide(x, pad, at):
        y = torch.full((x.shape[0], x.shape[1] + pad), 7.0, dtype=x.dtype, device="cuda")
        y[:, at:at + x.shape[1]] = x
        return y[:, at:at + x.shape[1]]

    forms = [dict(c, U=wide(c["U"], 8, 0), V=wide(c["V"], 40, 16)),
             dict(c, U=wide(c["U"], 3, 1), V=wide(c["V"], 5, 3)),
             dict(c, U=c["U"].t().contiguous().t(), V=c["V"].t().contiguous().t()),
             dict(c, b=torch.stack([c["b"], c["b"]], 1)[:, 0],
                  items=torch.stack([c["items"], c["items"]], 1)[:, 1])]
    for e in forms:
        got = forward(e, 4)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        for a, b in zip(backward(e, got, g, None), gw):
            assert torch.equal(a, b)


def test_no_rows_and_no_items_given():
    d = make(4, 50, 8, F32, seed=12)
    c = to_gpu(d)
    c["users"] = torch.zeros(0, dtype=torch.int32, device="cuda")
    c["items"] = None
    r = forward(c, 3)
    assert r.log_norm.shape == (0,) and r.top_items.shape == (0, 3)
    gu, gv, gb = backward(c, r, None, None)
    assert gu.shape == (0, 8) and (gv == 0).all() and (gb == 0).all()
    d["items"] = None
    check_forward(d, forward(to_gpu(d), 2), 2)


def test_two_streams_at_once():
    """Calls on two side streams, their tensors made there, and the same result every time."""
    d = make(200, 5000, 64, F32, seed=13, n_users=300, seen=20)
    c = to_gpu(d)
    g = torch.full((200,), -0.005)
    want = forward(c, 10)
    gw = backward(c, want, g, None)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                e = dict(c, U=c["U"] * 1.0)
                r = forward(e, 10)
                got.append((r, backward(e, r, g, None)))
    torch.cuda.synchronize()
    for r, b in got:
        for x, y in zip((*r, *b), (*want, *gw)):
            assert torch.equal(x, y)


def test_captured_graphs():
    """Two graphs of forward and backward, replayed in turn with new inputs and eager work between
    the replays, equal the eager results bit for bit."""
    d = make(70, 3001, 32, F32, seed=14, n_users=100, seen=10)
    c = to_gpu(d)
    g = torch.full((70,), -0.01, device="cuda")

    def both(e):
        r = forward(e, 7)
        return (*r, *item_log_probs_grad(e["U"], e["V"], e["b"], items=e["items"],
                                         users=e["users"], exclude=e["ex"], log_norm=r.log_norm,
                                         entropy=r.entropy, grad_log_probs=g, grad_entropy=g))

    both(c)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        e = dict(c, U=c["U"].clone())
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = both(e)
        graphs.append((gr, e, out))
    for i in range(6):
        gr, e, out = graphs[i % 2]
        e["U"].copy_(c["U"] * (1.0 + 0.1 * i))
        gr.replay()
        want = both(e)
        torch.cuda.synchronize()
        for x, y in zip(out, want):
            assert torch.equal(x, y)


def test_refusals():
    d = make(4, 50, 8, F32)
    c = to_gpu(d)
    ok = dict(user_factors=c["U"], item_factors=c["V"], item_bias=c["b"], items=c["items"])

    def refuse(error, text, **kw):
        with pytest.raises(error, match=text):
            item_log_probs(**dict(ok, **kw))

    refuse(ValueError, "must be float32", user_factors=c["U"].double(), item_factors=c["V"].double())
    refuse(ValueError, "one dtype", item_factors=c["V"].to(BF16))
    refuse(ValueError, "on the GPU", user_factors=d["U"])
    refuse(ValueError, "2-D", item_factors=c["V"][0])
    refuse(ValueError, "item factors", item_factors=c["V"][:, :5])
    refuse(ValueError, "item_bias has", item_bias=c["b"][:9])
    refuse(ValueError, "items must be", items=c["items"].long())
    refuse(ValueError, "items has", items=c["items"][:2])
    refuse(ValueError, "is on cpu", item_bias=d["b"])
    refuse(ValueError, r"exclude\[0\] has", exclude=(torch.zeros(4, dtype=torch.int64, device="cuda"),
                                                     c["items"]))
    refuse(N.MMLError, "n_top", n_top=129)
    refuse(N.MMLError, "n_top", n_top=-1)
    refuse(N.MMLError, "num_factors", user_factors=torch.zeros(4, 257, device="cuda"),
           item_factors=torch.zeros(50, 257, device="cuda"))
    refuse(N.MMLError, "n_items", item_factors=c["V"][:0], item_bias=None)
    with pytest.raises(N.MMLError, match="grad_entropy without entropy"):
        item_log_probs_grad(**ok, log_norm=torch.zeros(4, device="cuda"),
                            grad_entropy=torch.ones(4, device="cuda"))
    with pytest.raises(ValueError, match="log_norm is required"):
        item_log_probs_grad(**ok, log_norm=None)
    check_forward(d, forward(c))  # and the next call is unharmed


@pytest.mark.parametrize("rows,n_items", [(5, 333), (300, 30_001)], ids=["few", "many"])
@pytest.mark.parametrize("up,vp", [(60, -60), (-60, 60), (-30, -30), (-100, 0), (0, -100), (-24, 13)])
def test_factors_of_any_magnitude(rows, n_items, up, vp):
    """f32 factors times 2^up and 2^vp: what is held of them does not depend on their size."""
    d = make(rows, n_items, 17, F32, seed=8)
    d["U"] *= 2.0 ** up
    d["V"] *= 2.0 ** vp
    c = to_gpu(d)
    r = forward(c, 3)
    g_lp, g_ent = torch.full((rows,), -1.0 / rows), torch.full((rows,), 0.1 / rows)
    ref = reference(d, 3, g_lp, g_ent)
    check_forward(d, r, 3, ref)
    check_backward(d, backward(c, r, g_lp, g_ent), ref)


@pytest.mark.parametrize("dtype,huge", [(F32, 1e20), (F32, 2e38), (F32, float("inf")), (BF16, 1e38),
                                        (F16, 6e4)])
@pytest.mark.parametrize("rows,n_items", [(5, 333), (300, 30_001)], ids=["few", "many"])
def test_excluded_items_factors_do_not_matter(rows, n_items, dtype, huge):
    """Items that their bias excludes, with factors of any size: every result is the one of zeros."""
    d = make(rows, n_items, 17, dtype, seed=9)
    out = torch.arange(0, n_items, 11)
    d["b"][out] = torch.tensor([-np.inf, -1e30, -3e38], dtype=F32).repeat(len(out))[:len(out)]
    d["V"][out] = 0
    clean = dict(d, V=d["V"].clone())
    d["V"][out] = torch.randn(len(out), 17).sign().mul(huge).to(dtype)
    c = to_gpu(d)
    r = forward(c, 3)
    g_lp, g_ent = torch.full((rows,), -1.0 / rows), torch.full((rows,), 0.1 / rows)
    ref = reference(clean, 3, g_lp, g_ent)
    check_forward(clean, r, 3, ref)
    got = backward(c, r, g_lp, g_ent)
    check_backward(clean, got, ref)
    assert (got[1][out.cuda()] == 0).all() and (got[2][out.cuda()] == 0).all()


def test_products_beyond_f32_are_nan():
    """Factors whose products leave f32 (2^121) give NaN, not a number of the wrong size."""
    for rows, n_items in ((5, 333), (300, 30_001)):
        d = make(rows, n_items, 17, F32, seed=10)
        d["U"] *= 2.0 ** 62
        d["V"] *= 2.0 ** 62
        r = forward(to_gpu(d), 2)
        assert torch.isnan(r.log_norm).all() and torch.isnan(r.log_probs).all()
        assert (r.top_items == -1).all()


@pytest.mark.parametrize("dtype,k", [(F32, 5), (BF16, 130)], ids=["f32", "bf16"])
def test_gradient_with_a_few_items_more_than_fit(dtype, k):
    """A catalogue just above what the CUs hold at once: the items behind it are split over the rows
    and joined, the others are not."""
    rows, n_items = 300, (98_500 if dtype == F32 else 65_700)
    d = make(rows, n_items, k, dtype, seed=12, seen=3)
    c = to_gpu(d)
    r = forward(c)
    g_lp, g_ent = torch.full((rows,), -1.0 / rows), torch.full((rows,), 0.1 / rows)
    check_backward(d, backward(c, r, g_lp, g_ent), reference(d, 0, g_lp, g_ent))


@pytest.mark.parametrize("rows,n_items", [(3, 1682), (600, 1682), (520, 4100), (2, 4100), (530, 900)])
def test_many_top_items_of_few(rows, n_items):
    """128 top items of a catalogue with few tiles of 32; the last rows tie in all of it."""
    d = make(rows, n_items, 12, F32, seed=13, seen=40)
    d["b"][:] = torch.randn(n_items)
    d["U"][-1] = 0
    check_forward(d, forward(to_gpu(d), 128), 128)
    d["b"] = None
    r = forward(to_gpu(d), 128)
    check_forward(d, r, 128)
    ids, off = d["ex"][1].numpy(), d["ex"][0].numpy()
    rest = np.setdiff1d(np.arange(n_items), ids[off[rows - 1]:off[rows]])
    np.testing.assert_array_equal(r.top_items[-1].cpu().numpy(), rest[:128])


def test_odd_factors_and_idle_waves():
    """k not a multiple of 4 over one long array (the scale is found one value at a time) and one tile
    of users more than a block keeps."""
    d = make(257, 20_011, 19, F32, seed=14, seen=10)
    d["V"][20_010, 18] = 300.0
    d["b"][20_010] = -600.0
    c = to_gpu(d)
    r = forward(c, 4)
    g_lp, g_ent = torch.full((257,), -1.0 / 257), torch.full((257,), 0.1 / 257)
    ref = reference(d, 4, g_lp, g_ent)
    check_forward(d, r, 4, ref)
    check_backward(d, backward(c, r, g_lp, g_ent), ref)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", [(40, 700, 65, 41), (300, 9000, 96, 300), (5, 333, 90, 9),
                                   (70, 1100, 129, 70), (290, 6000, 192, 300), (3, 500, 170, 3)],
                         ids=lambda s: "x".join(map(str, s)))
def test_factors_between_powers_of_two(shape, dtype):
    R, n, k, nu = shape
    d = make(R, n, k, dtype, seed=R + k, n_users=nu, seen=9)
    g_lp, g_ent = torch.full((R,), -1.0 / R), torch.full((R,), 0.1 / R)
    c = to_gpu(d)
    r = forward(c, 5)
    ref = reference(d, 5, g_lp, g_ent)
    check_forward(d, r, 5, ref)
    check_backward(d, backward(c, r, g_lp, g_ent), ref)


@pytest.mark.parametrize("k", [1, 2, 3, 5, 7, 90, 97])
@pytest.mark.parametrize("where", ["first", "last", "excluded"])
def test_largest_factor_anywhere(k, where):
    """The scale counts the first and the last value of one long array, and no excluded item's."""
    rows, n_items = 300, 20_003
    d = make(rows, n_items, k, F32, seed=15)
    d["U"] *= 1e-3
    big = {"first": (0, 0), "last": (n_items - 1, k - 1), "excluded": (777, 0)}[where]
    d["V"][big] = 2.0 ** 20
    clean = d
    if where == "excluded":  # counted, it would leave the others 2^-37 2^100
        d["b"][777] = -np.inf
        clean = dict(d, V=d["V"].clone())
        clean["V"][777] = 0
        d["V"][big] = 2.0 ** 100
    else:
        d["U"][:, big[1]] *= 1e-4
    c = to_gpu(d)
    r = forward(c, 3)
    g_lp, g_ent = torch.full((rows,), -1.0 / rows), torch.full((rows,), 0.1 / rows)
    ref = reference(clean, 3, g_lp, g_ent)
    check_forward(clean, r, 3, ref)
    check_backward(clean, backward(c, r, g_lp, g_ent), ref)


@pytest.mark.parametrize("rows", [3, 40], ids=["few", "prepared"])
def test_exclusions_of_a_catalogue_in_parts(rows):
    """More items than one block's exclusion bits (516,096), f32, items of every part excluded."""
    d = make(rows, 1_050_000, 2, F32, seed=16, seen=200)
    d["items"][1] = int(d["ex"][1][int(d["ex"][0][1])])  # one that user 1 excludes
    c = to_gpu(d)
    r = forward(c, 2)
    g_lp = torch.full((rows,), -1.0 / rows)
    ref = reference(d, 2, g_lp)
    check_forward(d, r, 2, ref)
    assert r.log_probs[1] == -np.inf
    check_backward(d, backward(c, r, g_lp, None), ref)
