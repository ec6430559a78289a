"""The softmax over the catalogue of a trained recommender (BPRMF.log_probs, WRMF.log_probs) and the
steps on its loss (BPRMF.apply_softmax), which run item_log_probs, item_log_probs_grad and AdamW
together, against the definitions in 64 bits.

Tolerances.  Here |s| <= A = sum_f |u_f v_f| + |b| <= 8 and k <= 16 (one matrix step): a score is off
by (12 + 12 + 8) 2^-24 A <= 2^-16 = 1.6e-5 (f32 factors in two f16 planes: 12 units of 2^-24, the
accumulations 12, bias and exponent 8), a log probability and the normaliser by twice that and the
roundings of the sum: 5e-5; an entropy by 4 d (H + 1) with d = 5e-5 / 2.
A step: the mean loss' gradient is sum_r w_r (p - delta) x with sum |w_r| (p + delta) <= 2 and |x| <= X,
each term off by 4 d' relative (d' the score's error, A <= 1 in that test: 2e-6) and by 2^-16 of the
split of G at most: |dg| <= 2 X (8e-6 + 1.6e-5) = 5e-5 X.  A parameter then moves by at most
learn_rate (|dm| / epsilon + |m| |d sqrt v| / epsilon^2) more; sqrt v <= |g| scale and d sqrt v <= dg,
|m| / (sqrt v + epsilon) <= 8 over the steps here, so 9 learn_rate dg / epsilon a step.
"""
import numpy as np
import pytest

import mymedialite_amd as mml
from mymedialite_amd import _native as N

pytestmark = pytest.mark.gpu


def model(cls, n_users=70, n_items=133, k=10, seed=3, std=0.6, **kw):
    rs = np.random.default_rng(seed)
    fb = mml.PosOnlyFeedback(rs.integers(0, n_users, 900).astype(np.int32),
                             rs.integers(0, n_items, 900).astype(np.int32))
    # the last ids, so that the model has these sizes
    fb.users[-1], fb.items[-1] = n_users - 1, n_items - 1
    fb = mml.PosOnlyFeedback(fb.users, fb.items)
    r = cls(NumFactors=k, NumIter=1, InitStdDev=std, **kw)
    r.feedback = fb
    r.init_model()
    return r


def definition(r, users, items, exclude):
    """(log_probs, log_norm, entropy, scores with -inf for the excluded) in 64 bits"""
    m = r.get_model()
    U, V = m["U"].astype(np.float64), m["V"].astype(np.float64)
    b = m["bias"].astype(np.float64) if "bias" in m else np.zeros(len(V))
    s = np.full((len(users), len(V)), np.nan)
    ok = (users >= 0) & (users < len(U))
    s[ok] = U[users[ok]] @ V.T + b
    if exclude:
        for x, u in enumerate(users):
            if ok[x]:
                s[x, r.feedback.items[r.feedback.users == u]] = -np.inf
    with np.errstate(invalid="ignore", divide="ignore"):
        top = s.max(1, keepdims=True)
        norm = np.log(np.exp(s - top).sum(1)) + top[:, 0]
        lp = s - norm[:, None]
        p = np.exp(lp)
        H = -np.where(p > 0, p * lp, 0.0).sum(1)
    H[~ok] = np.nan
    given = np.zeros(len(users))
    for x in range(len(users)):
        if items is not None and 0 <= items[x] < len(V):
            given[x] = lp[x, items[x]]
        elif not ok[x]:
            given[x] = np.nan
    return given, norm, H, s


def check(r, users, items, n_top, exclude):
    users = np.asarray(users, np.int32)
    got = r.log_probs(users, items, n_top=n_top, exclude_training=exclude)
    given, norm, H, s = definition(r, users, items, exclude)
    np.testing.assert_allclose(got.log_norm, norm, rtol=0, atol=5e-5)
    np.testing.assert_allclose(got.log_probs, given, rtol=0, atol=5e-5)
    assert np.all((np.abs(got.entropy - H) <= 1e-4 * (H + 1)) | np.isnan(H))
    assert np.array_equal(np.isnan(got.entropy), np.isnan(H))
    if not n_top:
        assert got.top_items is None and got.top_log_probs is None
        return
    for x in range(len(users)):
        live = np.flatnonzero(np.isfinite(s[x]))
        best = live[np.lexsort((live, -s[x][live]))][:n_top]
        want = np.concatenate([best, np.full(n_top - len(best), -1)])
        assert np.array_equal(got.top_items[x], want)
        none = np.nan if np.isnan(norm[x]) else -np.inf  # a user beyond the model: NaN
        lp = np.concatenate([s[x][best] - norm[x], np.full(n_top - len(best), none)])
        np.testing.assert_allclose(got.top_log_probs[x], lp, rtol=0, atol=5e-5)


@pytest.mark.parametrize("cls", [mml.BPRMF, mml.WRMF])
@pytest.mark.parametrize("k", [1, 10, 16])
@pytest.mark.parametrize("exclude", [False, True])
def test_log_probs(cls, k, exclude):
    r = model(cls, k=k, std=0.6 / k ** 0.25)
    r.iterate()
    users = [0, 69, 5, 5, 33, 70, -1]  # one twice, two beyond the model
    items = [3, 132, 7, 8, -1, 0, 2]
    check(r, users, items, 5, exclude)
    check(r, users, None, 0, exclude)
    check(r, [4], [4], 128, exclude)
    check(r, np.arange(70), np.arange(70), 1, exclude)
    empty = r.log_probs([], [], n_top=2)
    assert empty.log_probs.shape == (0,) and empty.top_items.shape == (0, 2)


@pytest.mark.parametrize("cls", [mml.BPRMF, mml.WRMF])
def test_after_load(cls, tmp_path):
    """A loaded model has no training data to exclude."""
    r = model(cls)
    r.iterate()
    r.save_model(str(tmp_path / "m"))
    s = cls(NumFactors=10)
    s.load_model(str(tmp_path / "m"))
    s.feedback = r.feedback
    check(s, [0, 1, 2], [0, 1, 2], 3, False)
    with pytest.raises(N.MMLError, match="no training data"):
        s.log_probs([0], exclude_training=True)


@pytest.mark.parametrize("cls", [mml.BPRMF, mml.WRMF])
def test_refusals(cls):
    r = model(cls)
    for n_top in (-1, 129):
        with pytest.raises(N.MMLError, match="n_top"):
            r.log_probs([0], n_top=n_top)
    with pytest.raises(ValueError, match="one length"):
        r.log_probs([0, 1], [0])
    with pytest.raises(ValueError, match="1-D"):
        r.log_probs([[0, 1]])
    check(r, [0, 1], [0, 1], 3, True)


def test_shards():
    """A context of user shards on one GPU gives each row as the single device does."""
    a, b = model(mml.BPRMF), model(mml.BPRMF, Gpus="0,0")
    m = a.get_model()
    N.check(N.lib().mml_bpr_set_model(b._h, N.ptr(m["U"], N._f32p), N.ptr(m["V"], N._f32p),
                                      N.ptr(m["bias"], N._f32p)))
    b._host = None
    users = np.concatenate([np.arange(69, -1, -1), [70, -1]])
    for n_top in (0, 3):
        check(b, users, np.arange(72) - 1, n_top, True)
    with pytest.raises(NotImplementedError):
        b.apply_softmax([0], [0])


def test_rows_in_ranges():
    """More rows than one workspace of 1 GiB holds: every range's rows are those of the small call."""
    r = model(mml.BPRMF, n_users=40, n_items=20_000, k=2)
    n = 500_003  # the exclusion bits alone would take 1.2 GiB
    rs = np.random.default_rng(0)
    users = rs.integers(0, 40, n).astype(np.int32)
    items = rs.integers(0, 20_000, n).astype(np.int32)
    got = r.log_probs(users, items, n_top=1, exclude_training=True)
    given, norm, H, s = definition(r, np.arange(40), None, True)
    np.testing.assert_allclose(got.log_norm, norm[users], rtol=0, atol=5e-5)
    assert np.all(np.abs(got.entropy - H[users]) <= 1e-4 * (H[users] + 1))
    np.testing.assert_allclose(got.log_probs, (s - norm[:, None])[users, items], rtol=0, atol=5e-5)
    assert np.array_equal(got.top_items[:, 0], np.argmax(s, 1)[users])


# ------------------------------------------------------------------ steps on the loss
LR, EPSILON, DECAY, BETA1, BETA2 = 0.01, 0.01, 0.02, 0.9, 0.99


def steps_64(m, users, items, batch, start=None):
    """The same steps in 64 bits; start: (step, m, v)."""
    P = [x.astype(np.float64) for x in (m["U"], m["V"], m["bias"])]
    t, M, S = start or (0, [0.0] * 3, [0.0] * 3)
    M, S, losses = list(M), list(S), []
    for a in range(0, len(users), batch):
        u, i = users[a:a + batch], items[a:a + batch]
        s = P[0][u] @ P[1].T + P[2]
        lp = s - np.log(np.exp(s).sum(1, keepdims=True))
        losses.append(-lp[np.arange(len(u)), i].mean())
        G = np.exp(lp)
        G[np.arange(len(u)), i] -= 1.0
        G /= len(u)
        gU = np.zeros_like(P[0])
        np.add.at(gU, u, G @ P[1])
        t += 1
        for x, g in enumerate((gU, G.T @ P[0][u], G.sum(0))):
            M[x] = BETA1 * M[x] + (1 - BETA1) * g
            S[x] = BETA2 * S[x] + (1 - BETA2) * g * g
            P[x] = P[x] * (1 - LR * DECAY) - LR * M[x] / (1 - BETA1 ** t) / (
                np.sqrt(S[x] / (1 - BETA2 ** t)) + EPSILON)
    return P, np.array(losses), (t, M, S)


HYPER = dict(LearnRate=LR, Epsilon=EPSILON, WeightDecay=DECAY, Beta1=BETA1, Beta2=BETA2)


@pytest.mark.parametrize("n,batch", [(1, 1), (7, 100), (300, 64)])
def test_apply_softmax(n, batch):
    r = model(mml.BPRMF, std=0.2)
    before = {k: v.copy() for k, v in r.get_model().items()}
    rs = np.random.default_rng(n)
    users = rs.integers(0, 70, n).astype(np.int32)  # 300 events of 70 users: many twice in a batch
    items = rs.integers(0, 133, n).astype(np.int32)
    losses, state = r.apply_softmax(users, items, BatchSize=batch, **HYPER)
    want, loss64, at = steps_64(before, users, items, batch)
    n_steps = -(-n // batch)
    X = max(1.0, max(np.abs(p).max() for p in want))
    tol = n_steps * 9 * LR * 5e-5 * X / EPSILON
    np.testing.assert_allclose(losses, loss64, rtol=0, atol=5e-5 + tol)
    m = r.get_model()
    for got, p in zip((m["U"], m["V"], m["bias"]), want):
        assert np.abs(got - p).max() <= tol + n_steps * 2.0 ** -23 * X
    assert state["step"] == n_steps
    # what the model then answers is of the new factors
    r._host = None
    check(r, users[:5], items[:5], 3, False)
    # a second pass goes on from the state
    start = {k: v.copy() for k, v in r.get_model().items()}
    _, state = r.apply_softmax(users, items, BatchSize=batch, state=state, **HYPER)
    assert state["step"] == 2 * n_steps
    want, _, _ = steps_64(start, users, items, batch, at)
    m = r.get_model()
    for got, p in zip((m["U"], m["V"], m["bias"]), want):
        assert np.abs(got - p).max() <= 3 * tol + n_steps * 2.0 ** -23 * X


def test_apply_softmax_repeats_exactly():
    rs = np.random.default_rng(1)
    users, items = rs.integers(0, 70, 500), rs.integers(0, 133, 500)
    out = []
    for _ in range(2):
        r = model(mml.BPRMF)
        fixed(r)
        r.apply_softmax(users, items, BatchSize=128, **HYPER)
        out.append({k: v.copy() for k, v in r.get_model().items()})
    for k in out[0]:
        assert np.array_equal(out[0][k], out[1][k])


def fixed(r):
    """A fixed model in place of the drawn one."""
    rs = np.random.default_rng(9)
    m = r.get_model()
    new = [rs.normal(0, 0.3, m[k].shape).astype(np.float32) for k in ("U", "V", "bias")]
    N.check(N.lib().mml_bpr_set_model(r._h, *(N.ptr(x, N._f32p) for x in new)))
    r._host = None


def test_apply_softmax_8_bits_and_none():
    r = model(mml.BPRMF)
    before = {k: v.copy() for k, v in r.get_model().items()}
    losses, state = r.apply_softmax([], [], StateBits=8)
    assert losses.shape == (0,) and state["step"] == 0 and "m_scale" in state
    for k, v in r.get_model().items():
        assert np.array_equal(v, before[k])
    losses, state = r.apply_softmax([1, 1], [2, 3], StateBits=8, state=state)
    assert state["step"] == 1 and np.isfinite(losses).all()
    assert not np.array_equal(r.get_model()["U"], before["U"])


@pytest.mark.parametrize("users,items,kw,text", [
    ([70], [0], {}, "beyond"), ([-1], [0], {}, "beyond"), ([0], [133], {}, "beyond"),
    ([0], [-1], {}, "beyond"), ([0, 1], [0], {}, "one length"), ([0], [0], dict(BatchSize=0), "BatchSize"),
    ([0], [0], dict(StateBits=16), "StateBits")])
def test_apply_softmax_refusals(users, items, kw, text):
    r = model(mml.BPRMF)
    before = {k: v.copy() for k, v in r.get_model().items()}
    with pytest.raises(ValueError, match=text):
        r.apply_softmax(users, items, **kw)
    r._host = None
    for k, v in r.get_model().items():
        assert np.array_equal(v, before[k])
