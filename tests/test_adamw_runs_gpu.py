"""AdamW's 8-bit moments over long runs."""
import numpy as np
import pytest
import torch

from mymedialite_amd import AdamW

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24
HYPER = dict(LearnRate=1e-3, Beta1=0.9, Beta2=0.999, Epsilon=1e-8, WeightDecay=0.0)
SIZES = [1024, 1324, 7]  # a whole chunk, one with a rest behind it, less than a block


def finite(opt):
    return all(torch.isfinite(x.float()).all() for n in opt._names for x in getattr(opt, n))


def test_moments_decay_to_nothing():
    """One gradient, then 1,200 steps of zeros: the first moment's scale runs through all of f32's small
    numbers (0.9^1200 = 1e-55) and neither it nor a parameter ever stops being finite.

    Tolerance: every value's m and root are the same multiples of its gradient, so they keep their ratio
    to their block's largest, and their codes, all the way: m and the root are off by a code's half
    spacing, 2^-4, from the first step on, and the steps after it by (1 + 2^-4) / (1 - 2^-4) = 1.134."""
    rs = np.random.default_rng(0)
    ps = [torch.tensor(rs.normal(0, 1, n), dtype=torch.float32, device="cuda") for n in SIZES]
    start = [p.double().clone() for p in ps]
    gs = [torch.tensor(rs.choice([-1.0, 1.0], n) * rs.uniform(0.5, 1.0, n), dtype=torch.float32,
                       device="cuda") for n in SIZES]
    zero = [torch.zeros_like(g) for g in gs]
    opt = AdamW(ps, StateBits=8, **HYPER)
    opt.step(gs)
    for i in range(1200):
        opt.step(zero)
        if i % 50 == 49 or 700 < i < 900:
            assert finite(opt) and all(torch.isfinite(p).all() for p in ps), i
    b1, b2, m, v, move = 0.9, 0.999, 0.1, 0.001, 0.0
    for t in range(1, 1202):  # of a gradient of 1, which the others' ratios are too
        move += m / (1 - b1 ** t) / np.sqrt(v / (1 - b2 ** t)) * HYPER["LearnRate"]
        m, v = b1 * m, b2 * v
    for p, s, g in zip(ps, start, gs):
        np.testing.assert_allclose(((s - p.double()) * g.sign()).cpu().numpy(), move, rtol=0.134)


@pytest.mark.parametrize("largest", [1e-36, 3e-39, 1e-42, 8e-43, 2e-45])
def test_first_moments_under_the_smallest_scale(largest):
    """A state whose first moments' scale is subnormal or next to it (as an earlier library left it, or
    zero): steps without a gradient leave finite codes, scales and parameters, and nothing moves: a
    step is lr m / eps <= 1e-3 1e-36 / 1e-8 = 1e-31, under half a unit of a parameter of 1."""
    ps = [torch.ones(n, device="cuda") for n in SIZES]
    blocks = [-(-n // 256) for n in SIZES]
    code = [torch.full((n,), 448.0, device="cuda").to(torch.float8_e4m3fn) for n in SIZES]
    for c in code:
        c.view(torch.uint8)[1::3] = 0xF8  # -256
    state = {"step": 1000, "m": code,
             "m_scale": [torch.full((b,), largest, device="cuda") / 448 for b in blocks],
             "v": [torch.zeros(n, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
                   for n in SIZES],
             "v_scale": [torch.zeros(b, device="cuda") for b in blocks]}
    opt = AdamW(ps, StateBits=8, state=state, **HYPER)
    for _ in range(60):
        opt.step([torch.zeros_like(p) for p in ps])
        assert finite(opt)
    for p in ps:
        assert (p == 1).all()


def spacing(code):
    """of the e4m3 numbers at a code's value (subnormal ones below 2^-6)"""
    a = np.maximum(np.abs(code), 2.0 ** -6)
    return 2.0 ** (np.floor(np.log2(a)) - 3)


def stored(opt, i):
    """(m, sqrt(v)) that the state stands for, in 64 bits"""
    rest = opt.rest[i].cpu().numpy().astype(np.int32)
    out = []
    for q, scale, units, r in ((opt.m[i], opt.m_scale[i], 6, (rest << 29) >> 29),
                               (opt.v[i], opt.v_scale[i], 30, (rest << 24) >> 27)):
        code = q.cpu().double().numpy()
        s = np.repeat(scale.cpu().double().numpy(), 256)[:len(code)]
        assert np.abs(r).max() <= units // 2
        out.append((code + r * spacing(code) / units) * s)
    return out


HALF = np.arange(1324) % 256 < 128
PATTERNS = {  # the gradients' sizes at step t, from t = 1
    "equal": lambda t, rs: np.ones(1324),
    "log-normal": lambda t, rs: np.exp(np.random.default_rng(1).normal(0, 1, 1324)),
    "one in fifty": lambda t, rs: rs.random(1324) < 0.02,
    "rows of 64, one in fifty": lambda t, rs: np.repeat(rs.random(21) < 0.02, 64)[:1324] * 1.0
    if t > 1 else np.ones(1324),
    "half falls": lambda t, rs: np.where(HALF & (t > 500), 0.1, 1.0),
    "half rises": lambda t, rs: np.where(HALF & (t > 500), 10.0, 1.0),
    "half stops": lambda t, rs: np.where(HALF & (t > 1500), 0.0, 1.0),
}


@pytest.mark.parametrize("steady", [False, True], ids=["noise", "steady"])
@pytest.mark.parametrize("name", PATTERNS)
def test_moments_follow_their_definition(name, steady):
    """3,000 steps against the recurrences in 64 bits (the blocks' values side by side, a whole chunk
    and a partial one): codes alone are off by factors of 2 to 9 in some of these, since a step's
    change is lost where it is below half a spacing.

    Tolerance.  A root is rounded once a step to a unit, 1/30 of a spacing (at most 2^-3 of the value):
    an error under a unit, h <= 2^-3 / 30, of zero mean, with a variance of h^2 / 4 at most (a value's
    place u between two units: u (1 - u) h^2).  A root's error shrinks by beta2 a step while the root
    stays, so the sum's variance is under h^2 / 4 / (2 (1 - beta2)) = 125 h^2; a root without gradients
    shrinks along with it, so its relative errors add up, 1,500 h^2 / 4 more: 22.4 h = 9.4 % as a
    deviation.  Where the errors are spread as a sum of many, 5 % are beyond two of it: a tenth are
    allowed, and none beyond six.  A first moment: units of 2^-3 / 6 of the value or of 2^-9 / 6 of the scale below, whose
    values reach 448, a variance of h^2 / 4 / (1 - 0.81), so 2.4 % of the largest |m| over the last 20
    steps, of its block for the smallest; six times that."""
    rs = np.random.default_rng(5)
    n = 1324
    opt = AdamW([torch.zeros(n, device="cuda")], StateBits=8, **HYPER)
    m, v, recent = np.zeros(n), np.zeros(n), np.zeros(n)
    sign = rs.choice([-1.0, 1.0], n)
    for t in range(1, 3001):
        g = (PATTERNS[name](t, rs) * (sign if steady else rs.normal(0, 1, n))).astype(np.float32)
        opt.step([torch.tensor(g, device="cuda")])
        m = 0.9 * m + 0.1 * g
        v = 0.999 * v + 0.001 * g.astype(np.float64) ** 2
        recent = np.maximum(0.9 ** 0.5 * recent, np.abs(m))
    got_m, got_root = stored(opt, 0)
    ratio = got_root[v > 0] / np.sqrt(v[v > 0])
    sigma = 0.094
    assert abs(np.median(ratio) - 1) < 0.02, np.median(ratio)
    assert (np.abs(ratio - 1) <= 6 * sigma).all(), (ratio.min(), ratio.max())
    assert (np.abs(ratio - 1) <= 2 * sigma).mean() >= 0.9
    assert (got_root[v == 0] == 0).all()
    block = np.repeat([recent[b:b + 256].max() for b in range(0, n, 256)], 256)[:n]
    assert (np.abs(got_m - m) <= 6 * 0.024 * recent + 2.0 ** -9 / 448 * block).all()


@pytest.mark.parametrize("at", [0, 1])
def test_steps_repeat_bit_for_bit(at):
    """Two runs, one of them resumed from its state and one of them captured, and one whose tensors
    begin at any byte: the same bits in every tensor of the state."""
    rs = np.random.default_rng(6)
    n = 3000
    gs = [torch.tensor(rs.normal(0, 1, n), dtype=torch.float32, device="cuda") for _ in range(12)]
    buf = torch.zeros(n + 8, device="cuda")
    a = AdamW([torch.zeros(n, device="cuda")], StateBits=8, **HYPER)
    if at:  # a state at odd bytes: the path without vectors
        u8 = lambda: torch.zeros(n + 8, dtype=torch.uint8, device="cuda")[at:at + n]
        blocks = -(-n // 256)
        state = {"step": 0, "rest": [u8()], "m": [u8().view(torch.float8_e4m3fn)],
                 "v": [u8().view(torch.float8_e4m3fn)],
                 "m_scale": [torch.zeros(blocks, device="cuda")],
                 "v_scale": [torch.zeros(blocks, device="cuda")]}
        b = AdamW([buf[at:at + n]], StateBits=8, state=state, **HYPER)
    else:
        b = AdamW([buf[at:at + n]], StateBits=8, **HYPER)
    for g in gs[:6]:
        a.step([g])
        b.step([g])
    b = AdamW(b.params, StateBits=8, state=b.state(), **HYPER)
    g = gs[0].clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.step([g])
    for x in gs[6:]:
        a.step([x])
        g.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert a.state()["step"] == b.state()["step"]
    assert torch.equal(a.params[0], b.params[0]) and (a.rest[0] != 0).any()
    for name in ("m", "v", "m_scale", "v_scale", "rest"):
        x, y = getattr(a, name)[0], getattr(b, name)[0]
        assert torch.equal(x.view(torch.uint8), y.contiguous().view(torch.uint8)), name


def test_states_without_rests_and_refusals():
    """A state of codes and scales alone goes on as one, whatever the step: each step is that of the
    definition from the codes, to nearest (tolerance: codes whose quotient lies within 16 EPS of the
    middle of two may be either).  Rests of another type or size are refused."""
    rs = np.random.default_rng(9)
    n = 1324
    p = torch.ones(n, device="cuda")
    a = AdamW([p], StateBits=8, **HYPER)
    gs = [torch.tensor(rs.normal(0, 1, n), dtype=torch.float32, device="cuda") for _ in range(9)]
    for g in gs[:6]:
        a.step([g])
    s = {k: v if k == "step" else [x.clone() for x in v] for k, v in a.state().items() if k != "rest"}
    b = AdamW([p], StateBits=8, state=s, **HYPER)
    assert "rest" not in b.state() and not hasattr(b, "rest")
    for t, g in enumerate(gs[6:], 7):
        m, root = (np.repeat(scale[0].cpu().double().numpy(), 256)[:n] * q[0].cpu().double().numpy()
                   for q, scale in ((b.m, b.m_scale), (b.v, b.v_scale)))
        b.step([g])
        g = g.cpu().double().numpy()
        m, v = 0.9 * m + 0.1 * g, 0.999 * root ** 2 + 0.001 * g * g
        for q, scale, x in ((b.m, b.m_scale, m), (b.v, b.v_scale, np.sqrt(v))):
            block = np.array([np.abs(x[i:i + 256]).max() / 448 for i in range(0, n, 256)])
            np.testing.assert_allclose(scale[0].cpu().double().numpy(), block, rtol=16 * EPS)
            want = x / np.repeat(block, 256)[:n]
            slack = 16 * EPS * (np.abs(want) + (np.abs(g) / np.repeat(block, 256)[:n] if x is m else 0))
            e4m3 = lambda y: torch.tensor(y).float().to(torch.float8_e4m3fn).double().numpy()
            lo, hi, got = e4m3(want - slack), e4m3(want + slack), q[0].cpu().double().numpy()
            assert ((got >= np.minimum(lo, hi)) & (got <= np.maximum(lo, hi))).all(), t
    short = torch.ones(300, device="cuda")
    c = AdamW([short], StateBits=8, **HYPER)
    s = c.state()
    for bad in (torch.zeros(300, device="cuda"), torch.zeros(299, dtype=torch.uint8, device="cuda")):
        with pytest.raises(ValueError, match="state's rest must"):
            AdamW([short], StateBits=8, state=dict(s, rest=[bad]), **HYPER)
    with pytest.raises(ValueError, match="state has 1 m, expected 2"):
        AdamW([short, short.clone()], StateBits=8, state=s, **HYPER)


def test_overlapping_states_and_negative_steps_are_refused():
    p = torch.ones(300, device="cuda")
    x, y = torch.zeros(300, device="cuda"), torch.zeros(400, device="cuda")
    for state in ({"m": [x], "v": [x]}, {"m": [y[:300]], "v": [y[100:]]}, {"m": [p], "v": [x]}):
        with pytest.raises(ValueError, match="overlap"):
            AdamW([p], state=dict(state, step=1))
    with pytest.raises(ValueError, match="negative"):
        AdamW([p], state={"m": [x], "v": [y[:300]], "step": -1})
    o = AdamW([p], state={"m": [x], "v": [y[:300]], "step": 1})
    with pytest.raises(ValueError, match="gradient 0 is not a tensor"):
        o.step([None])
    assert o.state()["step"] == 1


@pytest.mark.parametrize("bits", [32, 8])
def test_not_finite_gradients_in_whole_chunks(bits):
    """As test_adamw_gpu.py's, in the chunks that are read four values at a time: a NaN or infinite
    gradient spoils its own value and no neighbour's."""
    rs = np.random.default_rng(7)
    n = 9000
    gs = [torch.tensor(rs.normal(0, 1, n), dtype=torch.float32, device="cuda") for _ in range(8)]
    bad = torch.zeros(n, dtype=torch.bool, device="cuda")
    bad[[3, 300, 2047, 2048, 4444, n - 1]] = True
    ps = [torch.ones(n, device="cuda") for _ in range(2)]
    a, b = (AdamW([p], StateBits=bits, **HYPER) for p in ps)
    for t, g in enumerate(gs):
        g[bad] = 0.0
        spoiled = g.clone()
        if t == 5:
            spoiled[3], spoiled[300], spoiled[2047] = float("nan"), float("inf"), -float("inf")
            spoiled[2048], spoiled[4444], spoiled[n - 1] = float("inf"), float("nan"), float("inf")
        a.step([spoiled])
        b.step([g])
    assert torch.equal(ps[0][~bad], ps[1][~bad]) and torch.isnan(ps[0][bad]).all()
    for name in a._names:
        x, y = getattr(a, name)[0], getattr(b, name)[0]
        if name.endswith("scale"):
            assert torch.equal(x, y)
        else:
            assert torch.equal(x.float()[~bad], y.float()[~bad])


@pytest.mark.parametrize("bits", [32, 8])
def test_more_chunks_than_blocks(bits):
    """A tensor that the grid's blocks walk in several turns (2,048 blocks of 1,024 or 2,048 values): each
    value as in a tensor of its block alone."""
    n, part = 9_000_011, 8_399_872  # the part begins at a block of 256 and is behind 4 M values
    g = torch.randn(n, device="cuda", generator=torch.Generator("cuda").manual_seed(3))
    whole, some = torch.ones(n, device="cuda"), torch.ones(n - part, device="cuda")
    a = AdamW([whole], StateBits=bits, **HYPER)
    b = AdamW([some], StateBits=bits, **HYPER)
    for t in range(3):  # (the first steps leave no rests, whose dither goes by place)
        a.step([g * (t + 1)])
        b.step([g[part:] * (t + 1)])
    assert part % 256 == 0 and torch.equal(whole[part:], some)
    assert torch.equal(a.m[0][part:].view(torch.uint8), b.m[0].view(torch.uint8))
    assert ((whole != 1) | (g.abs() < 1e-7)).all()  # (randn gives a few zeros)
