"""AdamW with moments in 32 and in 8 bits against its definition in 64 bits.

Tolerances (f32 parameters, EPS = 2^-24 a rounding).  m: the product, the fma and the coefficient
round once each, 4 EPS (|m| + |g|) is above that; v likewise 4 EPS v.  The step lr m / (root + eps)
takes the root, three coefficients, an fma and a division: 16 EPS of its size, and m's error at the
step's rate, 4 EPS (|m before| + |g|) lr / (root + eps) (m may cancel, so it is not a share of the
step).  The parameter rounds three times: its decay factor and the product, 2 EPS |p before|, and the
final sum, EPS |p after|.  A half-precision parameter is off by half a step more (finfo.eps / 2).
8 bits: a code is the nearest e4m3 to value / scale.  The value is known to 8 EPS, so the code may be
the neighbour where value / scale lies within 16 EPS of the middle of two codes; everywhere else it
is equal.
"""
import numpy as np
import pytest
import torch

from mymedialite_amd import AdamW
from mymedialite_amd import _native as N

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
E4M3 = torch.float8_e4m3fn
EPS = 2.0 ** -24
B = 256


def blocks(x):
    x = np.asarray(x, np.float64).reshape(-1)
    y = np.zeros(-(-len(x) // B) * B)
    y[:len(x)] = x
    return y.reshape(-1, B)


def values(q, scale):
    return (blocks(q.cpu().double().numpy()) * scale.cpu().double().numpy()[:, None]).reshape(-1)[
        :q.numel()]


def e4m3(x):
    return torch.tensor(x).float().to(E4M3).double().numpy()


def quantise(x, root):
    b = blocks(x)
    scale = np.abs(b).max(1) / 448.0
    q = b / np.where(scale > 0, scale, 1.0)[:, None]
    if root:
        q = np.where((q > 0) & (q < 2.0 ** -9), 2.0 ** -9, q)
    return q.reshape(-1)[:len(x)], scale


class Reference:
    """The definition in 64 bits for one tensor, from the same starting values."""

    def __init__(self, p, h, bits, m, v):
        self.p, self.h, self.bits = p.double().cpu().numpy().reshape(-1), h, bits
        self.m, self.v = m, v

    def step(self, g, t):
        h = self.h
        g = g.double().cpu().numpy().reshape(-1)
        self.m0 = np.abs(self.m)
        self.m = h["Beta1"] * self.m + (1 - h["Beta1"]) * g
        self.v = h["Beta2"] * self.v + (1 - h["Beta2"]) * g * g
        self.root = np.sqrt(self.v)
        self.rate = h["LearnRate"] / (1 - h["Beta1"] ** t) / (
            self.root / np.sqrt(1 - h["Beta2"] ** t) + h["Epsilon"])
        self.move = self.rate * self.m
        self.p = self.p * (1 - h["LearnRate"] * h["WeightDecay"]) - self.move


HYPER = dict(LearnRate=2e-3, Beta1=0.9, Beta2=0.999, Epsilon=1e-8, WeightDecay=0.05)
SIZES = [(1,), (3,), (255,), (256,), (257,), (33, 7), (2047,), (2049,), (943, 10), (1682,), (4, 5, 600)]


def tensors(sizes, dtype, gdtype, seed=0):
    rs = np.random.default_rng(seed)
    t = lambda x, d: torch.tensor(x, dtype=F32).to(d).cuda()
    return ([t(rs.normal(0, 0.1, s), dtype) for s in sizes],
            [[t(rs.normal(0, 10.0 ** rs.uniform(-4, 0), s), gdtype) for s in sizes]
             for _ in range(3)])


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype,gdtype", [(F32, F32), (BF16, BF16), (F16, F16), (BF16, F32),
                                          (F32, F16)], ids=str)
def test_steps(bits, dtype, gdtype):
    """Three steps from zero moments; each step is checked from the state that it began with."""
    ps, gs = tensors(SIZES, dtype, gdtype)
    opt = AdamW(ps, StateBits=bits, **HYPER)
    half = 0.0 if dtype == F32 else torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == F16 else 0.0
    for t, g in enumerate(gs, 1):
        refs = []
        for i, p in enumerate(ps):
            if bits == 32:
                m, v = (x[i].cpu().double().numpy().reshape(-1) for x in (opt.m, opt.v))
            else:
                m = values(opt.m[i], opt.m_scale[i])
                v = values(opt.v[i], opt.v_scale[i]) ** 2
            refs.append(Reference(p, HYPER, bits, m, v))
        old = [p.double().cpu().numpy().reshape(-1) for p in ps]
        opt.step(g)
        for i, (p, r) in enumerate(zip(ps, refs)):
            r.step(g[i], t)
            got = p.double().cpu().numpy().reshape(-1)
            gabs = np.abs(g[i].double().cpu().numpy().reshape(-1))
            tol = (2 * np.abs(old[i]) + np.abs(r.p) + 16 * np.abs(r.move)
                   + 4 * (r.m0 + gabs) * r.rate) * EPS + half * np.abs(r.p) + tiny
            assert (np.abs(got - r.p) <= tol).all(), (i, np.max(np.abs(got - r.p) / tol))
            tm, tv = 4 * EPS * (r.m0 + gabs), 4 * EPS * r.v
            if bits == 32:
                assert (np.abs(opt.m[i].cpu().double().numpy().reshape(-1) - r.m) <= tm).all()
                assert (np.abs(opt.v[i].cpu().double().numpy().reshape(-1) - r.v) <= tv).all()
                continue
            for q, scale, x, root in ((opt.m[i], opt.m_scale[i], r.m, False),
                                      (opt.v[i], opt.v_scale[i], r.root, True)):
                want, ws = quantise(x, root)
                np.testing.assert_allclose(scale.cpu().double().numpy(), ws, rtol=16 * EPS)
                got = q.cpu().double().numpy().reshape(-1)
                # where a change of 16 EPS of the largest of m and g changes the code, either is right
                slack = 16 * EPS * np.abs(want) if root else 16 * EPS * (
                    (r.m0 + gabs) / np.maximum(ws.repeat(B)[:len(want)], 1e-300))
                lo, hi = e4m3(want - slack), e4m3(want + slack)
                assert ((got >= np.minimum(lo, hi)) & (got <= np.maximum(lo, hi))).all()
                if root:
                    assert ((got > 0) == (x > 0)).all()
    assert opt.state()["step"] == 3


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_and_none(bits):
    """More tensors than one launch takes, empty ones among them: as one by one, bit for bit."""
    sizes = [(1 + 37 * i % 700,) for i in range(95)]
    sizes[5] = sizes[50] = sizes[94] = (0,)
    ps, gs = tensors(sizes, F32, F32, seed=3)
    one = [p.clone() for p in ps]
    a = AdamW(ps, StateBits=bits, **HYPER)
    b = [AdamW([p], StateBits=bits, **HYPER) for p in one]
    for g in gs:
        a.step(g)
        for o, x in zip(b, g):
            o.step([x])
    for x, y in zip(ps, one):
        assert torch.equal(x, y)
    assert a.state()["step"] == 3 and b[5].state()["step"] == 3
    empty = AdamW([], StateBits=bits)
    empty.step([])
    assert empty.state()["step"] == 1


@pytest.mark.parametrize("bits", [32, 8])
def test_resume_is_the_same_run(bits):
    ps, gs = tensors([(300, 9), (77,)], F32, F32, seed=4)
    other = [p.clone() for p in ps]
    a = AdamW(ps, StateBits=bits, **HYPER)
    b = AdamW(other, StateBits=bits, **HYPER)
    for g in gs:
        a.step(g)
    b.step(gs[0])
    s = {n: (x if n == "step" else [y.clone() for y in x]) for n, x in b.state().items()}
    c = AdamW(other, StateBits=bits, state=s, **HYPER)
    c.step(gs[1])
    c.step(gs[2])
    for x, y in zip(ps, other):
        assert torch.equal(x, y)
    assert c.state()["step"] == 3


@pytest.mark.parametrize("bits", [32, 8])
def test_not_finite_gradients_stay_put(bits):
    """A NaN or infinite gradient spoils its own value and no neighbour of its block."""
    ps, gs = tensors([(600,)], F32, F32, seed=5)
    clean = [p.clone() for p in ps]
    a, b = AdamW(ps, StateBits=bits, **HYPER), AdamW(clean, StateBits=bits, **HYPER)
    bad = torch.zeros(600, dtype=torch.bool, device="cuda")
    bad[[3, 300, 599]] = True
    # the largest values of their blocks stay elsewhere, so that the scales are the same
    for g in gs:
        g[0][bad] = 0.0
    spoiled = gs[0][0].clone()
    spoiled[3], spoiled[300], spoiled[599] = float("nan"), float("inf"), -float("inf")
    a.step([spoiled])
    b.step([gs[0][0]])
    a.step([gs[1][0]])
    b.step([gs[1][0]])
    assert torch.equal(ps[0][~bad], clean[0][~bad])
    assert torch.isnan(ps[0][bad]).all()
    for x, y in ((a.m[0], b.m[0]), (a.v[0], b.v[0])):
        assert torch.equal(x.float()[~bad], y.float()[~bad])


def test_zero_gradients_and_zero_blocks():
    """With zero moments and gradients only the decay moves a parameter, in both forms."""
    for bits in (32, 8):
        p = torch.full((513,), 2.0, device="cuda")
        o = AdamW([p], StateBits=bits, **HYPER)
        o.step([torch.zeros(513, device="cuda")])
        want = np.float32(2.0) * np.float32(1 - HYPER["LearnRate"] * HYPER["WeightDecay"])
        assert (p == float(want)).all()
        assert (o.m[0].float() == 0).all() and (o.v[0].float() == 0).all()


def test_strided_gradients_and_streams():
    ps, gs = tensors([(40, 30)], F32, F32, seed=6)
    want = ps[0].clone()
    AdamW([want], **HYPER).step(gs[0])
    got = ps[0].clone()
    AdamW([got], **HYPER).step([gs[0][0].t().contiguous().t()])
    assert torch.equal(got, want)
    side = torch.cuda.Stream()
    got = ps[0].clone()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        o = AdamW([got], **HYPER)
        o.step([gs[0][0] * 1.0])
    side.synchronize()
    assert torch.equal(got, want)
    # views that begin at any element of a buffer
    buf = torch.zeros(1300, device="cuda")
    buf[1:1201] = ps[0].reshape(-1)
    g = torch.zeros(1203, device="cuda")
    g[3:] = gs[0][0].reshape(-1)
    for bits in (32, 8):
        v = buf.clone()
        AdamW([v[1:1201]], StateBits=bits, **HYPER).step([g[3:]])
        w = ps[0].reshape(-1).clone()
        AdamW([w], StateBits=bits, **HYPER).step([gs[0][0].reshape(-1)])
        assert torch.equal(v[1:1201], w) and v[0] == 0 and (v[1201:] == 0).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_count_on(bits):
    ps, gs = tensors([(500, 12), (77,)], F32, F32, seed=7)
    eager = [p.clone() for p in ps]
    a, b = AdamW(ps, StateBits=bits, **HYPER), AdamW(eager, StateBits=bits, **HYPER)
    g = [x.clone() for x in gs[0]]
    a.step(g)
    b.step(gs[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step(g)
    assert a.state()["step"] == 1  # capturing runs nothing
    for i in range(5):
        for x, y in zip(g, gs[i % 3]):
            x.copy_(y)
        graph.replay()
        b.step(gs[i % 3])
        torch.cuda.synchronize()
        for x, y in zip(ps, eager):
            assert torch.equal(x, y)
    assert a.state()["step"] == b.state()["step"] == 6


def test_refusals():
    p, g = torch.zeros(10, device="cuda"), torch.zeros(10, device="cuda")
    for bad, text in (([p.double()], "must be float32"), ([p.cpu()], "on the GPU"),
                      ([p.view(2, 5).t()], "contiguous"), ([p, p], "twice")):
        with pytest.raises(ValueError, match=text):
            AdamW(bad)
    with pytest.raises(ValueError, match="StateBits"):
        AdamW([p], StateBits=16)
    with pytest.raises(ValueError, match="state has no v"):
        AdamW([p], state={"m": [p]})
    with pytest.raises(ValueError, match="state's m must"):
        AdamW([p], state={"m": [p[:3]], "v": [p]})
    o = AdamW([p])
    for bad, text in (([], "0 gradients"), ([g[:4]], "shape and device"),
                      ([g.cpu()], "shape and device"), ([g.double()], "must be float32")):
        with pytest.raises(ValueError, match=text):
            o.step(bad)
    for name, x in (("LearnRate", -1.0), ("LearnRate", float("nan")), ("Beta1", 1.0),
                    ("Beta2", -0.1), ("Epsilon", float("inf")), ("WeightDecay", -1.0)):
        o = AdamW([p], **{name: x})
        with pytest.raises(N.MMLError):
            o.step([g])
        assert o.state()["step"] == 0


def test_overlapping_and_moved_parameters_are_refused():
    x = torch.zeros(10, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        AdamW([x[:6], x[5:]])
    a, b, none = x[:5], x[5:], torch.zeros(0, device="cuda")
    o = AdamW([a, b, none])
    o.step([torch.ones(5, device="cuda"), torch.ones(5, device="cuda"), none])
    a.data = torch.zeros(5, device="cuda")
    with pytest.raises(ValueError, match="parameter 0 is in other memory"):
        o.step([torch.ones(5, device="cuda"), torch.ones(5, device="cuda"), none])
    assert o.state()["step"] == 1
