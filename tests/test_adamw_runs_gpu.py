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
