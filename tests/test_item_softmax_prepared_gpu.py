"""The softmax over the catalogue on its path with preparation (more than one tile of 32 users and
user tiles x item tiles x steps of 16 factors above 16,384), where most small cases of
test_item_softmax_gpu.py do not come: every width and type of the forward kernel, and the cases where
masks, values and sizes go wrong.  Definitions and tolerances are that file's."""
import numpy as np
import pytest
import torch

from test_item_softmax_gpu import (BF16, F16, F32, backward, check_backward, check_forward, forward,
                                   make, reference, to_gpu, tol_score)

pytestmark = pytest.mark.gpu

TYPES = pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])


def tiles(rows, n_items, k):
    kt = next(x for x in (1, 2, 4, 6, 8, 12, 16) if 16 * x >= k)
    return -(-rows // 32) * (-(-n_items // 256) * 8) * kt


@TYPES
@pytest.mark.parametrize("rows,n_items,k", [(545, 31_000, 16), (545, 31_000, 3), (290, 30_001, 32),
                                            (97, 33_001, 64), (65, 30_011, 96), (65, 22_001, 128),
                                            (33, 22_001, 192), (33, 17_001, 256), (64, 17_000, 255)])
def test_every_width(rows, n_items, k, dtype):
    assert tiles(rows, n_items, k) > 16384
    d = make(rows, n_items, k, dtype, seed=k, n_users=rows + 5, seen=30)
    g_lp, g_ent = torch.full((rows,), -1.0 / rows), torch.full((rows,), 0.1 / rows)
    c = to_gpu(d)
    r = forward(c, 10)
    ref = reference(d, 10, g_lp, g_ent)
    check_forward(d, r, 10, ref)
    check_backward(d, backward(c, r, g_lp, g_ent), ref)
    plain = dict(d, b=None, ex=None)
    check_forward(plain, forward(to_gpu(plain)))


ROWS, ITEMS, K = 600, 30_001, 12


@TYPES
def test_masks_and_empty_rows(dtype):
    d = make(ROWS, ITEMS, K, dtype, seed=4, n_users=ROWS)
    assert tiles(ROWS, ITEMS, K) > 16384
    d["b"][3] = -np.inf
    d["b"][50] = torch.finfo(F32).min
    d["b"][ITEMS - 1] = -1e30
    d["V"][3] = float("nan")
    d["V"][50, 2] = float("inf")
    off = np.zeros(ROWS + 1, np.int64)
    off[6:] = 2 * ITEMS      # user 5: every item, twice, unsorted
    off[590:] = 2 * ITEMS + 4  # user 589: two items and two ids outside
    ids = np.concatenate([np.arange(ITEMS)[::-1], np.arange(ITEMS), [4, -1, ITEMS, 9]])
    d["ex"] = (torch.tensor(off), torch.tensor(ids, dtype=torch.int32))
    d["items"][0] = 3
    d["items"][589] = 9
    d["items"][1], d["items"][2] = -1, ITEMS
    c = to_gpu(d)
    r = forward(c, 4)
    g_lp, g_ent = torch.full((ROWS,), 0.25), torch.full((ROWS,), -0.5)
    ref = reference(d, 4, g_lp, g_ent)
    check_forward(d, r, 4, ref)
    assert r.log_norm[5] == -np.inf and r.entropy[5] == 0 and (r.top_items[5] == -1).all()
    assert r.log_probs[5] == -np.inf and r.log_probs[0] == -np.inf and r.log_probs[589] == -np.inf
    assert r.log_probs[1] == 0 and r.log_probs[2] == 0
    got = backward(c, r, g_lp, g_ent)
    check_backward(d, got, ref)
    assert (got[0][5] == 0).all()
    for i in (3, 50, ITEMS - 1):
        assert (got[1][i] == 0).all() and got[2][i] == 0
    d["b"][:] = -np.inf
    c = to_gpu(d)
    r = forward(c, 2)
    assert (r.log_norm == -np.inf).all() and (r.entropy == 0).all() and (r.top_items == -1).all()
    assert all((g == 0).all() for g in backward(c, r, g_lp, g_ent))


@TYPES
def test_not_finite_values_stay_in_their_rows(dtype):
    d = make(ROWS, ITEMS, K, dtype, seed=6, n_users=ROWS)
    d["users"] = torch.arange(ROWS, dtype=torch.int32)
    clean = reference(d)
    d["U"][10, 3] = float("nan")
    d["U"][ROWS - 1, 0] = float("inf")
    d["users"][4], d["users"][5] = ROWS, -7
    c = to_gpu(d)
    r = forward(c, 3)
    bad = np.zeros(ROWS, bool)
    bad[[10, ROWS - 1, 4, 5]] = True
    for x in (r.log_norm, r.entropy, r.log_probs):
        np.testing.assert_array_equal(np.isnan(x.cpu().numpy()), bad)
    assert (r.top_items.cpu().numpy()[bad] == -1).all()
    tol = tol_score(d, clean)
    assert (np.abs(r.log_norm.cpu().numpy() - clean["lse"])[~bad] <= tol[~bad]).all()

    d = make(ROWS, ITEMS, K, dtype, seed=6, n_users=ROWS)
    d["users"] = torch.arange(ROWS, dtype=torch.int32)
    d["V"][20_007, 1] = float("nan")  # all rows but those that exclude it
    off = np.zeros(ROWS + 1, np.int64)
    off[8:] = 1
    d["ex"] = (torch.tensor(off), torch.tensor([20_007], dtype=torch.int32))
    c = to_gpu(d)
    r = forward(c, 3)
    np.testing.assert_array_equal(np.isnan(r.log_norm.cpu().numpy()), np.arange(ROWS) != 7)
    check = reference(d, 3)
    assert abs(float(r.log_norm[7]) - check["lse"][7]) <= tol_score(d, check)[7]
    np.testing.assert_array_equal(r.top_items[7].cpu().numpy(), check["top"][7])


@TYPES
def test_ties_and_large_scores(dtype):
    d = make(ROWS, ITEMS, K, dtype, seed=8)
    d["b"] = None
    d["U"][1] = 0
    d["V"][100:260] = d["V"][7]
    c = to_gpu(d)
    check_forward(d, forward(c, 120), 120)
    assert (forward(c, 128).top_items[1].cpu() == torch.arange(128)).all()
    d = make(ROWS, ITEMS, K, dtype, seed=10, std=9.0)  # scores of several hundred
    g_lp, g_ent = torch.ones(ROWS), torch.full((ROWS,), 0.1)
    c = to_gpu(d)
    r = forward(c, 3)
    ref = reference(d, 3, g_lp, g_ent)
    assert ref["lse"].max() > 300
    check_forward(d, r, 3, ref)
    # reference() takes a given item whose p is 0 in 64 bits for an excluded one and leaves its
    # w (1 - p) = w out; log p of -746 and less comes from the scores here
    for x in np.flatnonzero(ref["lp"] < -745):
        t = int(d["items"][x])
        u, v = d["U"][x].double().numpy(), d["V"][t].double().numpy()
        if np.exp(ref["lp"][x]) == 0:
            ref["gu"][x] += v
            ref["gv"][t] += u
            ref["gb"][t] += 1
            for name, y in (("magu", x), ("magv", t), ("magb", t)):
                ref[name][y] += {"magu": np.abs(v), "magv": np.abs(u), "magb": 1}[name]
            ref["mag"][x, t] += 1
            # and the row's own -w p, which it left out along with it
            p = np.exp(d["V"].double().numpy() @ u + d["b"].double().numpy() - ref["lse"][x])
            ref["gu"][x] -= p @ d["V"].double().numpy()
            ref["gv"] -= p[:, None] * u
            ref["gb"] -= p
            ref["mag"][x] += p
            ref["magu"][x] += p @ np.abs(d["V"].double().numpy())
            ref["magv"] += p[:, None] * np.abs(u)
            ref["magb"] += p
    check_backward(d, backward(c, r, g_lp, g_ent), ref)


@TYPES
def test_strides_streams_and_graphs(dtype):
    """Padded rows, an unaligned base, a transposed matrix; two side streams; two graphs in turn: the same
    numbers bit for bit."""
    d = make(ROWS, ITEMS, K, dtype, seed=11, n_users=ROWS + 3, seen=5)
    c = to_gpu(d)
    g = torch.full((ROWS,), 0.5, device="cuda")
    want = forward(c, 4)
    gw = backward(c, want, g, None)

    def wide(x, pad, at):
        y = torch.full((x.shape[0], x.shape[1] + pad), 7.0, dtype=x.dtype, device="cuda")
        y[:, at:at + x.shape[1]] = x
        return y[:, at:at + x.shape[1]]

    for e in (dict(c, U=wide(c["U"], 4, 0), V=wide(c["V"], 20, 4)),
              dict(c, U=wide(c["U"], 3, 1), V=wide(c["V"], 5, 3)),
              dict(c, U=c["U"].t().contiguous().t(), V=c["V"].t().contiguous().t())):
        got = forward(e, 4)
        for a, b in zip((*got, *backward(e, got, g, None)), (*want, *gw)):
            assert torch.equal(a, b)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for s in streams * 2:
        with torch.cuda.stream(s):
            e = dict(c, U=c["U"] * 1.0)
            r = forward(e, 4)
            got.append((*r, *backward(e, r, g, None)))
    torch.cuda.synchronize()
    for x in got:
        assert all(torch.equal(a, b) for a, b in zip(x, (*want, *gw)))

    def both(e):
        r = forward(e, 4)
        return (*r, *backward(e, r, g, g))

    graphs = []
    for _ in range(2):
        e = dict(c, U=c["U"].clone())
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = both(e)
        graphs.append((gr, e, out))
    for i in range(4):
        gr, e, out = graphs[i % 2]
        e["U"].copy_(c["U"] * (1.0 + 0.1 * i))
        gr.replay()
        again = both(e)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, again))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_large_derivatives(dtype):
    """dL/dH of 1e8 beside excluded items (the largest that is promised): nothing overflows.  (Results
    in f16 end at 65504.)"""
    d = make(100, 2000, 20, dtype, seed=12, seen=50)
    d["b"][::7] = -np.inf
    c = to_gpu(d)
    g_ent = torch.full((100,), 1e8)
    check_backward(d, backward(c, forward(c), None, g_ent), reference(d, 0, None, g_ent))
