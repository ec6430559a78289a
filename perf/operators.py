"""Timed cases of the softmax-over-the-catalogue operators and of the AdamW step.

* ``log_probs``: for a batch of users, the log probability of a given item under the softmax over
  the whole catalogue (score = <U_u, V_i> + b_i, the user's seen items left out), the entropy of
  that distribution and its top items.
* ``grad``: the gradient of a loss on those log probabilities and entropies with respect to the
  users' factors, the items' factors and the item biases.
* ``adamw``: one AdamW step over a model's parameter tensors, moments in 32 or in 8 bits (e4m3,
  one scale per 256 values; the second moment is held as its root).

Factors, biases and moments are synthetic: scores with a spread of about 2 around Zipf(0.8) item
popularity, moments as they are some steps into a training run.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BLOCK = 256      # values per scale of the 8-bit moments
E4M3_MAX = 448.0
E4M3_MIN = 2.0 ** -9  # smallest nonzero e4m3 value


# ------------------------------------------------------------------ the cases
def listed():
    lp = {"op": "log_probs", "dtype": "f32", "seen": 100, "top": 10}
    gr = {"op": "grad", "dtype": "f32", "seen": 0, "entropy": 1}
    ad = {"op": "adamw", "dtype": "f32", "bits": 32, "k": 64}
    return [
        # a recommendation request: one user against a 100 k catalogue
        dict(lp, name="lp_one_user", rows=1, items=100_000, k=64),
        # a handful of users on the ML-100k shape, reference default k = 10
        dict(lp, name="lp_small", rows=37, items=1682, k=10, top=5),
        # held-out evaluation of a batch of users on the 100 k catalogue
        dict(lp, name="lp_eval", rows=4096, items=100_000, k=64),
        # the same on the 1 M catalogue of the k = 128 configuration, factors held in bf16
        dict(lp, name="lp_million", rows=2048, items=1_000_000, k=128, dtype="bf16", top=20),
        # a small training batch on the ML-100k shape
        dict(gr, name="grad_small", rows=200, items=1682, k=10, seen=20),
        # a training batch on the 100 k catalogue, entropy term included
        dict(gr, name="grad_batch", rows=2048, items=100_000, k=64),
        # half-precision factors, odd sizes, seen items left out
        dict(gr, name="grad_f16_odd", rows=1001, items=30_011, k=100, dtype="f16", seen=50),
        # the widest factors the models take, bf16, 500 k items
        dict(gr, name="grad_k256", rows=1024, items=500_000, k=256, dtype="bf16", entropy=0),
        # a BiasedMF model of the ML-100k shape: four small tensors, latency
        dict(ad, name="adam_small", users=943, items=1682, k=10),
        # 1 M x 100 k at k = 64, moments in 32 bits
        dict(ad, name="adam_32", users=1_000_000, items=100_000),
        # the same with moments in 8 bits
        dict(ad, name="adam_8", users=1_000_000, items=100_000, bits=8),
        # bf16 factors, odd k, moments in 8 bits
        dict(ad, name="adam_8_bf16", users=200_003, items=30_011, k=33, bits=8, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["log_probs", "grad", "adamw"])
    dtype = rng.choice(["f32", "f32", "bf16", "f16"])
    if op == "adamw":
        return {"op": op, "dtype": dtype, "bits": rng.choice([8, 32]), "k": _log(rng, 4, 256),
                "users": _log(rng, 100, 250_000), "items": _log(rng, 50, 100_000)}
    k, items = _log(rng, 4, 256), _log(rng, 200, 1_000_000)
    most = 1.2e11 if op == "log_probs" else 2.5e10  # rows * items * k
    rows = min(_log(rng, 1, 4096), max(1, int(most / (items * k))))
    if op == "log_probs":
        return {"op": op, "dtype": dtype, "rows": rows, "items": items, "k": k,
                "seen": rng.choice([0, 30, 150]), "top": rng.choice([0, 1, 10, 50, 100])}
    return {"op": op, "dtype": dtype, "rows": rows, "items": items, "k": k,
            "seen": rng.choice([0, 0, 30]), "entropy": rng.choice([0, 1])}


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "adamw":
        n = (case["users"] + case["items"]) * (case["k"] + 1)
        moments = 4 * 4 if case["bits"] == 32 else 4 * 1 + 4 * 4 / BLOCK
        return {"bytes": n * (3 * size + moments), "flops": 15 * n}
    R, N, k = case["rows"], case["items"], case["k"]
    factors = (R + N) * k * size + 4 * N
    if case["op"] == "log_probs":
        return {"bytes": factors + 4 * R * case["seen"] + R * (16 + 8 * case["top"]),
                "flops": 2 * R * N * k}
    return {"bytes": 2 * factors + 4 * R * case["seen"] + R * 20, "flops": 6 * R * N * k}


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 7919 + 17)
    return _prepare_adamw(case, g) if case["op"] == "adamw" else _prepare_softmax(case, g)


def _normal(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _prepare_softmax(case, g):
    R, N, k = case["rows"], case["items"], case["k"]
    dtype = DTYPES[case["dtype"]]
    n_users = 2 * R + 3
    std = math.sqrt(2.0 / math.sqrt(k))
    s = {"case": case, "U": (_normal(g, n_users, k) * std).to(dtype),
         "V": (_normal(g, N, k) * std).to(dtype)}
    rank = torch.randperm(N, device="cuda", generator=g).float() + 1
    s["bias"] = -0.8 * torch.log(rank) + 0.1 * _normal(g, N)
    s["users"] = torch.randint(0, n_users, (R,), device="cuda", generator=g, dtype=torch.int32)
    s["items"] = torch.randint(0, N, (R,), device="cuda", generator=g, dtype=torch.int32)
    if R > 8:
        s["items"][::97] = -1  # rows padded to the batch
    s["seen"] = None
    if case["seen"]:
        count = torch.randint(0, 2 * case["seen"] + 1, (n_users,), device="cuda", generator=g)
        off = torch.zeros(n_users + 1, dtype=torch.int64, device="cuda")
        off[1:] = torch.cumsum(count, 0)
        n = int(off[-1])
        who = torch.repeat_interleave(torch.arange(n_users, device="cuda"), count)
        key = torch.sort(who * N + torch.randint(0, N, (n,), device="cuda", generator=g)).values
        s["seen"] = (off, (key % N).int())
    if case["op"] == "grad":
        w = torch.full((R,), -1.0 / R, device="cuda")  # the mean negative log likelihood
        s["g_log_probs"] = w * (0.5 + torch.rand(R, device="cuda", generator=g))
        s["g_entropy"] = 0.1 * w if case["entropy"] else None
        S = _scores(s, torch.float64)
        lse = torch.logsumexp(S, 1)
        S -= lse[:, None]
        P = torch.exp(S)
        S.clamp_(min=-1e300)
        s["log_norm"] = lse.float()
        s["entropy"] = -P.mul_(S).sum(1).float()
    return s


def _prepare_adamw(case, g):
    dtype = DTYPES[case["dtype"]]
    shapes = [(case["users"], case["k"]), (case["items"], case["k"]), (case["users"],),
              (case["items"],)]
    p = [(_normal(g, *x) * 0.1).to(dtype) for x in shapes]
    grads = [(_normal(g, *x) * 1e-3).to(dtype) for x in shapes]
    m = [_normal(g, *x) * 3e-4 for x in shapes]
    v = [(_normal(g, *x) * 1e-3).square() + 1e-10 for x in shapes]
    s = {"case": case, "p": p, "g": grads, "step": 100,
         "hyper": dict(LearnRate=1e-3, Beta1=0.9, Beta2=0.999, Epsilon=1e-8, WeightDecay=0.01)}
    if case["bits"] == 32:
        s["m"], s["v"] = m, v
    else:
        mq = [_quantise(x, False) for x in m]
        vq = [_quantise(torch.sqrt(x), True) for x in v]
        s["m"], s["m_scale"] = [x[0] for x in mq], [x[1] for x in mq]
        s["v"], s["v_scale"] = [x[0] for x in vq], [x[1] for x in vq]
    if own:  # the optimizer that a program keeps between its steps
        from mymedialite_amd import AdamW
        state = {n: s[n] for n in ("step", "m", "v", "m_scale", "v_scale") if n in s}
        s["optimizer"] = AdamW(p, StateBits=case["bits"], state=state, **s["hyper"])
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    op = s["case"]["op"]
    if own:
        if op == "adamw":
            s["optimizer"].step(s["g"])
            return _adamw_outputs(s)
        from mymedialite_amd import item_log_probs, item_log_probs_grad
        if op == "log_probs":
            r = item_log_probs(s["U"], s["V"], s["bias"], items=s["items"], users=s["users"],
                               exclude=s["seen"], n_top=s["case"]["top"])
            return {"log_probs": r.log_probs, "log_norm": r.log_norm, "entropy": r.entropy,
                    "top_items": r.top_items, "top_log_probs": r.top_log_probs}
        gu, gi, gb = item_log_probs_grad(
            s["U"], s["V"], s["bias"], items=s["items"], log_norm=s["log_norm"],
            entropy=s["entropy"], grad_log_probs=s["g_log_probs"], grad_entropy=s["g_entropy"],
            users=s["users"], exclude=s["seen"])
        return {"grad_users": gu, "grad_items": gi, "grad_bias": gb}
    return {"log_probs": _plain_log_probs, "grad": _plain_grad, "adamw": _plain_adamw}[op](s)


def _scores(s, dtype):
    """Scores [rows, items] in `dtype`, -inf where the row's user has seen the item."""
    users = s["users"].long()
    S = torch.addmm(s["bias"].to(dtype), s["U"][users].to(dtype), s["V"].to(dtype).t())
    if s["seen"] is not None:
        off, seen = s["seen"]
        first, count = off[users], off[users + 1] - off[users]
        row = torch.repeat_interleave(torch.arange(len(users), device="cuda"), count)
        begin = torch.cumsum(count, 0) - count
        at = torch.arange(len(row), device="cuda") - begin[row] + first[row]
        S[row, seen[at].long()] = -math.inf
    return S


def _given(s, S):
    """(rows' item, whether it is one, its score): an item of -1 is none."""
    t = s["items"].long()
    has = (t >= 0) & (t < S.shape[1])
    t = torch.where(has, t, 0)
    return t, has, S.gather(1, t[:, None])[:, 0]


def _top(s, S, n):
    """The n best items of every row by score in 64 bits, the lowest id first among equals."""
    some = torch.topk(S, min(n + 16, S.shape[1]), dim=1).indices.sort(1).values
    gone = torch.isinf(S.gather(1, some))
    u = s["U"][s["users"].long()].double()
    exact = torch.bmm(s["V"][some].double(), u[:, :, None].contiguous())[:, :, 0]
    exact += s["bias"][some].double()
    exact.masked_fill_(gone, -math.inf)
    best, at = torch.sort(exact, dim=1, descending=True, stable=True)
    return best[:, :n], some.gather(1, at)[:, :n].int()


def _plain_log_probs(s):
    n = s["case"]["top"]
    S = _scores(s, torch.float32)
    lse = torch.logsumexp(S, 1)
    t, has, given = _given(s, S)
    zero = torch.zeros_like(lse)
    out = {"log_probs": torch.where(has, given - lse, zero), "log_norm": lse}
    best, ids = _top(s, S, n) if n else (None, None)
    S -= lse[:, None]
    P = torch.exp(S)
    out["entropy"] = -torch.where(P > 0, P * S, 0).sum(1)
    out["top_items"] = ids
    out["top_log_probs"] = (best - lse[:, None].double()).float() if n else None
    return out


def _gradient(s, S):
    """d loss / d scores, from scores in the dtype of `S` (which is overwritten)."""
    t, has, given = _given(s, S)
    lse = s["log_norm"].to(S.dtype)
    w = torch.where(has & ~torch.isinf(given), s["g_log_probs"], 0).to(S.dtype)
    S -= lse[:, None]
    G = torch.exp(S)
    if s["g_entropy"] is None:
        G *= -w[:, None]
    else:
        h = s["g_entropy"].to(S.dtype)
        S.clamp_(min=-1e30)
        c = S.add_(s["entropy"].to(S.dtype)[:, None]).mul_(h[:, None]).add_(w[:, None])
        G.mul_(c).neg_()
    G[torch.arange(len(t), device="cuda"), t] += w
    return G


def _plain_grad(s):
    dtype = s["U"].dtype
    G = _gradient(s, _scores(s, torch.float32))
    u, v = s["U"][s["users"].long()].float(), s["V"].float()
    return {"grad_users": (G @ v).to(dtype), "grad_items": (G.t() @ u).to(dtype),
            "grad_bias": G.sum(0)}


def _quantise(x, root):
    """(e4m3 codes, scale per BLOCK values) of a moment; a root that is not zero stays so."""
    n = x.numel()
    pad = -n % BLOCK
    b = torch.nn.functional.pad(x.reshape(-1), (0, pad)).view(-1, BLOCK)
    scale = b.abs().amax(1) / E4M3_MAX
    q = b / torch.where(scale > 0, scale, 1)[:, None]
    if root:
        q = torch.where(q > 0, q.clamp(min=E4M3_MIN), q)
    return q.to(torch.float8_e4m3fn).view(-1)[:n].view(x.shape).clone(), scale


def _values(q, scale):
    """The values that codes stand for."""
    n = q.numel()
    return q.reshape(-1).float() * scale.repeat_interleave(BLOCK)[:n]


def _adamw_outputs(s):
    return {n: s[n] for n in ("p", "m", "v", "m_scale", "v_scale") if n in s}


def _plain_adamw(s):
    h, bits = s["hyper"], s["case"]["bits"]
    s["step"] += 1
    c1, c2 = 1 - h["Beta1"] ** s["step"], 1 - h["Beta2"] ** s["step"]
    for i, p in enumerate(s["p"]):
        g = s["g"][i].float()
        if bits == 32:
            m, v = s["m"][i], s["v"][i]
        else:
            m = _values(s["m"][i], s["m_scale"][i]).view(p.shape)
            v = _values(s["v"][i], s["v_scale"][i]).view(p.shape).square_()
        m.mul_(h["Beta1"]).add_(g, alpha=1 - h["Beta1"])
        v.mul_(h["Beta2"]).addcmul_(g, g, value=1 - h["Beta2"])
        root = torch.sqrt(v)
        x = p.float()
        x = x - h["LearnRate"] * h["WeightDecay"] * x
        p.copy_(x - (h["LearnRate"] / c1) * m / (root / math.sqrt(c2) + h["Epsilon"]))
        if bits == 8:
            q, scale = _quantise(m, False)
            s["m"][i].copy_(q)
            s["m_scale"][i].copy_(scale)
            q, scale = _quantise(root, True)
            s["v"][i].copy_(q)
            s["v_scale"][i].copy_(scale)
    return _adamw_outputs(s)


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return (_exact_adamw if case["op"] == "adamw" else _exact_softmax)(s)


def _exact_softmax(s):
    case = s["case"]
    R, N, n = case["rows"], case["items"], case.get("top", 0)
    U, V, bias = s["U"].double(), s["V"].double(), s["bias"].double()
    off = seen = None
    if s["seen"] is not None:
        off, seen = s["seen"][0].tolist(), s["seen"][1].long()
    users, items = s["users"].tolist(), s["items"].tolist()
    parts = {}
    grad_items = torch.zeros_like(V)
    grad_bias = torch.zeros_like(bias)
    step = max(1, min(R, 400_000_000 // N))
    for r0 in range(0, R, step):
        rows = range(r0, min(R, r0 + step))
        u = U[[users[r] for r in rows]]
        z = torch.mm(u, V.t()) + bias
        if off is not None:
            for x, r in enumerate(rows):
                z[x, seen[off[users[r]]:off[users[r] + 1]]] = -math.inf
        top = z.max(1, keepdim=True).values
        lse = (top + torch.log(torch.exp(z - top).sum(1, keepdim=True)))[:, 0]
        given = [(x, items[r]) for x, r in enumerate(rows) if 0 <= items[r] < N]
        gx = torch.tensor([x for x, _ in given], device="cuda", dtype=torch.long)
        gt = torch.tensor([t for _, t in given], device="cuda", dtype=torch.long)
        got = {}
        if case["op"] == "log_probs":
            lp = torch.zeros_like(lse)
            lp[gx] = z[gx, gt] - lse[gx]
            got["log_probs"], got["log_norm"] = lp, lse
            if n:
                best, ids = torch.topk(z, n, dim=1)
                got["top_items"], got["top_log_probs"] = ids.int(), best - lse[:, None]
        z -= lse[:, None]  # log p
        p = torch.exp(z)
        z[p == 0] = 0.0
        if case["op"] == "log_probs":
            got["entropy"] = -(p * z).sum(1)
        else:
            w = torch.zeros_like(lse)
            w[gx] = s["g_log_probs"][r0:r0 + len(rows)].double()[gx] * (p[gx, gt] > 0)
            d = -w[:, None] * p
            d[gx, gt] += w[gx]
            if s["g_entropy"] is not None:
                h = s["g_entropy"][r0:r0 + len(rows)].double()
                ent = -(p * z).sum(1, keepdim=True)
                d -= h[:, None] * p * (z + ent)
            got["grad_users"] = d @ V
            grad_items += d.t() @ u
            grad_bias += d.sum(0)
        for name, x in got.items():
            parts.setdefault(name, []).append(x)
    out = {name: torch.cat(x) for name, x in parts.items()}
    if case["op"] == "grad":
        return dict(out, grad_items=grad_items, grad_bias=grad_bias)
    if not n:
        out["top_items"] = out["top_log_probs"] = None
    return out


def _exact_adamw(s):
    h, bits, t = s["hyper"], s["case"]["bits"], s["step"] + 1
    out = {"p": [], "m": [], "v": []}
    if bits == 8:
        out.update(m_scale=[], v_scale=[])
    b1, b2 = h["Beta1"], h["Beta2"]

    def blocks(x):
        flat = torch.zeros(-(-x.numel() // BLOCK) * BLOCK, dtype=torch.float64, device="cuda")
        flat[:x.numel()] = x.reshape(-1)
        return flat.view(-1, BLOCK)

    for i, p in enumerate(s["p"]):
        g, m, v = s["g"][i].double(), s["m"][i].double(), s["v"][i].double()
        if bits == 8:
            m = (blocks(m) * s["m_scale"][i].double()[:, None]).view(-1)[:p.numel()].view(p.shape)
            v = (blocks(v) * s["v_scale"][i].double()[:, None]).view(-1)[:p.numel()].view(p.shape)
            v = v * v
        m = b1 * m + (1 - b1) * g
        v = b2 * v + (1 - b2) * g * g
        x = p.double() * (1 - h["LearnRate"] * h["WeightDecay"])
        x = x - h["LearnRate"] * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t))
                                                        + h["Epsilon"])
        out["p"].append(x)
        if bits == 32:
            out["m"].append(m)
            out["v"].append(v)
            continue
        for name, val in (("m", m), ("v", torch.sqrt(v))):
            b = blocks(val)
            scale = b.abs().amax(1) / E4M3_MAX
            q = b / torch.where(scale > 0, scale, 1.0)[:, None]
            if name == "v":
                q = torch.where((q > 0) & (q < E4M3_MIN), E4M3_MIN, q)
            q = q.float().to(torch.float8_e4m3fn).double()
            out[name].append(q.view(-1)[:p.numel()].view(p.shape))
            out[name + "_scale"].append(scale)
    return out
