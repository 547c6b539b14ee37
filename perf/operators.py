"""Cases of the operators that follow neighbour search in a point transformer layer, and how each is computed.

``gather_rows``   features of the neighbours along an edge list, or embeddings of node types, with the gradient
``norm_rotate``   RMS norm of every head's query and key and rotation by the point's coordinates, with the gradient
``attention``     softmax attention inside each example of a ragged batch, the score capped by a tanh and biased by
                  the distance of the two points, with the gradient; few queries over many keys included

``run`` computes them in elementary tensor operations in 32 bits, or, with ``own`` set, through the public
entry points of ``pytorch_cluster_b200``.  ``exact`` evaluates the definitions in 64 bits, example by example.
"""
import math
import random

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


# ---- cases ---------------------------------------------------------------------------------------------------

def attention_case(name, dtype, train, clouds, points, spread, queries, heads, groups, channels, dims, cap, layout):
    # points: mean rows per cloud, spread: their relative half-width; queries: 0 = the points themselves, else that many
    # queries of their own per cloud; groups: heads of keys and values; dims: coordinates of the bias (0: none)
    return {"name": name, "op": "attention", "dtype": dtype, "train": train, "clouds": clouds, "points": points,
            "spread": spread, "queries": queries, "heads": heads, "groups": groups, "channels": channels, "dims": dims,
            "cap": cap, "layout": layout}


def rotate_case(name, dtype, train, rows, heads, groups, channels, dims, far):
    return {"name": name, "op": "norm_rotate", "dtype": dtype, "train": train, "rows": rows, "heads": heads,
            "groups": groups, "channels": channels, "dims": dims, "far": far}


def gather_case(name, dtype, train, rows, edges, channels, pattern):
    # pattern "near": indices around the edge's own place, as neighbours of ordered points are; "types": a skewed choice
    # of few rows, as node types are
    return {"name": name, "op": "gather_rows", "dtype": dtype, "train": train, "rows": rows, "edges": edges,
            "channels": channels, "pattern": pattern}


def listed():
    return [
        # one cloud of 1024 points at inference: the smallest graph the library is measured on, latency counts
        attention_case("attention-one-cloud", "bfloat16", False, 1, 1024, 0.0, 0, 4, 4, 32, 3, 0.0, 1),
        # a training step's layer over 16 clouds of about 2048 points with 64 channels per head
        attention_case("attention-clouds-train", "bfloat16", True, 16, 2048, 0.25, 0, 8, 8, 64, 3, 0.0, 2),
        # many small molecules: batches of graphs of a few dozen atoms
        attention_case("attention-molecules-train", "float16", True, 2048, 30, 0.8, 0, 8, 8, 32, 3, 0.0, 3),
        # wide heads with shared keys and capped scores over feature vectors without coordinates, inference
        attention_case("attention-capped-grouped", "bfloat16", False, 8, 4096, 0.1, 0, 8, 2, 128, 0, 30.0, 4),
        # one query per cloud over tens of thousands of points: pooling, or a new token over a long memory
        attention_case("attention-one-query", "bfloat16", False, 32, 32768, 0.3, 1, 8, 2, 64, 3, 0.0, 5),
        # full precision, odd channel count, both the cap and the bias, small ragged clouds
        attention_case("attention-float32-train", "float32", True, 8, 511, 0.5, 0, 4, 4, 44, 2, 20.0, 6),
        # 32 clouds of 4096 points in training, coordinates in three dimensions
        rotate_case("rotate-clouds-train", "bfloat16", True, 131072, 8, 8, 64, 3, False),
        # one small cloud at inference
        rotate_case("rotate-one-cloud", "float32", False, 1024, 4, 4, 32, 3, False),
        # sequence positions far from zero, shared keys, wide heads
        rotate_case("rotate-far-train", "float16", True, 4099, 16, 4, 128, 1, True),
        # 20 neighbours of each of 131072 points: the edges of the batched graph workload, training
        gather_case("gather-neighbours-train", "bfloat16", True, 131072, 131072 * 20, 64, "near"),
        # a million atoms of 100 types: few rows, each used thousands of times
        gather_case("gather-types-train", "float32", True, 100, 1000003, 128, "types"),
        # the 16384 edges of one cloud of 1024 points, inference
        gather_case("gather-one-cloud", "float32", False, 1024, 16384, 32, "near"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "norm_rotate", "gather_rows"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    train = rng.random() < 0.5
    if op == "attention":
        groups = rng.choice([1, 2, 4, 8])
        heads = min(16, groups * rng.choice([1, 1, 2, 4]))
        channels = rng.choice([16, 24, 32, 40, 64, 64, 72, 96, 128])
        dims, cap = rng.choice([0, 1, 2, 3, 3]), rng.choice([0.0, 0.0, 15.0, 50.0])
        few = rng.random() < 0.3
        points = _log(rng, 12, 32768 if few else 4096)
        # at most about 5e8 scores (1e8 in 32 bits), and 2^20 keys of all clouds
        most = (1e8 if dtype == "float32" else 5e8) / heads
        queries = rng.randint(1, 8) if few else 0
        clouds = int(max(1, min(2048, most / (1.5 * points * (queries or 1.5 * points)), (1 << 20) / points)))
        clouds = _log(rng, 1, clouds) if clouds > 1 else 1
        return attention_case("", dtype, train and not few, clouds, points, rng.choice([0.0, 0.2, 0.7]), queries, heads,
                              groups, channels, dims, cap, rng.randrange(1 << 20))
    if op == "norm_rotate":
        groups = rng.choice([1, 2, 4, 8])
        heads = min(16, groups * rng.choice([1, 1, 2, 4]))
        channels = rng.choice([16, 24, 32, 48, 64, 96, 128])
        return rotate_case("", dtype, train, _log(rng, 64, (1 << 26) // (heads * channels)), heads, groups, channels,
                           rng.choice([1, 2, 3]), rng.random() < 0.4)
    channels = rng.choice([8, 20, 32, 64, 100, 128, 256])
    pattern = rng.choice(["near", "near", "types"])
    edges = _log(rng, 1000, (1 << 27) // channels)
    rows = _log(rng, 16, 1000) if pattern == "types" else max(16, edges // rng.choice([5, 16, 20, 32]))
    return gather_case("", dtype, train, rows, edges, channels, pattern)


# ---- inputs --------------------------------------------------------------------------------------------------

def _lengths(case):
    r = random.Random(case["layout"])
    p, s = case["points"], case["spread"]
    return [max(1, int(round(p * (1 + s * (2 * r.random() - 1))))) for _ in range(case["clouds"])]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dt)

    s = {"case": case}
    if case["op"] == "attention":
        lens = torch.tensor(_lengths(case), device="cuda")
        n = int(lens.sum())
        s["batch_k"] = torch.arange(case["clouds"], device="cuda").repeat_interleave(lens)
        s["batch_q"] = s["batch_k"] if not case["queries"] else \
            torch.arange(case["clouds"], device="cuda").repeat_interleave(case["queries"])
        m = s["batch_q"].numel()
        # queries a little larger than unit, so that the softmax is neither flat nor a single key
        s["q"] = normal(m, case["heads"], case["channels"], scale=2.0)
        s["k"] = normal(n, case["groups"], case["channels"])
        s["v"] = normal(n, case["groups"], case["channels"])
        s["pos_q"] = s["pos_k"] = s["slope"] = None
        if case["dims"]:
            s["pos_k"] = torch.randn(n, case["dims"], generator=g, device="cuda")
            s["pos_q"] = s["pos_k"] if not case["queries"] else \
                torch.randn(m, case["dims"], generator=g, device="cuda")
            s["slope"] = 2.0 ** -torch.arange(case["heads"], device="cuda").float()
        if case["train"]:
            s["dout"] = normal(m, case["heads"], case["channels"])
    elif case["op"] == "norm_rotate":
        s["q"] = normal(case["rows"], case["heads"], case["channels"])
        s["k"] = normal(case["rows"], case["groups"], case["channels"])
        half, d = case["channels"] // 2, case["dims"]
        if case["far"]:
            # whole positions up to a million
            s["pos"] = torch.randint(0, 1000000, (case["rows"], d), generator=g, device="cuda").float()
            s["freq"] = (10000.0 ** (-torch.arange(half, device="cuda").float() / half)).expand(d, half).contiguous()
        else:
            s["pos"] = torch.randn(case["rows"], d, generator=g, device="cuda")
            s["freq"] = torch.randn(d, half, generator=g, device="cuda") * 4
        s["weight_q"] = 1 + 0.1 * torch.randn(case["channels"], generator=g, device="cuda")
        s["weight_k"] = 1 + 0.1 * torch.randn(case["channels"], generator=g, device="cuda")
        if case["train"]:
            s["dq"], s["dk"] = normal(*s["q"].shape), normal(*s["k"].shape)
    else:
        n, e = case["rows"], case["edges"]
        s["x"] = normal(n, case["channels"])
        if case["pattern"] == "near":
            home = torch.arange(e, device="cuda") * n // e
            step = (torch.randn(e, generator=g, device="cuda") * 200).long()
            s["index"] = (home + step).remainder(n)
        else:
            s["index"] = (torch.rand(e, generator=g, device="cuda") ** 3 * n).long().clamp_(max=n - 1)
        s["scale"] = math.sqrt(case["channels"])
        if case["train"]:
            s["dout"] = normal(e, case["channels"])
    return s


# ---- the plain form ------------------------------------------------------------------------------------------

def _padded(batch, clouds, rows):
    # row numbers [clouds, rows] of every cloud's places, and which of them are taken
    ptr = torch.searchsorted(batch, torch.arange(clouds + 1, device=batch.device))
    at = ptr[:-1, None] + torch.arange(rows, device=batch.device)
    return at.clamp(max=batch.numel() - 1), at < ptr[1:, None]


def _plain_attention(case, q, k, v, batch_q, batch_k, pos_q, pos_k, slope):
    b, h, g, c = case["clouds"], case["heads"], case["groups"], case["channels"]
    most = max(_lengths(case))
    at_k, ok_k = _padded(batch_k, b, most)
    at_q, ok_q = _padded(batch_q, b, case["queries"] or most)
    qf = q.float()[at_q].view(b, -1, g, h // g, c).permute(0, 2, 3, 1, 4)            # [b, g, h/g, m, c]
    kf = k.float()[at_k].permute(0, 2, 3, 1).unsqueeze(2)                            # [b, g, 1, c, n]
    vf = v.float()[at_k].permute(0, 2, 1, 3).unsqueeze(2)                            # [b, g, 1, n, c]
    s = (qf * c ** -0.5) @ kf
    if case["cap"]:
        s = case["cap"] * torch.tanh(s / case["cap"])
    if pos_q is not None:
        far = (pos_q[at_q].unsqueeze(2) - pos_k[at_k].unsqueeze(1)).square().sum(-1).sqrt()
        s = s - slope.view(1, g, h // g, 1, 1) * far[:, None, None]
    s = s.masked_fill(~ok_k[:, None, None, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-3e38))
    p = p / p.sum(-1, keepdim=True)
    o = (p @ vf).permute(0, 3, 1, 2, 4).reshape(b, -1, h, c)
    return o[ok_q].to(q.dtype)


def _plain_rotate(x, pos, freq, weight, eps):
    xf = x.float()
    u = xf * torch.rsqrt(xf.square().mean(-1, keepdim=True) + eps) * weight
    angle = (pos.double() @ freq.double())[:, None]
    cos, sin = angle.cos().float(), angle.sin().float()
    a, b = u.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(x.dtype)


def _plain_gather_gradient(dout, index, rows, scale):
    dx = torch.zeros(rows, dout.size(1), device=dout.device)
    return (dx.index_add_(0, index, dout.float()) * scale).to(dout.dtype)


def _leaf(t):
    return t.detach().requires_grad_()


def run(state):
    s, case = state, state["case"]
    train = case["train"]
    if own:
        import pytorch_cluster_b200 as ops
    if case["op"] == "attention":
        q, k, v = (_leaf(s[n]) if train else s[n] for n in "qkv")
        rest = (s["batch_q"], s["batch_k"], s["pos_q"], s["pos_k"], s["slope"])
        if own:
            out = ops.attention(q, k, v, *rest, cap=case["cap"] or None, batch_size=case["clouds"])
        else:
            out = _plain_attention(case, q, k, v, *rest)
        return [out.detach(), *torch.autograd.grad(out, (q, k, v), s["dout"])] if train else out
    if case["op"] == "norm_rotate":
        leaves = [_leaf(s[n]) if train else s[n] for n in ("q", "k", "weight_q", "weight_k")]
        q, k, wq, wk = leaves
        if own:
            a, b = ops.norm_rotate(q, k, s["pos"], s["pos"], s["freq"], wq, wk, eps=1e-6)
        else:
            a, b = (_plain_rotate(x, s["pos"], s["freq"], w, 1e-6) for x, w in ((q, wq), (k, wk)))
        if not train:
            return [a, b]
        return [a.detach(), b.detach(), *torch.autograd.grad((a, b), leaves, (s["dq"], s["dk"]))]
    if own:
        x = _leaf(s["x"]) if train else s["x"]
        out = ops.gather_rows(x, s["index"], s["scale"])
        return [out.detach(), *torch.autograd.grad(out, x, s["dout"])] if train else out
    out = (s["x"].float().index_select(0, s["index"]) * s["scale"]).to(s["x"].dtype)
    return [out, _plain_gather_gradient(s["dout"], s["index"], case["rows"], s["scale"])] if train else out


# ---- the definition in 64 bits -------------------------------------------------------------------------------

def _exact_attention(case, s):
    b, h, g, c = case["clouds"], case["heads"], case["groups"], case["channels"]
    lens_k = _lengths(case)
    lens_q = [case["queries"] or n for n in lens_k]
    rep = h // g
    out, grads = [], ([], [], [])
    i = j = 0
    for mq, nk in zip(lens_q, lens_k):
        q = s["q"][i:i + mq].double().transpose(0, 1)                                    # [h, m, c]
        k = s["k"][j:j + nk].double().transpose(0, 1).repeat_interleave(rep, 0)         # [h, n, c]
        v = s["v"][j:j + nk].double().transpose(0, 1).repeat_interleave(rep, 0)
        raw = torch.einsum("hmc,hnc->hmn", q, k) / math.sqrt(c)
        bent = torch.tanh(raw / case["cap"]) if case["cap"] else None
        z = raw if bent is None else case["cap"] * bent
        if case["dims"]:
            z = z - s["slope"].double()[:, None, None] * torch.cdist(
                s["pos_q"][i:i + mq].double(), s["pos_k"][j:j + nk].double(),
                compute_mode="donot_use_mm_for_euclid_dist")
        p = torch.softmax(z, -1)
        o = torch.einsum("hmn,hnc->hmc", p, v)
        out.append(o.transpose(0, 1))
        if case["train"]:
            do = s["dout"][i:i + mq].double().transpose(0, 1)
            dz = p * (torch.einsum("hmc,hnc->hmn", do, v) - (do * o).sum(-1, keepdim=True))
            if bent is not None:
                dz = dz * (1 - bent * bent)
            dz = dz / math.sqrt(c)
            grads[0].append(torch.einsum("hmn,hnc->hmc", dz, k).transpose(0, 1))
            for n, t in ((1, torch.einsum("hmn,hmc->hnc", dz, q)), (2, torch.einsum("hmn,hmc->hnc", p, do))):
                grads[n].append(t.view(g, rep, nk, c).sum(1).transpose(0, 1))
        i, j = i + mq, j + nk
    out = torch.cat(out)
    return [out, *(torch.cat(t) for t in grads)] if case["train"] else out


def _exact_rotate(x, pos, freq, weight, eps, dy):
    n, h, c = x.shape
    x, w = x.double(), weight.double()
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device),
                       torch.einsum("nd,dp->np", pos.double(), freq.double()))[:, None]
    r = 1 / torch.sqrt((x * x).sum(-1, keepdim=True) / c + eps)
    z = torch.complex(*torch.split(x * r * w, c // 2, -1)) * turn
    y = torch.cat([z.real, z.imag], -1)
    if dy is None:
        return y, None, None
    gz = torch.complex(*torch.split(dy.double(), c // 2, -1)) * turn.conj()
    gu = torch.cat([gz.real, gz.imag], -1)
    dw = (gu * x * r).sum((0, 1))
    t = gu * w
    return y, t * r - x * r ** 3 * (t * x).sum(-1, keepdim=True) / c, dw


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(case, s)
    if case["op"] == "norm_rotate":
        train = case["train"]
        a, da, dwa = _exact_rotate(s["q"], s["pos"], s["freq"], s["weight_q"], 1e-6, s["dq"] if train else None)
        b, db, dwb = _exact_rotate(s["k"], s["pos"], s["freq"], s["weight_k"], 1e-6, s["dk"] if train else None)
        return [a, b, da, db, dwa, dwb] if train else [a, b]
    out = s["x"].double()[s["index"]] * s["scale"]
    if not case["train"]:
        return out
    dx = torch.zeros(case["rows"], case["channels"], dtype=torch.float64, device="cuda")
    dx.scatter_add_(0, s["index"][:, None].expand(-1, case["channels"]), s["dout"].double())
    return [out, dx * s["scale"]]


# ---- work ----------------------------------------------------------------------------------------------------

def work(case):
    size = DTYPES[case["dtype"]].itemsize
    train = case["train"]
    if case["op"] == "attention":
        lens = _lengths(case)
        n = sum(lens)
        m = case["queries"] * case["clouds"] or n
        pairs = sum((case["queries"] or t) * t for t in lens) * case["heads"]
        qo, kv = m * case["heads"] * case["channels"] * size, 2 * n * case["groups"] * case["channels"] * size
        places = 4 * case["dims"] * (n + (m if case["queries"] else 0)) + 8 * (n + (m if case["queries"] else 0))
        # forward: q, k, v in, o out; backward: dout in, dq, dk, dv out
        return {"bytes": 2 * qo + kv + places + (2 * qo + kv if train else 0),
                "flops": pairs * case["channels"] * (4 + (10 if train else 0))}
    if case["op"] == "norm_rotate":
        x = case["rows"] * (case["heads"] + case["groups"]) * case["channels"]
        places = 4 * case["rows"] * case["dims"] + 2 * case["dims"] * case["channels"] + 8 * case["channels"]
        # per value: square and sum, scale and weight, rotate (3); about twice that backward
        return {"bytes": x * size * (4 if train else 2) + places + (8 * case["channels"] if train else 0),
                "flops": x * (7 + (14 if train else 0))}
    used = min(case["rows"], case["edges"])
    e = case["edges"] * case["channels"]
    # forward: index and rows in, edges out; backward: edges in, rows out
    return {"bytes": 8 * case["edges"] + (used * case["channels"] + e) * size * (2 if train else 1),
            "flops": e * (2 if train else 1)}
